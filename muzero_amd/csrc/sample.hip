// mz_sample_actions: one entry of every row of logits, drawn from a given random number after temperature, top-k, top-p and
// min-p.  A row z[0..A) with its legal mask:
//     x_i = (z_i - max z) / T,  w_i = exp(x_i)                  over the legal, finite entries (a row of none: action -1)
//     ranking: z descending, index ascending on ties; each filter keeps a prefix of it, so all of them keep the shortest:
//       top-k: the first k;  top-p: entries whose predecessors (within the first k) hold less than p of those k's mass;
//       min-p: entries with w_i >= m (max w = 1)
//     draw: the first kept i in INDEX order with sum_{j <= i, kept} w_j > u * S,  S = the kept mass.
// Whether an entry is kept and which is drawn are decided by sums next to a border, so weights and sums are 64-bit: an entry of
// relative weight 1e-7 next to the border of a nucleus must not depend on the order of a sum.  Sums run in a fixed order, or
// (histograms, whose LDS atomics arrive in any order) in exact integers, so a row's answer is a function of the row and of the kernel,
// which goes by the numbers of rows and actions; between kernels the order of the sums differs.
//
//   A <= 256   k_sample_wave: a wavefront per row, the row in registers (<= 4 entries a lane); ranking = bitonic sort of
//              the keys over the lanes.  Bound by the issue of vector instructions, 64-bit exponentials first: 16384 rows of 82 with
//              top-k, top-p and min-p of their own and probabilities written: 22 us, 0.55 TB/s.  (By a workgroup per row, as
//              below, 4096 rows of 256 take 58 us instead of 13.)
//   A >  256   k_sample_block: a workgroup per row, passes over the row (its re-reads hit L2 / the memory-side cache):
//              maximum -> candidates.  With top-k <= 128 the k-th largest of 256 partial maxima bounds the k-th entry from
//              below, so about k entries pass and one wave finishes as above.  A nucleus without top-k needs the mass of the
//              whole row: a histogram of count and mass over log2-spaced bins gives it, and the bin the border falls in;
//              small nuclei are finished by one wave, large ones narrow the border's bin to one (value, index).  256 rows of 131072
//              bf16 entries: with top-k 50 30 us (2.2 TB/s), with top-p 0.9 131 us, bound by vector and LDS atomic work per entry.
//   few long rows   k_sample_maxima + k_sample_split: 2 to 16 workgroups per row, the last to finish ranks the candidates of
//              all; 64 rows of 50257 fp32 entries, top-k 40 and top-p 0.95: 16 us, bound by latency (two launches, one wave's end).
//              Rows that no short cut serves are left to one workgroup each: one row of 131072 bf16, top-p 0.9 100 us, no filter
//              46, top-k 1000 79.
#include "ops.h"

#include <float.h>
#include <math.h>

namespace mz {
namespace {

constexpr int W = 64;
constexpr int kWaveRows = 4;       // rows (waves) per workgroup of k_sample_wave
constexpr int kList = 256;         // candidates one wave ranks in registers
constexpr int kFastK = 128;        // top-k up to which the bound by partial maxima is tried
constexpr int kBins = 2048;
constexpr int kFix = 45;           // fraction bits of a histogram mass: 2^45.51 per entry * 2^18 entries < 2^64

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned long long u64;

// ---- weights -------------------------------------------------------------------------------------------------------------
// 2^f on [-0.5, 0.5]: 1 + f q(f), q the degree-9 polynomial through (2^f - 1) / f at the Chebyshev points (relative error of
// 2^f 6e-16); 2^0 is exactly 1.
__device__ __forceinline__ double exp2_frac(double f) {
    double q = 0x1.e5e9f548e5726p-28;
    q = fma(q, f, 0x1.b6571de2f2351p-24);
    q = fma(q, f, 0x1.62bfe46117445p-20);
    q = fma(q, f, 0x1.ffcb76789860fp-17);
    q = fma(q, f, 0x1.4309130378460p-13);
    q = fma(q, f, 0x1.5d87fe908f88ap-10);
    q = fma(q, f, 0x1.3b2ab6fba385fp-7);
    q = fma(q, f, 0x1.c6b08d7044119p-5);
    q = fma(q, f, 0x1.ebfbdff82c590p-3);
    q = fma(q, f, 0x1.62e42fefa39f7p-1);
    return fma(q, f, 1.0);
}
// The row's scale: x / ln 2 = (z - zmax) * c.  A maximum of +inf stands as 2^128 with a c that leaves no weight to finite
// entries; T = 5e-324 would make c infinite, and 0 * inf is not wanted.
struct Scale {
    double zmax, c;
};
__device__ __forceinline__ Scale make_scale(float zmax, double T) {
    const bool inf = zmax == INFINITY;
    Scale s;
    s.zmax = inf ? 0x1p128 : (double)zmax;
    s.c = inf ? 1e290 : fmin(1.4426950408889634 / T, 1e290);
    return s;
}
// y = (z - zmax) / (T ln 2) in [low, 0]
__device__ __forceinline__ double log2_weight(float z, const Scale& s, double low) { return fmax(fmin(((double)z - s.zmax) * s.c, 0.0), low); }
// log of the share of an entry: x - log(total)
__device__ __forceinline__ double log_share(float z, float zmax, double T, double total) {
    return (z == zmax ? 0.0 : ((double)z - (double)zmax) / T) - log(total);
}
// Integers and 64-bit floats meet in the low word of 1.5 * 2^52 + n: an addition rounds to the nearest integer and shows it
// there; conversions, rounding and ldexp instructions run at a quarter of the rate of an addition.
constexpr double kRound = 6755399441055744.0;
__device__ __forceinline__ int low_word(double v) { return (int)(uint32_t)__double_as_longlong(v); }
__device__ __forceinline__ double scaled(double p, int n) {   // p 2^n, p and the result normal numbers
    const u64 b = (u64)__double_as_longlong(p);
    return __longlong_as_double((long long)((u64)((uint32_t)(b >> 32) + ((uint32_t)n << 20)) << 32 | (uint32_t)b));
}
constexpr double kNoWeight = -1023.0;                          // and below: scaled(1.0, -1023) is 0, the weight of -inf too
__device__ __forceinline__ double weight(float z, const Scale& s) {
    const double y = log2_weight(z, s, kNoWeight), t = y + kRound;
    return scaled(exp2_frac(y - (t - kRound)), low_word(t));
}

// The same for N entries side by side: the constants of the polynomial stay in scalar registers (compiled from exp2_frac each step
// is a move and a two-operand FMA).  The results must not go into DPP operations directly - the compiler does not see that a
// vector instruction wrote them - but through a selection, an addition or the like.
__device__ __forceinline__ double fma_scalar(double a, double b, double c) {
    double r;
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "s"(c));
    return r;
}
template <int N>
__device__ __forceinline__ void exp2_fracs(const double (&f)[N], double (&p)[N]) {
    constexpr double k[10] = {0x1.e5e9f548e5726p-28, 0x1.b6571de2f2351p-24, 0x1.62bfe46117445p-20, 0x1.ffcb76789860fp-17, 0x1.4309130378460p-13,
                              0x1.5d87fe908f88ap-10, 0x1.3b2ab6fba385fp-7,  0x1.c6b08d7044119p-5,  0x1.ebfbdff82c590p-3,  0x1.62e42fefa39f7p-1};
#pragma unroll
    for (int i = 0; i < N; i++) p[i] = k[0];
#pragma unroll
    for (int j = 1; j < 10; j++)
#pragma unroll
        for (int i = 0; i < N; i++) p[i] = fma_scalar(p[i], f[i], k[j]);
#pragma unroll
    for (int i = 0; i < N; i++) p[i] = fma(p[i], f[i], 1.0);
}
template <int N>
__device__ __forceinline__ void weights(const float (&z)[N], const Scale& s, double (&w)[N]) {
    double f[N];
    int n[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        const double y = log2_weight(z[i], s, kNoWeight), t = y + kRound;
        n[i] = low_word(t);
        f[i] = y - (t - kRound);
    }
    exp2_fracs(f, w);
#pragma unroll
    for (int i = 0; i < N; i++) w[i] = scaled(w[i], n[i]);
}

// ---- order-preserving keys ---------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t key_of(float z) {
    const uint32_t b = __float_as_uint(z);
    return b ^ ((int)b < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k ^ ((int)k < 0 ? 0x80000000u : 0xffffffffu)); }
constexpr uint32_t kNoKey = 0x007fffffu;   // key of -inf: an entry that takes no part
// The upper end of a range of keys as the largest key that an entry can have: entries are keyed as z + 0, so none has the key of -0.
// As a float that end is equal to +0, whose key lies above it: a comparison of floats would take the zeros into the range.
__device__ __forceinline__ uint32_t upper_end(uint32_t k) { return k == 0x7fffffffu ? k - 1 : k; }
// ranking as an unsigned 64-bit order: larger z first, then smaller index; 0 = no entry
__device__ __forceinline__ u64 rank_of(float z, int i) { return z > -INFINITY ? ((u64)key_of(z + 0.0f) << 32) | (uint32_t)~i : 0ull; }
__device__ __forceinline__ int index_of_rank(u64 r) { return (int)~(uint32_t)r; }

// ---- wave primitives -----------------------------------------------------------------------------------------------------
// Lanes exchange through DPP (inside rows of 16) and row / half swaps, which need neither LDS nor its latency.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_rows(uint32_t v) {   // 0 in the rows that are not written and from lanes that are not there
    if constexpr (ROWS == 0xf) return dpp<CTRL>(v);
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
template <int J>
__device__ __forceinline__ uint32_t xor_lane(uint32_t v, int lane) {
    if constexpr (J == 1) return dpp<0xB1>(v);                 // quad_perm [1, 0, 3, 2]
    else if constexpr (J == 2) return dpp<0x4E>(v);            // quad_perm [2, 3, 0, 1]
    else if constexpr (J == 4) return dpp<0x141>(dpp<0x1B>(v));   // reversed quads, then reversed halves of 8
    else if constexpr (J == 8) return dpp<0x128>(v);           // rotate a row by 8
    else if constexpr (J == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);   // rows 0, 0, 2, 2 and 1, 1, 3, 3
        return lane & 16 ? r[0] : r[1];
    } else {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);   // lower halves, upper halves
        return lane & 32 ? r[0] : r[1];
    }
}
template <int J>
__device__ __forceinline__ u64 xor_lane(u64 v, int lane) {
    return (u64)xor_lane<J>((uint32_t)(v >> 32), lane) << 32 | xor_lane<J>((uint32_t)v, lane);
}
__device__ __forceinline__ uint32_t lane_value(uint32_t v, int l) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); }
__device__ __forceinline__ u64 lane_value(u64 v, int l) { return (u64)lane_value((uint32_t)(v >> 32), l) << 32 | lane_value((uint32_t)v, l); }
__device__ __forceinline__ double lane_value(double v, int l) { return __longlong_as_double((long long)lane_value((u64)__double_as_longlong(v), l)); }
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

template <int CTRL, int ROWS>
__device__ __forceinline__ void scan_step(double& v) {
    const u64 b = (u64)__double_as_longlong(v);
    v += __longlong_as_double((long long)((u64)dpp_rows<CTRL, ROWS>((uint32_t)(b >> 32)) << 32 | dpp_rows<CTRL, ROWS>((uint32_t)b)));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ void scan_step(int& v) { v += (int)dpp_rows<CTRL, ROWS>((uint32_t)v); }
template <typename V>
__device__ __forceinline__ V wave_scan(V v) {   // inclusive
    scan_step<0x111, 0xf>(v);                   // row_shr 1, 2, 4, 8
    scan_step<0x112, 0xf>(v);
    scan_step<0x114, 0xf>(v);
    scan_step<0x118, 0xf>(v);
    scan_step<0x142, 0xa>(v);                   // the end of rows 0 and 2 to rows 1 and 3
    scan_step<0x143, 0xc>(v);                   // the end of row 1 to rows 2 and 3
    return v;
}
__device__ __forceinline__ double one_lane_up(double v) {   // 0 into lane 0
    const u64 b = (u64)__double_as_longlong(v);
    return __longlong_as_double((long long)((u64)dpp_rows<0x138, 0xf>((uint32_t)(b >> 32)) << 32 | dpp_rows<0x138, 0xf>((uint32_t)b)));   // wave_shr 1
}
__device__ __forceinline__ double wave_sum(double v) { return lane_value(wave_scan(v), 63); }
__device__ __forceinline__ int wave_sum(int v) { return (int)lane_value((uint32_t)wave_scan(v), 63); }
__device__ __forceinline__ float wave_max(float v, int lane) {
    uint32_t k = key_of(v);
    k = max(k, xor_lane<1>(k, lane));
    k = max(k, xor_lane<2>(k, lane));
    k = max(k, xor_lane<4>(k, lane));
    k = max(k, xor_lane<8>(k, lane));
    k = max(k, xor_lane<16>(k, lane));
    k = max(k, xor_lane<32>(k, lane));
    return of_key((uint32_t)uniform((int)k));
}
template <int E, int K, int J, typename V>
__device__ __forceinline__ void sort_step(V (&r)[E], int lane) {
    if constexpr (J >= W) {
        constexpr int S = J / W;
#pragma unroll
        for (int e = 0; e < E; e++)
            if (!(e & S)) {
                const bool desc = ((e * W) & K) == 0;   // K > 64: the bit does not depend on the lane
                const V a = max(r[e], r[e | S]), b = min(r[e], r[e | S]);
                r[e] = desc ? a : b;
                r[e | S] = desc ? b : a;
            }
    } else {
#pragma unroll
        for (int e = 0; e < E; e++) {
            const V o = xor_lane<J>(r[e], lane);
            const bool big = (((e * W + lane) & K) == 0) == ((lane & J) == 0);   // this position keeps the larger of the pair
            r[e] = big ? max(r[e], o) : min(r[e], o);
        }
    }
    if constexpr (J > 1) sort_step<E, K, J / 2>(r, lane);
}
// descending bitonic sort of 64 E values, position e * 64 + lane
template <int E, typename V, int K = 2>
__device__ __forceinline__ void wave_sort(V (&r)[E], int lane) {
    sort_step<E, K, K / 2>(r, lane);
    if constexpr (K < W * E) wave_sort<E, V, K * 2>(r, lane);
}
template <int E, typename V>
__device__ __forceinline__ V at_position(const V (&r)[E], int p) {   // p uniform
    p = uniform(p);
    V v = 0;
#pragma unroll
    for (int e = 0; e < E; e++) {
        const V t = lane_value(r[e], p & 63);
        v = (p >> 6) == e ? t : v;
    }
    return v;
}

// ---- parameters of a row -------------------------------------------------------------------------------------------------
struct RowParams {
    double T, p, m, u;
    int k;
    bool valid;
};
__device__ __forceinline__ RowParams row_params(const SampleOp& op, int row) {
    RowParams r;
    r.T = op.row_temperature ? op.row_temperature[row] : op.temperature;
    r.k = op.row_top_k ? op.row_top_k[row] : op.top_k;
    r.p = op.row_top_p ? op.row_top_p[row] : op.top_p;
    r.m = op.row_min_p ? op.row_min_p[row] : op.min_p;
    r.u = op.u[row];
    // the host checks the scalars; what arrives in device arrays is checked here (every comparison is false for NaN)
    r.valid = r.T >= 0 && r.T <= DBL_MAX && r.k >= 0 && r.p > 0 && r.p <= 1 && r.m >= 0 && r.m <= 1 && r.u >= 0 && r.u <= 1;
    return r;
}
__device__ __forceinline__ void write_row(const SampleOp& op, int row, int action, double logprob, int kept) {
    op.action[row] = action;
    if (op.logprob) op.logprob[row] = (float)logprob;
    if (op.kept) op.kept[row] = kept;
}

__device__ __forceinline__ float z_of(uint32_t key) { return of_key(key); }
__device__ __forceinline__ float z_of(u64 rank) { return of_key((uint32_t)(rank >> 32)); }
// Entries ranked[] (keys or rank values, descending, position e * 64 + lane, `count` of them real): the length of the prefix
// that the filters keep.  `mass` < 0: top-p goes by the mass of the first k here; else by `mass`.
template <int E, typename V>
__device__ __forceinline__ int kept_prefix(const V (&ranked)[E], int count, const RowParams& rp, const Scale& sc, double mass, int lane) {
    int n = rp.k > 0 ? min(rp.k, count) : count;
    if (rp.p < 1 || rp.m > 0) {
        double before[E], carry = 0;
        int nm = 0;
        float z[E];
        double all[E];
#pragma unroll
        for (int e = 0; e < E; e++) z[e] = z_of(ranked[e]);
        weights(z, sc, all);
#pragma unroll
        for (int e = 0; e < E; e++) {
            const bool in = e * W + lane < n;
            const double w = in ? all[e] : 0.0;
            const double s = wave_scan(w);
            before[e] = carry + one_lane_up(s);
            carry += lane_value(s, 63);
            nm += __popcll(__ballot(in && w >= rp.m));
        }
        if (rp.p < 1) {
            const double target = rp.p * (mass < 0 ? carry : mass);
            int np = 0;
#pragma unroll
            for (int e = 0; e < E; e++) np += __popcll(__ballot(e * W + lane < n && before[e] < target));
            n = min(n, np);
        }
        n = min(n, nm);
    }
    return max(n, 1);   // the maximum always stays
}

// The draw over weights in index order, position e * 64 + lane: position of the drawn entry, and the sum of the weights.
template <int E>
__device__ __forceinline__ int wave_draw(const double (&w)[E], double u, double* total) {
    double cum[E], carry = 0;
#pragma unroll
    for (int e = 0; e < E; e++) {
        const double s = wave_scan(w[e]);
        cum[e] = carry + s;
        carry += lane_value(s, 63);
    }
    *total = carry;
    const double target = u * carry;
    int first = -1, last = 0;
#pragma unroll
    for (int e = 0; e < E; e++) {
        const u64 over = __ballot(w[e] > 0 && cum[e] > target), some = __ballot(w[e] > 0);
        if (first < 0 && over) first = e * W + __ffsll(over) - 1;
        if (some) last = e * W + 63 - __clzll(some);
    }
    return first < 0 ? last : first;   // u = 1
}

// ---- element access ------------------------------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
struct bf16_t {
    uint16_t b;
};
template <>
__device__ __forceinline__ float to_float<bf16_t>(bf16_t v) { return __uint_as_float((uint32_t)v.b << 16); }
template <>
__device__ __forceinline__ float to_float<_Float16>(_Float16 v) { return (float)v; }
// an entry that takes no part becomes -inf; -0 becomes +0 (they rank as equals)
__device__ __forceinline__ float clean(float z, bool legal) { return legal && z > -INFINITY ? z + 0.0f : -INFINITY; }

// ---- a wavefront per row (A <= 64 E) ---------------------------------------------------------------------------------------
template <typename T, int E>
__global__ __launch_bounds__(W * kWaveRows) void k_sample_wave(SampleOp op) {
    const int lane = threadIdx.x & 63, row = blockIdx.x * kWaveRows + (threadIdx.x >> 6);
    if (row >= op.rows) return;
    const int A = op.actions;
    const T* src = static_cast<const T*>(op.logits) + row * op.row_stride;
    const uint8_t* legal = op.legal ? op.legal + row * op.legal_stride : nullptr;
    float z[E];
    float zmax = -INFINITY;
    int count = 0;
#pragma unroll
    for (int e = 0; e < E; e++) {
        const int i = e * W + lane;
        z[e] = i < A ? clean(to_float(src[i]), !legal || legal[i]) : -INFINITY;
        zmax = fmaxf(zmax, z[e]);
        count += __popcll(__ballot(z[e] > -INFINITY));
    }
    const RowParams rp = row_params(op, row);
    zmax = wave_max(zmax, lane);
    float* probs = op.probs ? op.probs + row * op.probs_stride : nullptr;
    if (!rp.valid || count == 0) {
        if (lane == 0) write_row(op, row, -1, 0.0, 0);
        if (probs)
            for (int i = lane; i < A; i += W) probs[i] = 0.f;
        return;
    }
    if (rp.T == 0) {
        int pick = -1;
#pragma unroll
        for (int e = 0; e < E; e++) {
            const u64 b = __ballot(z[e] == zmax);
            if (pick < 0 && b) pick = e * W + __ffsll(b) - 1;
        }
        if (lane == 0) write_row(op, row, pick, 0.0, 1);
        if (probs)
            for (int i = lane; i < A; i += W) probs[i] = i == pick ? 1.f : 0.f;
        return;
    }
    const Scale sc = make_scale(zmax, rp.T);
    int n = count;
    uint32_t border = 0;     // kept: keys above it, and the first `ties` equal to it
    int ties = 64 * E;
    uint32_t key[E];
#pragma unroll
    for (int e = 0; e < E; e++) key[e] = z[e] > -INFINITY ? key_of(z[e]) : 0u;
    const bool cut = (rp.k > 0 && rp.k < count) || rp.p < 1;
    if (cut) {
        uint32_t r[E];
#pragma unroll
        for (int e = 0; e < E; e++) r[e] = key[e];
        wave_sort<E>(r, lane);
        n = kept_prefix<E>(r, count, rp, sc, -1.0, lane);
        border = at_position<E>(r, n - 1);
        ties = n;
#pragma unroll
        for (int e = 0; e < E; e++) ties -= __popcll(__ballot(r[e] > border));
    }
    double w[E];
    int before = 0, kept = 0;
    weights(z, sc, w);
#pragma unroll
    for (int e = 0; e < E; e++) {
        const u64 eq = __ballot(key[e] == border);
        const int nth = before + __builtin_amdgcn_mbcnt_hi((uint32_t)(eq >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)eq, 0));
        before += __popcll(eq);
        const bool keep = key[e] != 0 && (key[e] > border || (key[e] == border && nth < ties)) && (cut || w[e] >= rp.m);
        kept += __popcll(__ballot(keep));
        w[e] = keep ? w[e] : 0.0;
    }
    double total;
    const int pick = wave_draw<E>(w, rp.u, &total);
    const float zp = of_key(at_position<E>(key, pick));
    if (lane == 0) {
        write_row(op, row, pick, log_share(zp, zmax, rp.T, total), kept);
    }
    if (probs) {
        const double share = 1.0 / total;
#pragma unroll
        for (int e = 0; e < E; e++)
            if (e * W + lane < A) probs[e * W + lane] = (float)(w[e] * share);
    }
}

// ---- a workgroup per row ---------------------------------------------------------------------------------------------------
template <typename T>
struct Vec {
    static constexpr int N = 16 / sizeof(T);
    float z[N];
    int i0;                 // index of z[0]
};
template <typename T>
struct RowView {
    const T* src;
    const uint8_t* legal;
    int A, nvec;            // A >= Vec<T>::N; vector v = the entries [v N, v N + N), the last one moved back to end with the row
};
template <typename T>
struct Raw {
    u32x4 d;
    uint32_t legal[Vec<T>::N / 4];
};
// Vector v: 16 bytes wherever they start, and their legal flags
template <typename T>
__device__ __forceinline__ Raw<T> load_raw(const RowView<T>& r, int v) {
    constexpr int N = Vec<T>::N;
    const int i0 = min(v * N, r.A - N);
    Raw<T> o;
    __builtin_memcpy(&o.d, r.src + i0, 16);
    if (r.legal) __builtin_memcpy(o.legal, r.legal + i0, N);
    return o;
}
// Masked entries, and in the last vector those that the vector before has, become -inf; a vector behind the last (v >= end) is
// all that.  NaN and -0 are left in: every use compares (NaN is above and equal to nothing), and rank_of takes -0 for 0.
template <typename T>
__device__ __forceinline__ Vec<T> unpack(const RowView<T>& r, const Raw<T>& raw, int v, int end) {
    constexpr int N = Vec<T>::N;
    Vec<T> o;
    const int want = v * N;
    o.i0 = min(want, r.A - N);
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; i++) o.z[i] = __uint_as_float(raw.d[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint16_t h = (uint16_t)(raw.d[i >> 1] >> (16 * (i & 1)));
            T t;
            __builtin_memcpy(&t, &h, 2);
            o.z[i] = to_float(t);
        }
    }
    if (r.legal) {
#pragma unroll
        for (int i = 0; i < N; i++) o.z[i] = (raw.legal[i >> 2] >> (8 * (i & 3)) & 255u) ? o.z[i] : -INFINITY;
    }
    if (v >= end || want != o.i0) {
        const int skip = v >= end ? N : want - o.i0;
#pragma unroll
        for (int i = 0; i < N; i++)
            if (i < skip) o.z[i] = -INFINITY;
    }
    return o;
}
// f(vector) over this wave's vectors [v0, v1): lanes take consecutive vectors, all lanes take part in every call
template <typename T, typename F>
__device__ __forceinline__ void wave_pass(const RowView<T>& r, int v0, int v1, int lane, F f) {
    if (v0 >= v1) return;
    Raw<T> n0 = load_raw(r, v0 + lane), n1 = load_raw(r, v0 + W + lane);   // two loads ahead (behind the last vector: the last again)
#pragma unroll 1
    for (int v = v0; v < v1; v += W) {
        const Raw<T> c = n0;
        n0 = n1;
        n1 = load_raw(r, v + 2 * W + lane);
        f(unpack(r, c, v + lane, v1));
    }
}

template <int NT>
struct Shared {
    static constexpr int NW = NT / W;
    u64 mass[kBins];
    uint32_t cnt[kBins];
    u64 list[kList];
    alignas(16) uint32_t group[256];
    double wd[NW];
    int wi[NW];
    float wf[NW];
    int list_n, bin;
    uint32_t bound;
    double above_mass;
    int above_cnt, bin_cnt;
    double out_d;
    int out_i;
    float out_f;
    u64 out_r;
};

// First entry in index order at which the running sum of the weights exceeds target(total); the last entry with a weight if
// none does.  wf(vector, w) gives the weights of a vector's entries.  Sums in a fixed order: vector, lane, wave segments, then the segment of the border again in 1/NW pieces.
// Every thread returns the index; *total and the entry's z likewise.  `seen` is called once for every vector.
template <int NT, typename T, typename WF, typename TF, typename SF>
__device__ __forceinline__ int locate(const RowView<T>& r, Shared<NT>& sh, WF wf, TF target_of, SF seen, double* total, float* z_out) {
    constexpr int NW = NT / W, N = Vec<T>::N;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int lo = 0, hi = r.nvec;
    double base = 0, target = 0;
#pragma unroll 1
    for (int level = 0; level < 2; level++) {
        const int per = ((hi - lo + NW - 1) / NW + W - 1) / W * W;
        const int v0 = min(hi, lo + wave * per), v1 = min(hi, v0 + per);
        double s = 0;
        wave_pass(r, v0, v1, lane, [&](const Vec<T>& x) {
            double w[N];
            wf(x, w);
#pragma unroll
            for (int i = 0; i < N; i++) s += w[i];
            if (level == 0) seen(x);
        });
        s = wave_sum(s);
        __syncthreads();
        if (lane == 0) sh.wd[wave] = s;
        __syncthreads();
        if (level == 0) {
            double t = 0;
            for (int i = 0; i < NW; i++) t += sh.wd[i];
            *total = t;
            target = target_of(t);
        }
        int pick = -1, last = 0;
        double b = base, at = base, at_last = base;
        for (int i = 0; i < NW; i++) {
            const double t = sh.wd[i];
            if (t > 0) {
                last = i;
                at_last = b;
                if (pick < 0 && b + t > target) {
                    pick = i;
                    at = b;
                }
            }
            b += t;
        }
        if (pick < 0) {
            pick = last;
            at = at_last;
        }
        base = at;
        const int nlo = min(hi, lo + pick * per);
        hi = min(hi, nlo + per);
        lo = nlo;
    }
    // one wave walks the piece in index order
    if (wave == 0) {
        int found = -1, last = -1;
        float fz = 0, lz = 0;
#pragma unroll 1
        for (int v = lo; v < hi && found < 0; v += W) {
            const Vec<T> x = unpack(r, load_raw(r, v + lane), v + lane, hi);
            double w[N], s = 0;
            wf(x, w);
#pragma unroll
            for (int i = 0; i < N; i++) s += w[i];
            const double inc = wave_scan(s), prev = one_lane_up(inc);
            const u64 some = __ballot(s > 0), over = __ballot(s > 0 && base + inc > target);
            if (some) {
                const int who = over ? __ffsll(over) - 1 : 63 - __clzll(some);
                int mi = -1, ml = -1;
                float mz = 0, mlz = 0;
                if (lane == who) {
                    double c = base + prev;
#pragma unroll
                    for (int i = 0; i < N; i++) {
                        c += w[i];
                        if (w[i] > 0) {
                            ml = x.i0 + i;
                            mlz = x.z[i];
                            if (mi < 0 && c > target) {
                                mi = ml;
                                mz = mlz;
                            }
                        }
                    }
                    if (over && mi < 0) {   // the lane's sum and its parts may round differently
                        mi = ml;
                        mz = mlz;
                    }
                }
                last = __shfl(ml, who);
                lz = __shfl(mlz, who);
                if (over) {
                    found = __shfl(mi, who);
                    fz = __shfl(mz, who);
                }
            }
            base += lane_value(inc, 63);
        }
        if (lane == 0) {
            sh.out_i = found < 0 ? last : found;
            sh.out_f = found < 0 ? lz : fz;
        }
    }
    __syncthreads();
    const int res = sh.out_i;
    *z_out = sh.out_f;
    __syncthreads();
    return res;
}

// The first `keep` of ranked[], again in index order, and the draw among them.
template <int NT, int E>
__device__ __forceinline__ void draw_ranked(const SampleOp& op, int row, Shared<NT>& sh, const u64 (&ranked)[E], int keep, const RowParams& rp, const Scale& sc, float zmax, int lane) {
    u64 o[E];
#pragma unroll
    for (int e = 0; e < E; e++) o[e] = e * W + lane < keep ? (ranked[e] << 32) | (ranked[e] >> 32) : 0ull;   // ~index first: descending = index ascending
    wave_sort<E>(o, lane);
    float z[E];
    double w[E];
#pragma unroll
    for (int e = 0; e < E; e++) z[e] = of_key((uint32_t)o[e]);
    weights(z, sc, w);
#pragma unroll
    for (int e = 0; e < E; e++) w[e] = o[e] ? w[e] : 0.0;
    double total;
    const int pos = wave_draw<E>(w, rp.u, &total);
    const u64 d = at_position<E>(o, pos);
    if (lane == 0) {
        write_row(op, row, (int)~(uint32_t)(d >> 32), log_share(of_key((uint32_t)d), zmax, rp.T, total), keep);
        sh.out_d = total;
    }
}
// The list (unordered, n <= 64 E) finished by one wave: prefix, draw, output.  All entries of the row that can be kept are in it.
template <int NT, int E>
__device__ __forceinline__ void finish_list(const SampleOp& op, int row, Shared<NT>& sh, int n, const RowParams& rp, const Scale& sc, float zmax, double mass, int lane) {
    u64 r[E];
#pragma unroll
    for (int e = 0; e < E; e++) r[e] = e * W + lane < n ? sh.list[e * W + lane] : 0ull;
    wave_sort<E>(r, lane);
    const int keep = kept_prefix<E>(r, n, rp, sc, mass, lane);
    const u64 border = at_position<E>(r, keep - 1);
    if (lane == 0) sh.out_r = border;
    if (E > 1 && keep <= W) {
        const u64 first[1] = {r[0]};
        draw_ranked<NT, 1>(op, row, sh, first, keep, rp, sc, zmax, lane);
    } else {
        draw_ranked<NT, E>(op, row, sh, r, keep, rp, sc, zmax, lane);
    }
}
// The border inside a crossing bin whose entries are listed: its rank value.
template <int NT, int E>
__device__ __forceinline__ u64 border_of_list(Shared<NT>& sh, int n, int want, double before, double target, const Scale& sc, int lane) {
    u64 r[E];
#pragma unroll
    for (int e = 0; e < E; e++) r[e] = e * W + lane < n ? sh.list[e * W + lane] : 0ull;
    wave_sort<E>(r, lane);
    int keep = want;
    if (want < 0) {
        double carry = before, w[E];
        float z[E];
        keep = 0;
#pragma unroll
        for (int e = 0; e < E; e++) z[e] = z_of(r[e]);
        weights(z, sc, w);
#pragma unroll
        for (int e = 0; e < E; e++) {
            const bool in = e * W + lane < n;
            const double s = wave_scan(in ? w[e] : 0.0);
            keep += __popcll(__ballot(in && carry + one_lane_up(s) < target));
            carry += lane_value(s, 63);
        }
        keep = max(keep, 1);
    }
    return at_position<E>(r, keep - 1);
}

// log2-spaced bin of an entry, 32 to a factor of two below the maximum, the last one open (entries below 2^-63 of the maximum,
// whose mass is left out); its weight is 2^-bin_power(bin) times
// 2^f, |f| < 0.52, returned beside it
constexpr int kOpen = kBins - 1;
__device__ __forceinline__ int bin_power(int b) { return (b + 16) >> 5; }
__device__ __forceinline__ int bin_of(float z, const Scale& s, double* f) {
    const double y = log2_weight(z, s, -(double)kOpen / 32.0);
    const int b = -low_word(fma(y, 32.0, kRound));
    // kRound + power, its low word being the power
    *f = y + (__longlong_as_double(__double_as_longlong(kRound) + bin_power(b)) - kRound);
    return b;
}
// Smallest key in [lo, hi] that `is` holds for; it holds for hi and, monotone, for every key above one it holds for.  64 keys a
// step, the first ones around `guess`.
template <typename P>
__device__ __forceinline__ uint32_t first_key(uint32_t lo, uint32_t hi, float guess, int lane, P is) {
    uint32_t at = key_of(guess);
    at = max(lo, at < lo + 32 ? lo : at - 32);
    uint32_t step = 1;
#pragma unroll 1
    while (lo < hi) {
        const uint32_t k = at + step * lane;                      // keys above hi count as true
        const bool t = k < at || k >= hi || is(of_key(k));
        const u64 b = __ballot(t);
        if (b & 1) hi = min(hi, at);
        else if (b) {
            const int l = __ffsll(b) - 1;
            lo = at + step * (l - 1) + 1;
            const uint32_t h = at + step * l;
            hi = h < at ? hi : min(hi, h);
        } else lo = at + step * 63 + 1;
        step = (hi - lo) / 64 + 1;
        at = lo;
    }
    return lo;
}

struct Border {       // kept: z > z0 or (z == z0 and index <= i0); z0 > -inf
    float z0;
    int i0;
};
__device__ __forceinline__ bool inside(float z, int i, const Border& b) { return (z > b.z0) | ((z == b.z0) & (i <= b.i0)); }

// p in [0.7, 1.42] as an integer of kFix fraction bits on top of the bits of 128.0 (2^(52 - 45) = 128)
__device__ __forceinline__ u64 fixed_bits(double p) { return (u64)__double_as_longlong(p + 128.0); }
__device__ __forceinline__ double of_fixed(u64 sum, uint32_t n, int exponent) {
    const u64 v = sum - (u64)n * (u64)__double_as_longlong(128.0);
    return ldexp((double)v, exponent - kFix);
}

template <typename T>
struct LowBits {   // bits of a float key below the type's resolution
    static constexpr int N = 0;
};
template <>
struct LowBits<bf16_t> {
    static constexpr int N = 16;
};
template <>
struct LowBits<_Float16> {
    static constexpr int N = 13;
};

template <typename T, int NT>
struct Row {
    static constexpr int NW = NT / W, N = Vec<T>::N;
    Shared<NT>& sh;
    RowView<T> view;
    Scale sc;
    int lane, wave, v0, v1;

    __device__ __forceinline__ void clear_hist(bool with_mass) {
        __syncthreads();
        for (int i = threadIdx.x; i < kBins; i += NT) {
            sh.cnt[i] = 0;
            if (with_mass) sh.mass[i] = 0;
        }
        if (threadIdx.x == 0) sh.bin = -1;
        __syncthreads();
    }
    // entries with zlo <= z <= zhi inside `b` -> sh.list; returns how many there are (the list holds at most kList)
    __device__ __forceinline__ int gather(float zlo, float zhi, const Border& b) {
        __syncthreads();
        if (threadIdx.x == 0) sh.list_n = 0;
        __syncthreads();
        wave_pass(view, v0, v1, lane, [&](const Vec<T>& x) {
#pragma unroll
            for (int i = 0; i < N; i++)
                if (x.z[i] >= zlo && x.z[i] <= zhi && inside(x.z[i], x.i0 + i, b)) {
                    const int p = atomicAdd(&sh.list_n, 1);
                    if (p < kList) sh.list[p] = rank_of(x.z[i], x.i0 + i);
                }
        });
        __syncthreads();
        return sh.list_n;
    }
    // Scans the histogram: picks the last non-empty bin whose predecessors count < want (want >= 0) or hold mass < frac * total
    // (want < 0; *total receives the whole mass when `fresh`); counts and masses start at the given offsets.  A bin's masses
    // are in units of 2^-power (power < 0: of 2^-bin_power(bin)), and zero from bin `open` on.
    __device__ __forceinline__ int pick_bin(int want, double frac, bool fresh, double* total, int cnt0, double mass0, int power, int open, int* above_cnt,
                                            double* above_mass, int* bin_cnt) {
        constexpr int PER = kBins / NT;
        uint32_t c[PER];
        double m[PER];
        int ct = 0;
        double mt = 0;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int b = threadIdx.x * PER + i;
            c[i] = sh.cnt[b];
            m[i] = want < 0 && c[i] && b < open ? of_fixed(sh.mass[b], c[i], -(power < 0 ? bin_power(b) : power)) : 0.0;
            ct += (int)c[i];
            mt += m[i];
        }
        const int ci = wave_scan(ct);
        const double mi = wave_scan(mt);
        if (lane == 63) {
            sh.wi[wave] = ci;
            sh.wd[wave] = mi;
        }
        __syncthreads();
        int cb = cnt0;
        double mb = mass0, all = mass0;
        for (int i = 0; i < NW; i++) {
            if (i < wave) {
                cb += sh.wi[i];
                mb += sh.wd[i];
            }
            all += sh.wd[i];
        }
        if (fresh) *total = all;
        const double target = want < 0 ? frac * *total : 0.0;
        cb += ci - ct;
        mb += one_lane_up(mi);
        int mine = -1, mcb = 0;
        double mmb = 0;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            if (c[i] && (want < 0 ? mb < target : cb < want)) {
                mine = threadIdx.x * PER + i;
                mcb = cb;
                mmb = mb;
            }
            cb += (int)c[i];
            mb += m[i];
        }
        if (mine >= 0) atomicMax(&sh.bin, mine);
        __syncthreads();
        if (mine >= 0 && mine == sh.bin) {
            sh.above_cnt = mcb;
            sh.above_mass = mmb;
            sh.bin_cnt = (int)sh.cnt[mine];
        }
        __syncthreads();
        *above_cnt = sh.above_cnt;
        *above_mass = sh.above_mass;
        *bin_cnt = sh.bin_cnt;
        return sh.bin;
    }

    // The border of the prefix of the entries inside `b0` with `want` entries (want >= 0), or (want < 0) with the entries whose
    // predecessors hold less than frac of the whole mass.  A histogram over log2-spaced bins, then - inside the border's bin -
    // over its range of float keys, until 256 entries or a single value are left.
    // *small: set when everything down to the border's bin is a list of <= 256 entries: sh.list holds it, *mass the whole mass.
    __device__ __forceinline__ Border select(int want, double frac, const Border b0, bool* small, int* list_n, double* mass) {
        const bool wm = want < 0;
        int above = 0, cnt = 0, shift = 0, power = 0;
        double above_mass = 0;
        uint32_t klo = kNoKey + 1, khi = key_of((float)sc.zmax);
        bool open = false;
        *small = false;
#pragma unroll 1
        for (int level = 0;; level++) {
            clear_hist(wm);
            const float zl = of_key(klo), zh = of_key(khi);
            const uint32_t kh = khi;
            if (level == 0) {
                wave_pass(view, v0, v1, lane, [&](const Vec<T>& x) {
                    int b[N];
                    double f[N];
                    bool in[N];
#pragma unroll
                    for (int i = 0; i < N; i++) {
                        b[i] = bin_of(x.z[i], sc, &f[i]);
                        in[i] = inside(x.z[i], x.i0 + i, b0);
                    }
                    if (wm) {
                        double p[N];
                        exp2_fracs(f, p);
#pragma unroll
                        for (int i = 0; i < N; i++)
                            if (in[i]) atomicAdd(&sh.mass[b[i]], fixed_bits(p[i]));   // of the open bin: not used
                    }
#pragma unroll
                    for (int i = 0; i < N; i++)
                        if (in[i]) atomicAdd(&sh.cnt[b[i]], 1u);
                });
            } else {
                wave_pass(view, v0, v1, lane, [&](const Vec<T>& x) {
#pragma unroll
                    for (int i = 0; i < N; i++) {
                        const float z = x.z[i];
                        if (z >= zl && z <= zh && inside(z, x.i0 + i, b0)) {   // few
                            double f;
                            bin_of(z, sc, &f);
                            const int b = (int)((kh - key_of(z + 0.0f)) >> shift);
                            atomicAdd(&sh.cnt[b], 1u);
                            if (wm) atomicAdd(&sh.mass[b], fixed_bits(exp2_frac(f)));
                        }
                    }
                });
            }
            __syncthreads();
            if (level == 0) {
                const int bin = pick_bin(want, frac, true, mass, 0, 0.0, -1, kOpen, &above, &above_mass, &cnt);
                power = bin_power(bin);
                open = bin == kOpen;
                // the bin's range of keys
                const double zb = sc.zmax - (bin - 0.5) / 32.0 / sc.c, za = sc.zmax - (bin + 0.5) / 32.0 / sc.c;
                const Scale s = sc;
                const uint32_t top = khi;
                if (!open) klo = first_key(klo, top, (float)za, lane, [=](float z) { double f; return bin_of(z, s, &f) <= bin; });
                khi = upper_end(first_key(klo, top + 1, (float)zb, lane, [=](float z) { double f; return bin_of(z, s, &f) < bin; }) - 1);
                if (above + cnt <= kList) {
                    *list_n = gather(of_key(klo), INFINITY, b0);
                    *small = true;
                    return b0;
                }
            } else {
                const int a0 = above;
                const double m0 = above_mass;
                const int rb = pick_bin(want, frac, false, mass, a0, m0, power, open ? 0 : kBins, &above, &above_mass, &cnt);
                const uint32_t end = khi - ((uint32_t)rb << shift), width = (1u << shift) - 1;
                klo = end - klo > width ? end - width : klo;
                khi = upper_end(end);   // (a picked bin has entries, so it does not become empty)
            }
            if (cnt <= kList || (khi >> LowBits<T>::N) == (klo >> LowBits<T>::N)) break;
            shift = max(0, 32 - __clz((int)(khi - klo)) - 11);
        }
        const double target = frac * *mass;
        Border b;
        if (cnt <= kList) {
            const int n = gather(of_key(klo), of_key(khi), b0);
            if (wave == 0) {
                const u64 border = border_of_list<NT, kList / W>(sh, n, wm ? -1 : want - above, above_mass, target, sc, lane);
                if (lane == 0) sh.out_r = border;
            }
            __syncthreads();
            b.z0 = z_of(sh.out_r);
            b.i0 = index_of_rank(sh.out_r);
            __syncthreads();
            return b;
        }
        // one value, more than 256 times: so many of them, in index order
        constexpr uint32_t low = (1u << LowBits<T>::N) - 1;
        const float zv = of_key((int)khi < 0 ? khi & ~low : khi | low);
        int ties = cnt;
        if (!wm) ties = want - above;
        else {
            const double w = weight(zv, sc);
            if (w > 0) {
                const double t = ceil((target - above_mass) / w);   // entries whose predecessors hold less than the target
                ties = t < 1 ? 1 : t < cnt ? (int)t : cnt;
                if (ties > 1 && above_mass + (ties - 1) * w >= target) ties--;
                else if (ties < cnt && above_mass + ties * w < target) ties++;
            }
        }
        b.z0 = zv;
        b.i0 = b0.z0 == zv ? b0.i0 : 0x7fffffff;
        if (ties < cnt) {
            double tot;
            float zz;
            const Border bb = b0;
            b.i0 = locate<NT>(view, sh, [=](const Vec<T>& x, double (&w)[N]) {
#pragma unroll
                for (int i = 0; i < N; i++) w[i] = x.z[i] == zv && inside(x.z[i], x.i0 + i, bb) ? 1.0 : 0.0;
            }, [=](double) { return (double)ties - 1.0; },
                              [](const Vec<T>&) {}, &tot, &zz);
        }
        return b;
    }
};

// Smallest float whose weight is at least m: min-p as a border (the weights are monotone in z)
__device__ __forceinline__ float min_p_border(double m, double T, const Scale& sc, int lane) {
    if (!(m > 0)) return -FLT_MAX;
    if (sc.zmax == 0x1p128) return INFINITY;
    const float guess = (float)fmax(sc.zmax + T * log(m), -(double)FLT_MAX);
    return of_key(first_key(kNoKey + 1, key_of((float)sc.zmax), guess, lane, [=](float z) { return weight(z, sc) >= m; }));
}

// The k-th largest (k <= 128) of the 256 partial maxima in sh.group, as a key (at least k entries are not below it), to sh.bound:
// every thread counts, for one of them, how many of a share of the others are not below it.  Begins and ends with a barrier.
template <int NT>
__device__ __forceinline__ void kth_partial(Shared<NT>& sh, int k) {
    constexpr int SHARE = 256 * 256 / NT;
    const int tid = threadIdx.x;
    if (tid < 256) sh.cnt[tid] = 0;
    __syncthreads();
    const uint32_t mine = sh.group[tid & 255];
    const u32x4* others = reinterpret_cast<const u32x4*>(sh.group + (tid >> 8) * SHARE);
    uint32_t n = 0;
#pragma unroll 8
    for (int i = 0; i < SHARE / 4; i++) {
        const u32x4 o = others[i];
#pragma unroll
        for (int e = 0; e < 4; e++) n += o[e] >= mine;
    }
    atomicAdd(&sh.cnt[tid & 255], n);
    __syncthreads();
    if (tid < W) {
        uint32_t t = 0;
#pragma unroll
        for (int e = 0; e < 4; e++)
            if ((int)sh.cnt[e * W + tid] >= k) t = max(t, sh.group[e * W + tid]);
        t = max(t, xor_lane<1>(t, tid));
        t = max(t, xor_lane<2>(t, tid));
        t = max(t, xor_lane<4>(t, tid));
        t = max(t, xor_lane<8>(t, tid));
        t = max(t, xor_lane<16>(t, tid));
        t = max(t, xor_lane<32>(t, tid));
        if (tid == 0) sh.bound = t;
    }
    __syncthreads();
}
// maximum, number of entries and 2^LOG partial maxima (keys, to group[]) of this workgroup's vectors [a, b)
template <typename T, int NT>
__device__ __forceinline__ void partial_maxima(const RowView<T>& view, int a, int b, Shared<NT>& sh, uint32_t* group, int log_groups, float* zmax, int* count) {
    constexpr int NW = NT / W, N = Vec<T>::N;
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int per = ((b - a + NW - 1) / NW + W - 1) / W * W, v0 = min(b, a + wave * per), v1 = min(b, v0 + per);
    float tmax = -INFINITY;
    int tcnt = 0;
    wave_pass(view, v0, v1, lane, [&](const Vec<T>& x) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            tmax = fmaxf(tmax, x.z[i]);
            tcnt += x.z[i] > -INFINITY;
        }
    });
    tmax += 0.0f;
    const float m = wave_max(tmax, lane);
    const int c = wave_sum(tcnt);
    if (lane == 0) {
        sh.wf[wave] = m;
        sh.wi[wave] = c;
    }
    uint32_t g = key_of(tmax);
    const int lanes = NT >> log_groups;   // 1 .. 64 neighbouring threads share a group
    if (lanes > 1) g = max(g, xor_lane<1>(g, lane));
    if (lanes > 2) g = max(g, xor_lane<2>(g, lane));
    if (lanes > 4) g = max(g, xor_lane<4>(g, lane));
    if (lanes > 8) g = max(g, xor_lane<8>(g, lane));
    if (lanes > 16) g = max(g, xor_lane<16>(g, lane));
    if (lanes > 32) g = max(g, xor_lane<32>(g, lane));
    if (tid % lanes == 0) group[tid / lanes] = g;
    __syncthreads();
    *zmax = -INFINITY;
    *count = 0;
    for (int i = 0; i < NW; i++) {
        *zmax = fmaxf(*zmax, sh.wf[i]);
        *count += sh.wi[i];
    }
    __syncthreads();
}

template <typename T, int NT>
__device__ __forceinline__ RowView<T> view_of(const SampleOp& op, int row) {
    RowView<T> v;
    v.src = static_cast<const T*>(op.logits) + row * op.row_stride;
    v.legal = op.legal ? op.legal + row * op.legal_stride : nullptr;
    v.A = op.actions;
    v.nvec = (op.actions + Vec<T>::N - 1) / Vec<T>::N;
    return v;
}
// A row without an entry, or with parameters out of range
template <int NT>
__device__ __forceinline__ void write_none(const SampleOp& op, int row) {
    if (threadIdx.x == 0) write_row(op, row, -1, 0.0, 0);
    if (op.probs)
        for (int i = threadIdx.x; i < op.actions; i += NT) op.probs[row * op.probs_stride + i] = 0.f;
}
template <typename T, int NT>
__device__ __forceinline__ void write_probs(const SampleOp& op, int row, const RowView<T>& view, const Scale& sc, const Border& b, double total) {
    const double share = 1.0 / total;
    for (int i = threadIdx.x; i < op.actions; i += NT) {
        const float z = clean(to_float(view.src[i]), !view.legal || view.legal[i]);
        op.probs[row * op.probs_stride + i] = inside(z, i, b) ? (float)(weight(z, sc) * share) : 0.f;
    }
}
// The row's answer from sh.list, its ln <= 256 candidates (see finish_list for `mass`)
template <typename T, int NT>
__device__ __forceinline__ void answer_from_list(const SampleOp& op, int row, Shared<NT>& sh, const RowView<T>& view, int ln, const RowParams& rp, const Scale& sc, float zmax,
                                                 double mass) {
    const int lane = threadIdx.x & 63;
    if (threadIdx.x < W) {
        if (ln <= W) finish_list<NT, 1>(op, row, sh, ln, rp, sc, zmax, mass, lane);
        else if (ln <= 2 * W) finish_list<NT, 2>(op, row, sh, ln, rp, sc, zmax, mass, lane);
        else finish_list<NT, kList / W>(op, row, sh, ln, rp, sc, zmax, mass, lane);
    }
    __syncthreads();
    if (op.probs) write_probs<T, NT>(op, row, view, sc, Border{z_of(sh.out_r), index_of_rank(sh.out_r)}, sh.out_d);
}
// Short cuts: a lower bound of all that can be kept, from top-k or min-p, that mostly leaves few candidates
__device__ __forceinline__ bool short_cut(const RowParams& rp, int k) { return (k && k <= kFastK) || (rp.m > 0 && rp.p >= 1); }
template <int NT>
__device__ __forceinline__ float short_cut_bound(Shared<NT>& sh, const RowParams& rp, int k, const Scale& sc) {
    if (k && k <= kFastK) {
        kth_partial(sh, k);
        return sh.bound > kNoKey ? of_key(sh.bound) : -FLT_MAX;
    }
    return min_p_border(rp.m, rp.T, sc, threadIdx.x & 63);
}

// A row whose maximum, number of entries and partial maxima are known, by a workgroup.  tried: the short cut left too many.
template <typename T, int NT>
__device__ __forceinline__ void answer_row(const SampleOp& op, int row, Shared<NT>& sh, const RowView<T>& view, RowParams rp, float zmax, int count, bool tried) {
    constexpr int NW = NT / W, N = Vec<T>::N;
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    if (rp.T == 0) {   // the first of the ranking
        rp.T = 1;
        rp.k = 1;
        rp.p = 1;
        rp.m = 0;
    }
    const Scale sc = make_scale(zmax, rp.T);
    const int per = ((view.nvec + NW - 1) / NW + W - 1) / W * W;
    const int v0 = min(view.nvec, wave * per), v1 = min(view.nvec, v0 + per);
    Row<T, NT> R{sh, view, sc, lane, wave, v0, v1};
    rp.k = rp.k > 0 && rp.k < count ? rp.k : 0;
    Border b{-FLT_MAX, 0x7fffffff};
    bool small = false;
    int ln = 0;
    double mass = -1.0;
    if (!tried && short_cut(rp, rp.k)) {
        ln = R.gather(short_cut_bound(sh, rp, rp.k, sc), INFINITY, b);
        small = ln <= kList;
    }
#pragma unroll 1
    for (int step = 0; step < 2; step++) {   // top-k, then top-p within it
        if (small || (step == 0 ? !rp.k : rp.p >= 1)) continue;
        bool s2 = false;
        double mm;
        const Border nb = R.select(step == 0 ? rp.k : -1, rp.p, b, &s2, &ln, &mm);
        small = s2;
        b = nb;
        if (step) mass = mm;
    }
    if (small) {
        if (mass >= 0) rp.k = 0;   // a list from top-p's histogram has been cut by top-k before; its whole mass is `mass`
        answer_from_list<T, NT>(op, row, sh, view, ln, rp, sc, zmax, mass);
        return;
    }
    int kn = 0;
    const float zcut = min_p_border(rp.m, rp.T, sc, lane);
    if (zcut > b.z0) b = Border{zcut, 0x7fffffff};
    const Border bb = b;
    float zp;
    double total;
    const int pick = locate<NT>(view, sh, [=](const Vec<T>& x, double (&w)[N]) {
        weights(x.z, sc, w);
#pragma unroll
        for (int i = 0; i < N; i++) w[i] = inside(x.z[i], x.i0 + i, bb) ? w[i] : 0.0;
    }, [&](double t) { return rp.u * t; }, [&](const Vec<T>& x) {
#pragma unroll
        for (int i = 0; i < N; i++) kn += inside(x.z[i], x.i0 + i, bb);
    }, &total, &zp);
    kn = wave_sum(kn);
    if (lane == 0) sh.wi[wave] = kn;
    __syncthreads();
    if (tid == 0) {
        int n = 0;
        for (int i = 0; i < NW; i++) n += sh.wi[i];
        write_row(op, row, pick, log_share(zp, zmax, rp.T, total), n);
    }
    if (op.probs) write_probs<T, NT>(op, row, view, sc, b, total);
}

template <typename T, int NT>
__global__ __launch_bounds__(NT) void k_sample_block(SampleOp op) {
    __shared__ Shared<NT> sh;
    const int row = blockIdx.x;
    const RowView<T> view = view_of<T, NT>(op, row);
    const RowParams rp = row_params(op, row);
    float zmax;
    int count;
    partial_maxima<T, NT>(view, 0, view.nvec, sh, sh.group, 8, &zmax, &count);
    if (!rp.valid || count == 0) write_none<NT>(op, row);
    else answer_row<T, NT>(op, row, sh, view, rp, zmax, count, false);
}

// ---- few long rows: 2^LOG_SPLITS workgroups per row, in two launches ---------------------------------------------------------
// k_sample_maxima leaves each part's share of the 256 partial maxima; k_sample_split bounds and gathers the part's candidates
// into the row's list, and the last workgroup of a row to arrive finishes it (nothing waits).  Rows the short cut does not serve
// are answered by one of their workgroups.
constexpr int kSlots = 512;      // candidates of a row, shared out evenly over its parts
struct SplitRow {
    u64 slot[kSlots];
    uint32_t group[256];
    float part_max[16];
    int part_cnt[16];
    uint32_t arrived;            // parts, + 2^8 per candidate
};
constexpr int kSplitThreads = 1024;
template <typename T>
__device__ __forceinline__ void part_of(const RowView<T>& v, int part, int log_splits, int* a, int* b) {
    const int per = ((v.nvec + (1 << log_splits) - 1) >> log_splits) + 63 & ~63;
    *a = min(v.nvec, part * per);
    *b = min(v.nvec, *a + per);
}
template <typename T>
__global__ __launch_bounds__(kSplitThreads) void k_sample_maxima(SampleOp op, SplitRow* rows, int log_splits) {
    __shared__ Shared<kSplitThreads> sh;
    const int row = blockIdx.x >> log_splits, part = blockIdx.x & ((1 << log_splits) - 1);
    const RowView<T> view = view_of<T, kSplitThreads>(op, row);
    SplitRow& s = rows[row];
    int a, b, count;
    float zmax;
    part_of(view, part, log_splits, &a, &b);
    partial_maxima<T, kSplitThreads>(view, a, b, sh, s.group + (part << (8 - log_splits)), 8 - log_splits, &zmax, &count);
    if (threadIdx.x == 0) {
        s.part_max[part] = zmax;
        s.part_cnt[part] = count;
        if (part == 0) s.arrived = 0;
    }
}
template <typename T>
__global__ __launch_bounds__(kSplitThreads) void k_sample_split(SampleOp op, SplitRow* rows, int log_splits) {
    constexpr int NT = kSplitThreads, NW = NT / W;
    __shared__ Shared<NT> sh;
    const int row = blockIdx.x >> log_splits, part = blockIdx.x & ((1 << log_splits) - 1), tid = threadIdx.x;
    const int lane = tid & 63, wave = uniform(tid >> 6);
    const RowView<T> view = view_of<T, NT>(op, row);
    SplitRow& s = rows[row];
    // everything that is read first, in one go
    const uint32_t g = s.group[tid & 255];
    const int p16 = lane & ((1 << log_splits) - 1);
    float zmax = s.part_max[p16];
    int count = lane < 1 << log_splits ? s.part_cnt[p16] : 0;
    const RowParams rp = row_params(op, row);
    zmax = wave_max(zmax, lane);
    count = wave_sum(count);
    if (!rp.valid || count == 0) {
        if (part == 0) write_none<NT>(op, row);
        return;
    }
    if (tid < 256) sh.group[tid] = g;
    __syncthreads();
    RowParams q = rp;
    if (q.T == 0) {   // as in answer_row
        q.T = 1;
        q.k = 1;
        q.p = 1;
        q.m = 0;
    }
    q.k = q.k > 0 && q.k < count ? q.k : 0;
    const bool quick = short_cut(q, q.k);
    if (quick) {
        const Scale sc = make_scale(zmax, q.T);
        const float zl = short_cut_bound(sh, q, q.k, sc);
        int a, b;
        part_of(view, part, log_splits, &a, &b);
        const int per = ((b - a + NW - 1) / NW + W - 1) / W * W, v0 = min(b, a + wave * per), v1 = min(b, v0 + per);
        Row<T, NT> R{sh, view, sc, lane, wave, v0, v1};
        const int n = R.gather(zl, INFINITY, Border{-FLT_MAX, 0x7fffffff});
        // The workgroups of a row run on several XCDs, whose L2s do not see one another's writes.  What they exchange is written
        // and read by device-scope atomics, which go past the L2s, and a wait for the writes stands before the count of arrivals:
        // a release fence would write back the whole L2 (measured: 100 us instead of a few).
        const int slots = kSlots >> log_splits;
        if (tid < slots) __hip_atomic_store(&s.slot[part * slots + tid], tid < min(n, kList) ? sh.list[tid] : 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (tid == 0) {
            const uint32_t add = 1u + ((uint32_t)(n <= min(slots, kList) ? n : kSlots + 1) << 8);   // one that did not fit: too many in all
            sh.bound = add + __hip_atomic_fetch_add(&s.arrived, add, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            sh.list_n = 0;
        }
        __syncthreads();
        const uint32_t seen = sh.bound;
        if ((seen & 255u) != 1u << log_splits) return;
        const int ln = (int)(seen >> 8);
        if (ln <= kList) {
            if (tid < kSlots) {
                const u64 r = __hip_atomic_load(&s.slot[tid], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                if (r) sh.list[atomicAdd(&sh.list_n, 1)] = r;
            }
            __syncthreads();
            answer_from_list<T, NT>(op, row, sh, view, ln, q, sc, zmax, -1.0);
            return;
        }
    } else if (part) return;
    answer_row<T, NT>(op, row, sh, view, rp, zmax, count, quick);
}

// 0: a workgroup per row.  Splitting pays while workgroups of one row each leave most of the chip idle, and a row is long enough
// to be worth a second launch: one row of 131072 bf16 entries (top-k 50) 20.8 us whole, 12.2 by 16 workgroups; 64 rows 22.0, by 4 16.4;
// 64 rows of 50000 14.9 and 13.8, of 32768 12.8 and 13.0, of 24000 12.1 and 13.6; one row of 32768 11.3 and 12.6, of 24000 10.4 and 22.9;
// 100 rows of 131072 22.2, by 2 19.4, of 50000 15.4 and 15.5.
inline int log_splits(const SampleOp& op) {
    if (op.rows > 128 || op.actions < (op.rows <= 64 ? 49152 : 98304)) return 0;
    return op.rows <= 16 ? 4 : op.rows <= 32 ? 3 : op.rows <= 64 ? 2 : 1;
}

template <typename T>
hipError_t launch_typed(hipStream_t st, const SampleOp& op, void* workspace) {
    if (op.actions <= 4 * W) {
        const dim3 grid((op.rows + kWaveRows - 1) / kWaveRows), block(W * kWaveRows);
        return launch_kernel(st, grid, block, 0, op.actions <= W ? k_sample_wave<T, 1> : op.actions <= 2 * W ? k_sample_wave<T, 2> : k_sample_wave<T, 4>, op);
    } else if (op.actions <= 8192 || (op.rows > 256 && op.actions <= 64ll * op.rows)) {
        // Several workgroups to a CU hide one another's serial parts; a CU with one row needs all its waves.  256 and 1024 threads, top-p
        // 0.9 of bf16: 64 rows of 8192 10.9 and 13.2 us, 256 of 16384 39.2 and 33.9, 512 of 16384 47.4 and 63.6, 512 of 65536 156 and 148,
        // 1024 of 32768 139 and 171, 2048 of 16384 141 and 246, 256 of 131072 240 and 131
        return launch_kernel(st, dim3(op.rows), dim3(256), 0, k_sample_block<T, 256>, op);
    } else if (const int ls = log_splits(op)) {
        SplitRow* rows = static_cast<SplitRow*>(workspace);
        const dim3 grid(op.rows << ls), block(kSplitThreads);
        if (hipError_t e = launch_kernel(st, grid, block, 0, k_sample_maxima<T>, op, rows, ls)) return e;
        return launch_kernel(st, grid, block, 0, k_sample_split<T>, op, rows, ls);
    }
    return launch_kernel(st, dim3(op.rows), dim3(1024), 0, k_sample_block<T, 1024>, op);
}

}  // namespace

size_t sample_workspace_bytes(const SampleOp& op) { return log_splits(op) ? (size_t)op.rows * sizeof(SplitRow) : 0; }

hipError_t launch_sample(hipStream_t st, const SampleOp& op, void* workspace) {
    switch (op.type) {
        case kFp32: return launch_typed<float>(st, op, workspace);
        case kBf16: return launch_typed<bf16_t>(st, op, workspace);
        default: return launch_typed<_Float16>(st, op, workspace);
    }
}

}  // namespace mz

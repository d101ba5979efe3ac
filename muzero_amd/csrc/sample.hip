// mz_sample_actions: one entry of every row of logits, drawn from a given random number after temperature, top-k, top-p and
// min-p.  A row z[0..A) with its legal mask:
//     x_i = (z_i - max z) / T,  w_i = exp(x_i)                  over the legal, finite entries (a row of none: action -1)
//     ranking: z descending, index ascending on ties; each filter keeps a prefix of it, so all of them keep the shortest:
//       top-k: the first k;  top-p: entries whose predecessors (within the first k) hold less than p of those k's mass;
//       min-p: entries with w_i >= m (max w = 1)
//     draw: the first kept i in INDEX order with sum_{j <= i, kept} w_j > u * S,  S = the kept mass.
// Whether an entry is kept and which is drawn are decided by sums next to a border, so weights and sums are 64-bit: an entry of
// relative weight 1e-7 next to the border of a nucleus must not depend on the order of a sum.  Sums run in a fixed order, or
// (histograms, whose LDS atomics arrive in any order) in exact integers, so a row's answer is a function of the row alone.
//
//   A <= 256   k_sample_wave: a wavefront per row, the row in registers (<= 4 entries a lane); ranking = bitonic sort of
//              (key, index) pairs over the lanes.
//   A >  256   k_sample_block: a workgroup per row, passes over the row (its re-reads hit L2 / the memory-side cache):
//              maximum -> candidates.  With top-k <= 128 the k-th largest of 256 partial maxima bounds the k-th entry from
//              below, so about k entries pass and one wave finishes as above.  A nucleus without top-k needs the mass of the
//              whole row: a histogram of count and mass over log2-spaced bins gives it, and the bin the border falls in;
//              small nuclei are finished by one wave, large ones narrow the border's bin to one (value, index).
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
constexpr int kFix = 45;           // fraction bits of a histogram mass: 2^46 per entry * 2^17 entries < 2^63

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
// The row's scale: x / ln 2 = (z - zmax) * c.
struct Scale {
    double zmax, c;
};
__device__ __forceinline__ Scale make_scale(float zmax, double T) {
    Scale s;
    s.zmax = (double)zmax;
    s.c = fmin(1.4426950408889634 / T, 1e290);   // T = 5e-324: 0 * inf is not wanted
    return s;
}
// (z - zmax) / (T ln 2) in [-2000, 0]; z = zmax = +inf counts as 0
__device__ __forceinline__ double log2_weight(float z, const Scale& s) {
    const double d = (double)z == s.zmax ? 0.0 : (double)z - s.zmax;
    return fmax(d * s.c, -2000.0);
}
__device__ __forceinline__ double weight(float z, const Scale& s) {   // 0 for z = -inf
    const double y = log2_weight(z, s), n = rint(y);
    return ldexp(exp2_frac(y - n), (int)n);
}

// ---- order-preserving keys ---------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t key_of(float z) {
    const uint32_t b = __float_as_uint(z);
    return b ^ ((int)b < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k ^ ((int)k < 0 ? 0x80000000u : 0xffffffffu)); }
constexpr uint32_t kNoKey = 0x007fffffu;   // key of -inf: an entry that takes no part
// ranking as an unsigned 64-bit order: larger z first, then smaller index; 0 = no entry
__device__ __forceinline__ u64 rank_of(float z, int i) { return z > -INFINITY ? ((u64)key_of(z) << 32) | (uint32_t)~i : 0ull; }
__device__ __forceinline__ float z_of_rank(u64 r) { return r ? of_key((uint32_t)(r >> 32)) : -INFINITY; }
__device__ __forceinline__ int index_of_rank(u64 r) { return (int)~(uint32_t)r; }

// ---- wave primitives -----------------------------------------------------------------------------------------------------
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ int wave_sum(int v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}
template <typename V>
__device__ __forceinline__ V wave_scan(V v, int lane) {   // inclusive
#pragma unroll
    for (int o = 1; o < W; o <<= 1) {
        const V t = __shfl_up(v, o);
        v += lane >= o ? t : V(0);
    }
    return v;
}
// descending bitonic sort of 64 E values, position e * 64 + lane
template <int E>
__device__ __forceinline__ void wave_sort(u64 (&r)[E], int lane) {
#pragma unroll
    for (int k = 2; k <= W * E; k <<= 1) {
#pragma unroll
        for (int j = k >> 1; j; j >>= 1) {
            if (j >= W) {
                const int s = j / W;
#pragma unroll
                for (int e = 0; e < E; e++)
                    if (!(e & s)) {
                        const bool desc = ((e * W) & k) == 0;   // k > 64: the bit does not depend on the lane
                        const u64 a = r[e], b = r[e | s];
                        const bool sw = desc ? a < b : a > b;
                        r[e] = sw ? b : a;
                        r[e | s] = sw ? a : b;
                    }
            } else {
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const u64 o = __shfl_xor(r[e], j);
                    const bool desc = ((e * W + lane) & k) == 0, lower = (lane & j) == 0;
                    const bool big = desc == lower;   // this position keeps the larger of the pair
                    r[e] = (r[e] > o) == big ? r[e] : o;
                }
            }
        }
    }
}
template <int E>
__device__ __forceinline__ u64 at_position(const u64 (&r)[E], int p) {
    u64 v = 0;
#pragma unroll
    for (int e = 0; e < E; e++) {
        const u64 t = __shfl(r[e], p & 63);
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

// Entries ranked[] (descending, position e * 64 + lane, `count` of them real): the length of the prefix that the filters keep.
// `mass` < 0: top-p goes by the mass of the first k here; else by `mass`.
template <int E>
__device__ __forceinline__ int kept_prefix(const u64 (&ranked)[E], int count, const RowParams& rp, const Scale& sc, double mass, int lane) {
    int n = rp.k > 0 ? min(rp.k, count) : count;
    if (rp.p < 1 || rp.m > 0) {
        double before[E], carry = 0;
        int nm = 0;
#pragma unroll
        for (int e = 0; e < E; e++) {
            const bool in = e * W + lane < n;
            const double w = in ? weight(z_of_rank(ranked[e]), sc) : 0.0;
            const double s = wave_scan(w, lane);
            const double prev = __shfl_up(s, 1);
            before[e] = carry + (lane ? prev : 0.0);
            carry += __shfl(s, 63);
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
__device__ __forceinline__ int wave_draw(const double (&w)[E], double u, int lane, double* total) {
    double cum[E], carry = 0;
#pragma unroll
    for (int e = 0; e < E; e++) {
        const double s = wave_scan(w[e], lane);
        cum[e] = carry + s;
        carry += __shfl(s, 63);
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
    zmax = wave_max(zmax);
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
    u64 border = 1;   // the last kept entry of the ranking
    if ((rp.k > 0 && rp.k < count) || rp.p < 1) {
        u64 r[E];
#pragma unroll
        for (int e = 0; e < E; e++) r[e] = rank_of(z[e], e * W + lane);
        wave_sort<E>(r, lane);
        n = kept_prefix<E>(r, count, rp, sc, -1.0, lane);
        border = at_position<E>(r, n - 1);
    } else if (rp.m > 0) {
        n = 0;
    }
    double w[E];
#pragma unroll
    for (int e = 0; e < E; e++) {
        w[e] = weight(z[e], sc);
        bool keep = rank_of(z[e], e * W + lane) >= border;
        if (border == 1 && rp.m > 0) {
            keep = keep && w[e] >= rp.m;
            n += __popcll(__ballot(keep));
        }
        if (!keep) w[e] = 0.0;
    }
    double total;
    const int pick = wave_draw<E>(w, rp.u, lane, &total);
    if (op.logprob || lane == 0) {
        float zp = z[0];
#pragma unroll
        for (int e = 0; e < E; e++) {
            const float t = __shfl(z[e], pick & 63);
            zp = (pick >> 6) == e ? t : zp;
        }
        if (lane == 0) {
            const double d = (double)zp == sc.zmax ? 0.0 : (double)zp - sc.zmax;
            write_row(op, row, pick, d / rp.T - log(total), n);
        }
    }
    if (probs) {
#pragma unroll
        for (int e = 0; e < E; e++)
            if (e * W + lane < A) probs[e * W + lane] = (float)(w[e] / total);
    }
}

// ---- a workgroup per row ---------------------------------------------------------------------------------------------------
template <typename T>
struct RowView {
    const T* src;           // entry 0
    const uint8_t* legal;
    int A, shift, nvec;     // vector v = the 16 aligned bytes with the entries [v * VEC - shift, + VEC)
};
template <typename T>
struct Vec {
    static constexpr int N = 16 / sizeof(T);
    float z[N];
};
template <typename T>
__device__ __forceinline__ void unpack(const u32x4 d, float* z) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; i++) z[i] = __uint_as_float(d[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint16_t h = (uint16_t)(d[i >> 1] >> (16 * (i & 1)));
            T t;
            __builtin_memcpy(&t, &h, 2);
            z[i] = to_float(t);
        }
    }
}
// one vector of the row; entries outside the row, masked or without a value are -inf
template <typename T>
__device__ __forceinline__ Vec<T> load_vec(const RowView<T>& r, int v) {
    constexpr int N = Vec<T>::N;
    Vec<T> o;
    const int i0 = v * N - r.shift;
    if (i0 >= 0 && i0 + N <= r.A) {
        unpack<T>(*reinterpret_cast<const u32x4*>(r.src + i0), o.z);
        if (r.legal) {
            uint8_t l[N];
            __builtin_memcpy(l, r.legal + i0, N);
#pragma unroll
            for (int i = 0; i < N; i++) o.z[i] = clean(o.z[i], l[i] != 0);
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) o.z[i] = clean(o.z[i], true);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int j = i0 + i;
            o.z[i] = j >= 0 && j < r.A ? clean(to_float(r.src[j]), !r.legal || r.legal[j]) : -INFINITY;
        }
    }
    return o;
}

template <int NT>
struct Shared {
    static constexpr int NW = NT / W;
    u64 mass[kBins];
    uint32_t cnt[kBins];
    u64 list[kList];
    uint32_t group[256];
    double wd[NW];
    double wd2[NW];
    int wi[NW];
    float wf[NW], wf2[NW];
    int list_n, bin;
    uint32_t bound;
    double above_mass;
    int above_cnt, bin_cnt;
    double out_d[2];
    int out_i[4];
    u64 out_r;
};

// f(vector, first index) over this wave's vectors [v0, v1): lanes take consecutive vectors
template <typename T, typename F>
__device__ __forceinline__ void wave_pass(const RowView<T>& r, int v0, int v1, int lane, F f) {
    constexpr int N = Vec<T>::N;
    int v = v0 + lane;
    for (; v + 3 * W < v1; v += 4 * W) {
        const Vec<T> a = load_vec(r, v), b = load_vec(r, v + W), c = load_vec(r, v + 2 * W), d = load_vec(r, v + 3 * W);
        f(a, v * N - r.shift);
        f(b, (v + W) * N - r.shift);
        f(c, (v + 2 * W) * N - r.shift);
        f(d, (v + 3 * W) * N - r.shift);
    }
    for (; v < v1; v += W) f(load_vec(r, v), v * N - r.shift);
}

// First entry in index order at which the running sum of wf(z, index) exceeds target(total); the last entry with a weight if
// none does.  Sums in a fixed order: vector, lane, wave segments, then the segment of the border again in 1/NW pieces.
// Every thread returns the index; *total and the entry's z likewise.
template <typename T, int NT, typename WF, typename TF>
__device__ int locate(const RowView<T>& r, Shared<NT>& sh, WF wf, TF target_of, double* total, float* z_out) {
    constexpr int NW = NT / W, N = Vec<T>::N;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int lo = 0, hi = r.nvec;
    double base = 0, target = 0;
#pragma unroll 1
    for (int level = 0; level < 2; level++) {
        const int per = ((hi - lo + NW - 1) / NW + W - 1) / W * W;
        const int v0 = min(hi, lo + wave * per), v1 = min(hi, v0 + per);
        double s = 0;
        wave_pass(r, v0, v1, lane, [&](const Vec<T>& x, int i0) {
#pragma unroll
            for (int i = 0; i < N; i++) s += wf(x.z[i], i0 + i);
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
        for (int v = lo; v < hi && found < 0; v += W) {
            Vec<T> x;
            const bool on = v + lane < hi;
            if (on) x = load_vec(r, v + lane);
            const int i0 = (v + lane) * N - r.shift;
            double s = 0;
            if (on)
#pragma unroll
                for (int i = 0; i < N; i++) s += wf(x.z[i], i0 + i);
            const double inc = wave_scan(s, lane);
            const double prev = __shfl_up(inc, 1);
            const u64 some = __ballot(s > 0), over = __ballot(s > 0 && base + inc > target);
            if (some) {
                const int who = over ? __ffsll(over) - 1 : 63 - __clzll(some);
                int mi = -1, ml = -1;
                float mz = 0, mlz = 0;
                if (lane == who) {
                    double c = base + (lane ? prev : 0.0);
#pragma unroll
                    for (int i = 0; i < N; i++) {
                        const double w = wf(x.z[i], i0 + i);
                        c += w;
                        if (w > 0) {
                            ml = i0 + i;
                            mlz = x.z[i];
                            if (mi < 0 && c > target) {
                                mi = i0 + i;
                                mz = x.z[i];
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
            base += __shfl(inc, 63);
        }
        if (lane == 0) {
            sh.out_i[0] = found < 0 ? last : found;
            sh.wf[0] = found < 0 ? lz : fz;
        }
    }
    __syncthreads();
    const int res = sh.out_i[0];
    *z_out = sh.wf[0];
    __syncthreads();
    return res;
}

// Entry `list` (unordered, n <= 256) finished by one wave: prefix, draw, output.  All z of the row that can be kept are in it.
template <int NT, int E>
__device__ void finish_list(const SampleOp& op, int row, Shared<NT>& sh, int n, const RowParams& rp, const Scale& sc, double mass, int lane) {
    u64 r[E];
#pragma unroll
    for (int e = 0; e < E; e++) r[e] = e * W + lane < n ? sh.list[e * W + lane] : 0ull;
    wave_sort<E>(r, lane);
    const int keep = kept_prefix<E>(r, n, rp, sc, mass, lane);
    const u64 border = at_position<E>(r, keep - 1);
    // the kept ones again, in index order
    u64 o[E];
#pragma unroll
    for (int e = 0; e < E; e++) o[e] = e * W + lane < keep ? (r[e] << 32) | (r[e] >> 32) : 0ull;   // ~index first: descending = index ascending
    wave_sort<E>(o, lane);
    double w[E];
    float z[E];
#pragma unroll
    for (int e = 0; e < E; e++) {
        const u64 t = (o[e] << 32) | (o[e] >> 32);
        z[e] = o[e] ? of_key((uint32_t)(t >> 32)) : -INFINITY;
        w[e] = o[e] ? weight(z[e], sc) : 0.0;
    }
    double total;
    const int pos = wave_draw<E>(w, rp.u, lane, &total);
    const u64 d = at_position<E>(o, pos);
    const int pick = (int)~(uint32_t)(d >> 32);
    const float zp = of_key((uint32_t)d);
    if (lane == 0) {
        const double x = (double)zp == sc.zmax ? 0.0 : (double)zp - sc.zmax;
        write_row(op, row, pick, x / rp.T - log(total), keep);
        sh.out_r = border;
        sh.out_d[0] = total;
    }
}
// The border inside a crossing bin whose entries are listed: *border = its rank value, returns how many of the list are kept.
template <int NT, int E>
__device__ int border_of_list(Shared<NT>& sh, int n, int want, double before, double target, const Scale& sc, int lane, u64* border) {
    u64 r[E];
#pragma unroll
    for (int e = 0; e < E; e++) r[e] = e * W + lane < n ? sh.list[e * W + lane] : 0ull;
    wave_sort<E>(r, lane);
    int keep = want;
    if (want < 0) {
        double carry = before;
        keep = 0;
#pragma unroll
        for (int e = 0; e < E; e++) {
            const bool in = e * W + lane < n;
            const double s = wave_scan(in ? weight(z_of_rank(r[e]), sc) : 0.0, lane);
            const double prev = __shfl_up(s, 1);
            keep += __popcll(__ballot(in && carry + (lane ? prev : 0.0) < target));
            carry += __shfl(s, 63);
        }
        keep = max(keep, 1);
    }
    *border = at_position<E>(r, keep - 1);
    return keep;
}

// log2-spaced bin of an entry, 32 to a factor of two below the maximum, the last one open; its weight is 2^(-(bin >> 5)) times
// the value 2^f, f in [-0.5, 0.5], returned beside it
__device__ __forceinline__ int bin_of(float z, const Scale& s, double* f) {
    const double y = fmax(log2_weight(z, s), -63.4375);   // bin 2046 at the deepest
    const int b = z > -INFINITY && log2_weight(z, s) < -63.4375 ? kBins - 1 : (int)((0.5 - y) * 32.0);
    *f = y + (double)(b >> 5);
    return b;
}

struct Border {       // kept: z > z0 or (z == z0 and index <= i0)
    float z0;
    int i0;
};
__device__ __forceinline__ bool inside(float z, int i, const Border& b) { return z > b.z0 || (z == b.z0 && i <= b.i0 && z > -INFINITY); }

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
    const SampleOp& op;
    Shared<NT>& sh;
    RowView<T> view;
    Scale sc;
    int row, lane, wave, v0, v1;

    template <typename F>
    __device__ void pass(F f) { wave_pass(view, v0, v1, lane, f); }

    __device__ void clear_hist(bool with_mass) {
        __syncthreads();
        for (int i = threadIdx.x; i < kBins; i += NT) {
            sh.cnt[i] = 0;
            if (with_mass) sh.mass[i] = 0;
        }
        if (threadIdx.x == 0) sh.bin = -1;
        __syncthreads();
    }
    // entries with z >= zlo, z <= zhi inside `b` -> sh.list; returns how many there are (the list holds at most kList)
    __device__ int gather(float zlo, float zhi, const Border& b) {
        __syncthreads();
        if (threadIdx.x == 0) sh.list_n = 0;
        __syncthreads();
        pass([&](const Vec<T>& x, int i0) {
#pragma unroll
            for (int i = 0; i < N; i++)
                if (x.z[i] >= zlo && x.z[i] <= zhi && inside(x.z[i], i0 + i, b)) {
                    const int p = atomicAdd(&sh.list_n, 1);
                    if (p < kList) sh.list[p] = rank_of(x.z[i], i0 + i);
                }
        });
        __syncthreads();
        return sh.list_n;
    }
    // Scans the histogram: picks the last non-empty bin whose predecessors count < want (want >= 0) or hold mass < frac * total
    // (want < 0; *total_mass receives the total when `fresh`, is the given total otherwise); counts and masses start at the
    // given offsets.  exponent_of(bin) gives the power of two of a bin's masses.
    template <typename EX>
    __device__ int pick_bin(int want, double frac, bool fresh, double* total_mass, int cnt0, double mass0, EX exponent_of, int* above_cnt, double* above_mass,
                            int* bin_cnt) {
        constexpr int PER = kBins / NT;
        uint32_t c[PER];
        double m[PER];
        int ct = 0;
        double mt = 0;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int b = threadIdx.x * PER + i;
            c[i] = sh.cnt[b];
            m[i] = want < 0 && c[i] ? of_fixed(sh.mass[b], c[i], exponent_of(b)) : 0.0;
            ct += (int)c[i];
            mt += m[i];
        }
        const int ci = wave_scan(ct, lane);
        const double mi = wave_scan(mt, lane);
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
        if (fresh) *total_mass = all;
        const double target = want < 0 ? frac * *total_mass : 0.0;
        const double mprev = __shfl_up(mi, 1);
        cb += ci - ct;
        mb += lane ? mprev : 0.0;
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
    __device__ void add(int b, bool with_mass, double f) {
        atomicAdd(&sh.cnt[b], 1u);
        if (with_mass) atomicAdd(&sh.mass[b], fixed_bits(exp2_frac(f)));
    }

    // The border of the prefix of entries inside `b0` with `want` entries (want >= 0), or (want < 0) with the entries whose
    // predecessors hold less than frac of the whole mass.  A histogram over log2-spaced bins, then - inside the border's bin -
    // over its range of float keys, until 256 entries or a single value are left.
    // *small: set when everything down to the border's bin is a list of <= 256 entries: sh.list holds it, *mass the whole mass.
    __device__ Border select(int want, double frac, const Border& b0, bool* small, int* list_n, double* mass) {
        const bool wm = want < 0;
        clear_hist(wm);
        pass([&](const Vec<T>& x, int i0) {
#pragma unroll
            for (int i = 0; i < N; i++)
                if (inside(x.z[i], i0 + i, b0)) {
                    double f;
                    const int b = bin_of(x.z[i], sc, &f);
                    add(b, wm && b < kBins - 1, f);
                }
        });
        // the open bin: count without mass (each entry < 2^-63 of the maximum)
        __syncthreads();
        if (wm && threadIdx.x == 0) sh.mass[kBins - 1] = (u64)sh.cnt[kBins - 1] * (u64)__double_as_longlong(128.0);
        __syncthreads();
        int above, cnt;
        double above_mass;
        int bin = pick_bin(want, frac, true, mass, 0, 0.0, [](int b) { return -(b >> 5); }, &above, &above_mass, &cnt);
        const double target = frac * *mass;
        const int shift_n = bin >> 5;
        const bool open = bin == kBins - 1;
        // the bin's range of keys, by bisection on the (monotone) bin number
        uint32_t klo, khi;
        {
            uint32_t lo = kNoKey + 1, hi = key_of((float)sc.zmax);   // smallest key with bin <= `bin`
            while (lo < hi) {
                const uint32_t mid = lo + (hi - lo) / 2;
                double f;
                if (bin_of(of_key(mid), sc, &f) <= bin) hi = mid;
                else lo = mid + 1;
            }
            klo = lo;
            lo = klo;
            hi = key_of((float)sc.zmax);                             // largest key with bin >= `bin`
            while (lo < hi) {
                const uint32_t mid = hi - (hi - lo) / 2;
                double f;
                if (bin_of(of_key(mid), sc, &f) >= bin) lo = mid;
                else hi = mid - 1;
            }
            khi = lo;
        }
        *small = false;
        if (above + cnt <= kList) {
            *list_n = gather(of_key(klo), INFINITY, b0);
            *small = true;
            return b0;
        }
        while (cnt > kList && (khi >> LowBits<T>::N) != (klo >> LowBits<T>::N)) {
            const uint32_t range = khi - klo;
            const int sh_bits = max(0, 32 - __clz((int)range) - 11);
            clear_hist(wm);
            const float zl = of_key(klo), zh = of_key(khi);
            pass([&](const Vec<T>& x, int i0) {
#pragma unroll
                for (int i = 0; i < N; i++)
                    if (x.z[i] >= zl && x.z[i] <= zh && inside(x.z[i], i0 + i, b0)) {
                        double f;
                        bin_of(x.z[i], sc, &f);
                        add((int)((khi - key_of(x.z[i])) >> sh_bits), wm && !open, f);
                    }
            });
            __syncthreads();
            if (wm && open) {
                for (int i = threadIdx.x; i < kBins; i += NT) sh.mass[i] = (u64)sh.cnt[i] * (u64)__double_as_longlong(128.0);
                __syncthreads();
            }
            const int a0 = above;
            const double m0 = above_mass;
            const int rb = pick_bin(want, frac, false, mass, a0, m0, [=](int) { return -shift_n; }, &above, &above_mass, &cnt);
            khi = khi - ((uint32_t)rb << sh_bits);
            const uint32_t width = (1u << sh_bits) - 1;
            klo = khi - klo > width ? khi - width : klo;
        }
        Border b;
        if (cnt <= kList) {
            const int n = gather(of_key(klo), of_key(khi), b0);
            if (wave == 0) {
                u64 border;
                border_of_list<NT, kList / W>(sh, n, wm ? -1 : want - above, above_mass, target, sc, lane, &border);
                if (lane == 0) sh.out_r = border;
            }
            __syncthreads();
            b.z0 = z_of_rank(sh.out_r);
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
            b.i0 = locate<T, NT>(view, sh, [=](float z, int i) { return z == zv && inside(z, i, bb) ? 1.0 : 0.0; }, [=](double) { return (double)ties - 1.0; }, &tot, &zz);
        }
        return b;
    }
};

// Smallest float whose weight is at least m: min-p as a border (the weights are monotone in z)
__device__ __forceinline__ float min_p_border(double m, double T, const Scale& sc) {
    if (!(m > 0) || sc.zmax == INFINITY) return sc.zmax == INFINITY && m > 0 ? INFINITY : -FLT_MAX;
    uint32_t lo = kNoKey + 1, hi = key_of((float)sc.zmax);
    while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (weight(of_key(mid), sc) >= m) hi = mid;
        else lo = mid + 1;
    }
    return of_key(lo);
}

template <typename T, int NT>
__global__ __launch_bounds__(NT) void k_sample_block(SampleOp op) {
    constexpr int NW = NT / W, N = Vec<T>::N;
    __shared__ Shared<NT> sh;
    const int row = blockIdx.x, tid = threadIdx.x;
    const int lane = tid & 63, wave = tid >> 6;
    const int A = op.actions;
    RowView<T> view;
    view.src = static_cast<const T*>(op.logits) + row * op.row_stride;
    view.legal = op.legal ? op.legal + row * op.legal_stride : nullptr;
    view.A = A;
    view.shift = (int)((reinterpret_cast<uintptr_t>(view.src) & 15) / sizeof(T));
    view.nvec = (A + view.shift + N - 1) / N;
    const int per = ((view.nvec + NW - 1) / NW + W - 1) / W * W;
    const int v0 = min(view.nvec, wave * per), v1 = min(view.nvec, v0 + per);
    const RowParams rp = row_params(op, row);
    float* probs = op.probs ? op.probs + row * op.probs_stride : nullptr;

    float tmax = -INFINITY;
    int tcnt = 0;
    wave_pass(view, v0, v1, lane, [&](const Vec<T>& x, int) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            tmax = fmaxf(tmax, x.z[i]);
            tcnt += x.z[i] > -INFINITY;
        }
    });
    {
        const float m = wave_max(tmax);
        const int c = wave_sum(tcnt);
        if (lane == 0) {
            sh.wf[wave] = m;
            sh.wi[wave] = c;
        }
        // 256 partial maxima
        float g = tmax;
        if (NT == 1024) g = fmaxf(fmaxf(g, __shfl_xor(g, 1)), fmaxf(__shfl_xor(g, 2), __shfl_xor(g, 3)));
        if (tid % (NT / 256) == 0) sh.group[tid / (NT / 256)] = key_of(g);
    }
    __syncthreads();
    float zmax = -INFINITY;
    int count = 0;
    for (int i = 0; i < NW; i++) {
        zmax = fmaxf(zmax, sh.wf[i]);
        count += sh.wi[i];
    }
    __syncthreads();
    if (!rp.valid || count == 0) {
        if (tid == 0) write_row(op, row, -1, 0.0, 0);
        if (probs)
            for (int i = tid; i < A; i += NT) probs[i] = 0.f;
        return;
    }
    double total;
    float zp;
    if (rp.T == 0) {
        const int pick = locate<T, NT>(view, sh, [=](float z, int) { return z == zmax ? 1.0 : 0.0; }, [](double) { return 0.0; }, &total, &zp);
        if (tid == 0) write_row(op, row, pick, 0.0, 1);
        if (probs)
            for (int i = tid; i < A; i += NT) probs[i] = i == pick ? 1.f : 0.f;
        return;
    }
    const Scale sc = make_scale(zmax, rp.T);
    Row<T, NT> R{op, sh, view, sc, row, lane, wave, v0, v1};
    const int k = rp.k > 0 && rp.k < count ? rp.k : 0;
    const float zcut = min_p_border(rp.m, rp.T, sc);
    Border b{-INFINITY, 0x7fffffff};
    bool done = false, small = false;
    int ln = 0;
    double mass = -1.0;
    // short cuts: a lower bound of all that can be kept, from top-k or min-p, that leaves few candidates
    if ((k && k <= kFastK) || (rp.m > 0 && rp.p >= 1)) {
        if (wave == 0) {
            uint32_t t = 0;
            if (k && k <= kFastK) {   // the k-th largest partial maximum: at least k entries are not below it
                uint32_t g[4];
#pragma unroll
                for (int e = 0; e < 4; e++) g[e] = sh.group[e * W + lane];
                for (int bit = 31; bit >= 0; bit--) {
                    const uint32_t c = t | (1u << bit);
                    int n = 0;
#pragma unroll
                    for (int e = 0; e < 4; e++) n += __popcll(__ballot(g[e] >= c));
                    if (n >= k) t = c;
                }
            }
            if (lane == 0) sh.bound = t;
        }
        __syncthreads();
        float zl = sh.bound > kNoKey ? of_key(sh.bound) : -FLT_MAX;
        if (rp.p >= 1) zl = fmaxf(zl, zcut);   // top-p needs the mass of all of the first k
        ln = R.gather(zl, INFINITY, b);
        small = ln <= kList;
    }
    if (!small && k) {
        bool s2 = false;
        double mm;
        b = R.select(k, 0.0, b, &s2, &ln, &mm);
        small = s2;
    }
    if (!small && rp.p < 1) {
        bool s2 = false;
        const Border nb = R.select(-1, rp.p, b, &s2, &ln, &mass);
        if (s2) small = true;
        else b = nb;
    }
    if (small) {
        RowParams q = rp;
        q.k = k;
        // a list from top-p's histogram was cut by top-k before: its border is in it, its mass is `mass`
        if (mass >= 0) q.k = 0;
        if (wave == 0) {
            if (ln <= W) finish_list<NT, 1>(op, row, sh, ln, q, sc, mass, lane);
            else finish_list<NT, kList / W>(op, row, sh, ln, q, sc, mass, lane);
        }
        __syncthreads();
        if (probs) {
            b.z0 = z_of_rank(sh.out_r);
            b.i0 = index_of_rank(sh.out_r);
            total = sh.out_d[0];
        }
        done = true;
    }
    if (!done) {
        int kn = 0;
        const Border bb = b;
        const int pick = locate<T, NT>(
            view, sh, [=](float z, int i) { return z >= zcut && inside(z, i, bb) ? weight(z, sc) : 0.0; }, [&](double t) { return rp.u * t; }, &total, &zp);
        // how many are kept
        R.pass([&](const Vec<T>& x, int i0) {
#pragma unroll
            for (int i = 0; i < N; i++) kn += x.z[i] >= zcut && inside(x.z[i], i0 + i, bb);
        });
        kn = wave_sum(kn);
        if (lane == 0) sh.wi[wave] = kn;
        __syncthreads();
        if (tid == 0) {
            int n = 0;
            for (int i = 0; i < NW; i++) n += sh.wi[i];
            const double x = (double)zp == sc.zmax ? 0.0 : (double)zp - sc.zmax;
            write_row(op, row, pick, x / rp.T - log(total), n);
        }
    }
    if (probs) {
        const Border bb = b;
        R.pass([&](const Vec<T>& x, int i0) {
#pragma unroll
            for (int i = 0; i < N; i++)
                if (i0 + i >= 0 && i0 + i < A) probs[i0 + i] = x.z[i] >= zcut && inside(x.z[i], i0 + i, bb) ? (float)(weight(x.z[i], sc) / total) : 0.f;
        });
    }
}

template <typename T>
hipError_t launch_typed(hipStream_t st, const SampleOp& op) {
    if (op.actions <= 4 * W) {
        const dim3 grid((op.rows + kWaveRows - 1) / kWaveRows), block(W * kWaveRows);
        if (op.actions <= W) k_sample_wave<T, 1><<<grid, block, 0, st>>>(op);
        else if (op.actions <= 2 * W) k_sample_wave<T, 2><<<grid, block, 0, st>>>(op);
        else k_sample_wave<T, 4><<<grid, block, 0, st>>>(op);
    } else if (op.actions <= 8192) {
        k_sample_block<T, 256><<<dim3(op.rows), dim3(256), 0, st>>>(op);
    } else {
        k_sample_block<T, 1024><<<dim3(op.rows), dim3(1024), 0, st>>>(op);
    }
    return hipGetLastError();
}

}  // namespace

size_t sample_workspace_bytes(const SampleOp&) { return 0; }

hipError_t launch_sample(hipStream_t st, const SampleOp& op, void*) {
    switch (op.type) {
        case kFp32: return launch_typed<float>(st, op);
        case kBf16: return launch_typed<bf16_t>(st, op);
        default: return launch_typed<_Float16>(st, op);
    }
}

}  // namespace mz

// mz_adapter_linear: y[m] = x[m] W^T + bias + s_i (x[m] A_i^T) B_i^T with i = index[m], the row's own adapter.
//   k_shrink  t[m] = x[m] A_i^T in fp32, in parts over K, into the workspace.  The rows of a workgroup are ordered by adapter, so
//             that up to 16 rows of one adapter share its A on the matrix cores.
//   k_skinny  up to 48 rows (single tokens), and more where there are few tiles: bound by the bytes of W, which go straight from
//             memory into the matrix instructions' registers, once; the waves of a workgroup split K.  With one or two rows of
//             small rank t is computed by every workgroup for itself (A is read from L2), which saves the launch of k_shrink.
//   k_tile    else: a tiled product, operands staged through LDS; the rows of a tile are ordered by adapter, so that
//             t B_i^T is one more step of the same matrix instructions on the accumulators, per adapter in 16 rows.
// Both end with bias, the adapter's term and one rounding.  The adapter's term is computed apart from the accumulators and added
// where the row uses that adapter: no row sees another row's adapter, whatever values it holds.
#include "net.h"
#include "ops.h"

#include <math.h>

#include <utility>

namespace mz {
namespace {

// f(0), f(1), .. with constant arguments: accumulators indexed by them stay in registers however long f is
template <typename F, int... I>
__device__ __forceinline__ void static_for(F f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
struct bf16_t {
    uint16_t b;
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(bf16_t v) { return __uint_as_float((uint32_t)v.b << 16); }
__device__ __forceinline__ float to_float(_Float16 v) { return (float)v; }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ _Float16 from_float<_Float16>(float v) { return (_Float16)v; }
template <>
__device__ __forceinline__ bf16_t from_float<bf16_t>(float v) {   // to nearest, ties to even
    const __bf16 h = (__bf16)v;
    bf16_t r;
    __builtin_memcpy(&r, &h, 2);
    return r;
}

// One 16-byte chunk of each operand (8 k values of 16 bits, 4 of fp32) of 16 rows x 4 lane groups: acc += A B^T.  Lane l holds
// row l % 16, chunk l / 16 of both; acc[i] of lane l is (A row 4 (l / 16) + i, B row l % 16).
template <typename T>
__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 acc) {
    if constexpr (sizeof(T) == 4) {
        // each step takes element s of every lane: k = 4 (l / 16) + s for both operands
#pragma unroll
        for (int s = 0; s < 4; s++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[s]), __uint_as_float(b[s]), acc, 0, 0, 0);
        return acc;
    } else if constexpr (__is_same(T, bf16_t)) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), acc, 0, 0, 0);
    }
}

// k values [k, k + 16 / sizeof(T)) of a row of K, zero beyond its end; any alignment
template <typename T>
__device__ __forceinline__ u32x4 load_chunk(const T* row, int k, int K) {
    constexpr int N = 16 / sizeof(T);
    u32x4 v = {0, 0, 0, 0};
    if (k + N <= K) __builtin_memcpy(&v, row + k, 16);
    else if (k < K) {
        T t[N] = {};
#pragma unroll
        for (int i = 0; i < N; i++)
            if (k + i < K) t[i] = row[k + i];
        __builtin_memcpy(&v, t, 16);
    }
    return v;
}

// ---- shapes shared by the kernels ------------------------------------------------------------------------------------------
template <typename T>
constexpr int kChunk = 16 / sizeof(T);        // elements of a 16-byte chunk
constexpr int kRankTile = 16;
__host__ __device__ inline int padded_rank(int r) { return (r + kRankTile - 1) / kRankTile * kRankTile; }

template <typename T>
__device__ __forceinline__ u32x4 load16(const T* p) {   // any alignment
    u32x4 v;
    __builtin_memcpy(&v, p, 16);
    return v;
}
constexpr int kNone = -3, kForeign = -2, kNoRow = -1;   // as unsigned numbers: behind every adapter, in this order
__device__ __forceinline__ int adapter_of(const AdapterOp& op, int m) {
    const int i = op.index[m];
    return i >= 0 && i < op.adapters ? i : i == -1 ? kNone : kForeign;
}

// Orders the rows [m0, m0 + count) of a workgroup by adapter (rows of none last): order[p] = row, key[p] = its adapter, kNone or
// kForeign (p >= count: kNoRow), nth[p] = how many rows of that key are in front of it.  A row's place is the number of rows that
// go before it, counted by NTH / BR threads each; rows that stand in order already, as the tokens of one request after the other,
// are left there.  All arrays 16-byte aligned; ends with a barrier.
template <int BR, int NTH, bool NEED_NTH>
__device__ __forceinline__ void order_rows(const AdapterOp& op, int m0, int count, int* raw, int* order, int* key, int* nth) {
    constexpr int SHARE = BR * BR / NTH < 4 ? 4 : BR * BR / NTH;
    static_assert(NTH % BR == 0 && SHARE % 4 == 0, "threads");
    const int tid = threadIdx.x, r = tid % BR, first = tid / BR * SHARE;   // (a share behind the last row: nothing)
    if (tid < BR) {
        raw[tid] = tid < count ? adapter_of(op, m0 + tid) : kNoRow;
        order[tid] = 0;      // (counters until the end)
        nth[tid] = 0;
    }
    __syncthreads();
    const unsigned mine = (unsigned)raw[r];
    if (tid < BR && r + 1 < BR && mine > (unsigned)raw[r + 1]) order[0] = 1;
    __syncthreads();
    const bool sorted = order[0] == 0;
    if (!sorted || NEED_NTH) {
        __syncthreads();
        if (tid == 0) order[0] = 0;
        __syncthreads();
        int less = 0, eq = 0;
#pragma unroll 4
        for (int j = first; j < min(first + SHARE, BR); j += 4) {
            const u32x4 o = *reinterpret_cast<const u32x4*>(raw + j);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                less += o[e] < mine;
                eq += (int)(o[e] == mine) & (int)(j + e < r);
            }
        }
        atomicAdd(&order[r], less + eq);
        if (NEED_NTH) atomicAdd(&nth[r], eq);
        __syncthreads();
        int pos = 0, n = 0;
        if (tid < BR) {
            pos = order[r];
            n = nth[r];
        }
        __syncthreads();
        if (tid < BR) {
            order[pos] = r;
            key[pos] = (int)mine;
            nth[pos] = n;
        }
    } else {
        __syncthreads();
        if (tid < BR) {
            order[r] = r;
            key[r] = (int)mine;
        }
    }
    __syncthreads();
}

// 16-bit chunk with inf and NaN entries, which are rare, set to zero
template <typename T>
__device__ __forceinline__ u32x4 finite_only(u32x4 v) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    constexpr unsigned kExp = __is_same(T, bf16_t) ? 0x7f80u : 0x7c00u;
    u16x2 m = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; i++) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, v[i] & 0x7fff7fffu));
    if (__builtin_expect(m.x >= kExp || m.y >= kExp, 0)) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if ((v[i] & kExp) == kExp) v[i] &= 0xffff0000u;
            if ((v[i] >> 16 & kExp) == kExp) v[i] &= 0x0000ffffu;
        }
    }
    return v;
}

// The bf16 in front of each of 8 floats (truncated: none becomes inf), and what is left.  A float is the sum of three such parts
// exactly.
__device__ __forceinline__ u32x4 take_bf16(float (&v)[8]) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t a = __float_as_uint(v[2 * i]), b = __float_as_uint(v[2 * i + 1]) & 0xffff0000u;
        r[i] = a >> 16 | b;
        v[2 * i] -= __uint_as_float(a & 0xffff0000u);
        v[2 * i + 1] -= __uint_as_float(b);
    }
    return r;
}

// ---- t = x A^T -------------------------------------------------------------------------------------------------------------
// Workgroup (block of BR rows, part of K): jobs of up to 16 rows of one adapter, a wave each.  part[s][row][padded rank].
// 16 rows: a wave for every job there can be, in 4 workgroups; 128 rows: 8 waves, as many as 8 rank tiles leave registers for, in 2
// (2928 rows of 53 adapters, fp32: 15.7 us for the whole call with 2, 19.8 with one, 13.5 with 4; 16384 rows of 32: 29.2, 29.9, 31.2).
template <int BR>
constexpr int kShrinkWaves = BR == 16 ? 4 : 8;
template <int BR>
constexpr int kShrinkParts = BR == 16 ? 4 : 2;   // workgroups that share the jobs of a block
template <typename T, int RT, int BR>
__global__ __launch_bounds__(64 * kShrinkWaves<BR>) void k_shrink(AdapterOp op, float* part, int splits) {
    constexpr int CE = kChunk<T>;
    static_assert(BR <= 128, "starts are counted in two waves");
    __shared__ alignas(16) int raw[BR];
    __shared__ int order[BR], key[BR], nth[BR], job[BR], starts[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lr = lane & 15, kq = lane >> 4;
    const int m0 = blockIdx.x * BR, count = min(BR, op.rows - m0), split = blockIdx.y;
    order_rows<BR, 64 * kShrinkWaves<BR>, true>(op, m0, count, raw, order, key, nth);
    const bool start = tid < BR && key[tid < BR ? tid : 0] >= 0 && nth[tid < BR ? tid : 0] % 16 == 0;
    const unsigned long long sb = __ballot(start);
    if (wave < 2 && lane == 0) starts[wave] = __popcll(sb);
    __syncthreads();
    if (start) job[__builtin_amdgcn_mbcnt_hi((unsigned)(sb >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)sb, 0)) + (wave ? starts[0] : 0)] = tid;
    const int jobs = starts[0] + starts[1];
    __syncthreads();
    const int rp = padded_rank(op.rank);
    const int pairs = (op.K + 8 * CE - 1) / (8 * CE);           // 128-byte steps of k
    const int p0 = (int)((long long)pairs * split / splits), p1 = (int)((long long)pairs * (split + 1) / splits);
    const int pf = min(p1, op.K / (8 * CE));                    // whole ones
    for (int j = wave + kShrinkWaves<BR> * blockIdx.z; j < jobs; j += kShrinkWaves<BR> * kShrinkParts<BR>) {
        const int at = job[j], i = key[at], p = at + lr;
        const bool mine = p < count && key[p] == i;
        const int m = m0 + order[mine ? p : at];
        const T* x = static_cast<const T*>(op.x) + m * op.x_stride + kq * CE;
        const T* a[RT];
#pragma unroll
        for (int q = 0; q < RT; q++)   // ranks beyond the last: a row that is there, its results are dropped
            a[q] = static_cast<const T*>(op.a) + ((long long)i * op.rank + min(q * 16 + lr, op.rank - 1)) * op.K + kq * CE;
        f32x4 acc[RT] = {};
        int k = p0;
        constexpr int U = RT == 1 ? 4 : RT == 2 ? (BR == 16 ? 3 : 4) : RT == 8 && BR == 16 ? 1 : 2;   // what the registers hold
        const auto whole = [&](auto U) __attribute__((always_inline)) {   // that many whole steps
            u32x4 fx[U.value][2], fa[U.value][RT][2];
#pragma unroll
            for (int u = 0; u < U.value; u++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    fx[u][h] = load16(x + (k + u) * 8 * CE + h * 4 * CE);
#pragma unroll
                    for (int q = 0; q < RT; q++) fa[u][q][h] = load16(a[q] + (k + u) * 8 * CE + h * 4 * CE);
                }
            __builtin_amdgcn_sched_barrier(0);   // all loads in flight before the first use
#pragma unroll
            for (int u = 0; u < U.value; u++)
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int q = 0; q < RT; q++) acc[q] = mma<T>(fa[u][q][h], fx[u][h], acc[q]);
            k += U.value;
        };
        while (k + U <= pf) whole(std::integral_constant<int, U>{});
        while (U > 1 && k < pf) whole(std::integral_constant<int, 1>{});
        for (; k < p1; k++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int left = op.K - kq * CE;             // x and a already stand at this lane's first chunk
                const u32x4 fx = load_chunk(x, k * 8 * CE + h * 4 * CE, left);
#pragma unroll
                for (int q = 0; q < RT; q++) acc[q] = mma<T>(load_chunk(a[q], k * 8 * CE + h * 4 * CE, left), fx, acc[q]);
            }
        if (mine) {
            float* dst = part + ((long long)split * op.rows + m) * rp + kq * 4;
#pragma unroll
            for (int q = 0; q < RT; q++) {
                f32x4 v = acc[q];
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (q * 16 + kq * 4 + e >= op.rank) v[e] = 0.f;
                if (q * 16 < rp) *reinterpret_cast<f32x4*>(dst + q * 16) = v;
            }
        }
    }
}
// the parts of four ranks of a row, added in order; up to 8 loads in flight
__device__ __forceinline__ f32x4 sum_parts(const float* part, int splits, long long rows, long long m, int rp, int r) {
    f32x4 v = {};
    const float* p = part + m * rp + r;
    const long long step = rows * rp;
    for (int s = 0; s < splits; s += 8) {
        f32x4 t[8];
#pragma unroll
        for (int i = 0; i < 8; i++) t[i] = *reinterpret_cast<const f32x4*>(p + min(s + i, splits - 1) * step);
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (s + i < splits) v += t[i];
    }
    return v;
}

// four neighbouring results of a row
template <typename T>
__device__ __forceinline__ void store4(const AdapterOp& op, int m, int n, f32x4 v) {
    const long long at = m * op.y_stride + n;
    const bool whole = n + 4 <= op.N;
    if (op.bias) {
        const T* b = static_cast<const T*>(op.bias) + n;
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (n + e < op.N) v[e] += to_float(b[e]);
    }
    if (sizeof(T) == 4 || op.out_type == kFp32) {
        float* y = static_cast<float*>(op.y) + at;
        if (whole) __builtin_memcpy(y, &v, 16);
        else
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (n + e < op.N) y[e] = v[e];
    } else {
        T* y = static_cast<T*>(op.y) + at;
        T h[4];
#pragma unroll
        for (int e = 0; e < 4; e++) h[e] = from_float<T>(v[e]);
        if (whole) __builtin_memcpy(y, h, 4 * sizeof(T));
        else
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (n + e < op.N) y[e] = h[e];
    }
}

// ---- few tiles -----------------------------------------------------------------------------------------------------------
// Workgroup: 16 NT rows of W, 16 MT rows of x; the waves split K by 128-byte steps; partial sums meet in LDS.
// One row, 4096 to 4096 bf16: 13.3 us, 2.5 TB/s; 48 rows, 4096 to 11000 fp16 with 48 adapters of rank 32: 40 us, 3.3 TB/s (a large copy
// moves 5.1): bound by how many loads of W are in flight, which the registers bound.
// FJ > 0: t is computed here, FJ >= rows * rank tiles more tiles of 16 rows (of A).
template <int MT>
constexpr int kSkinnyWaves = MT == 1 ? 16 : 8;
template <int MT, int NT, int FJ>
constexpr size_t skinny_lds() {
    return (size_t)kSkinnyWaves<MT> * (MT * NT + FJ) * 64 * 16;
}
template <typename T>
__device__ __forceinline__ float dot_chunk(const float* t, u32x4 c) {
    T h[kChunk<T>];
    __builtin_memcpy(h, &c, 16);
    float d = 0;
#pragma unroll
    for (int k = 0; k < kChunk<T>; k++) d = fmaf(t[k], to_float(h[k]), d);
    return d;
}
template <typename T, int MT, int NT, int FJ>
__global__ __launch_bounds__(64 * kSkinnyWaves<MT>) void k_skinny(AdapterOp op, const float* part, int splits) {
    constexpr int CE = kChunk<T>, NW = kSkinnyWaves<MT>, TILES = MT * NT, NTH = 64 * NW;
    // the operation of this workgroup's rows
    const int all_rows = op.rows, m0 = blockIdx.y * 16 * MT;
    op.rows = min(16 * MT, all_rows - m0);
    op.x = static_cast<const T*>(op.x) + m0 * op.x_stride;
    op.y = static_cast<char*>(op.y) + m0 * op.y_stride * (op.out_type == kFp32 ? 4 : (int)sizeof(T));
    op.index += m0;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    f32x4* red = reinterpret_cast<f32x4*>(smem);                              // [NW][TILES + FJ][64]
    int* adapter = reinterpret_cast<int*>(smem + skinny_lds<MT, NT, FJ>());   // [16 MT]
    float* tl = reinterpret_cast<float*>(adapter + 16 * MT);                  // [rows][padded rank]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lr = lane & 15, kq = lane >> 4;
    const int n0 = blockIdx.x * 16 * NT, rp = padded_rank(op.rank), rt = rp / 16;
    const T *w[NT], *x[MT], *a[FJ ? FJ : 1];
#pragma unroll
    for (int i = 0; i < NT; i++) w[i] = static_cast<const T*>(op.w) + min(n0 + i * 16 + lr, op.N - 1) * op.w_stride + kq * CE;
#pragma unroll
    for (int i = 0; i < MT; i++) x[i] = static_cast<const T*>(op.x) + min(i * 16 + lr, op.rows - 1) * op.x_stride + kq * CE;
    f32x4 acc[NT][MT] = {}, ta[FJ ? FJ : 1] = {};
    const int pairs = (op.K + 8 * CE - 1) / (8 * CE), pf = op.K / (8 * CE);
    constexpr int U = MT + NT + FJ <= 2 ? 4 : MT + NT + FJ == 3 ? (MT == 1 ? 3 : 4) : MT == 1 && NT + FJ > 4 ? 1 : 2;   // what the registers hold
    int p = wave;
    u32x4 fw[U][NT][2], fx[U][MT][2], fa[U][FJ ? FJ : 1][2];
    const auto k_of = [&](int u, int h) { return (p + u * NW) * 8 * CE + h * 4 * CE; };
    const auto fetch = [&] {
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
#pragma unroll
                for (int i = 0; i < NT; i++) fw[u][i][h] = load16(w[i] + k_of(u, h));
#pragma unroll
                for (int i = 0; i < MT; i++) fx[u][i][h] = load16(x[i] + k_of(u, h));
            }
    };
    const auto more = [&] { return p + (U - 1) * NW < pf; };
    if (more()) fetch();                    // before anything that waits for the rows' adapters
    __builtin_amdgcn_sched_barrier(0);
    if (tid < op.rows) adapter[tid] = adapter_of(op, tid);
#pragma unroll
    for (int j = 0; j < FJ; j++) {
        const int m = min(j / rt, op.rows - 1), i = max(adapter_of(op, m), 0);   // of none: some A, its t is not used
        a[j] = static_cast<const T*>(op.a) + ((long long)i * op.rank + min((j % rt) * 16 + lr, op.rank - 1)) * op.K + kq * CE;
    }
    // t B^T is shared out as items (row, column, chunk of ranks): a thread keeps its column and chunk and walks the rows
    const int chunks = (op.rank + CE - 1) / CE, per = 16 * NT * chunks;
    const int wide = per <= NTH ? NTH / per : 1;   // rows at a time
    const bool items = op.rows * per * 4 <= (int)skinny_lds<MT, NT, FJ>();
    const int im0 = per <= NTH ? tid / per : 0, it0 = per <= NTH ? tid % per : tid;
    const auto b_chunk = [&](int m, int it) {
        const int i = max(adapter_of(op, min(m, op.rows - 1)), 0);
        return load_chunk(static_cast<const T*>(op.b) + ((long long)i * op.N + min(n0 + it / chunks, op.N - 1)) * op.rank, it % chunks * CE, op.rank);
    };
    u32x4 b0 = {0, 0, 0, 0};
    if (items && im0 < wide && it0 < per) b0 = b_chunk(im0, it0);
    if (!FJ) {
        for (int q = tid; q < op.rows * (rp / 4); q += NTH) {
            const int m = q / (rp / 4), r = q % (rp / 4) * 4;
            *reinterpret_cast<f32x4*>(tl + m * rp + r) = sum_parts(part, splits, all_rows, m0 + m, rp, r);
        }
    }
    while (more()) {
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int j = 0; j < FJ; j++) fa[u][j][h] = load16(a[j] + k_of(u, h));
        __builtin_amdgcn_sched_barrier(0);   // all loads in flight before the first use
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
#pragma unroll
                for (int i = 0; i < NT; i++)
#pragma unroll
                    for (int j = 0; j < MT; j++) acc[i][j] = mma<T>(fw[u][i][h], fx[u][j][h], acc[i][j]);
#pragma unroll
                for (int j = 0; j < FJ; j++) ta[j] = mma<T>(fa[u][j][h], fx[u][0][h], ta[j]);
            }
        p += U * NW;
        if (more()) fetch();
    }
    for (; p < pairs; p += NW)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int k = p * 8 * CE + h * 4 * CE, left = op.K - kq * CE;
            u32x4 fx[MT];
#pragma unroll
            for (int j = 0; j < MT; j++) fx[j] = load_chunk(x[j], k, left);
#pragma unroll
            for (int i = 0; i < NT; i++) {
                const u32x4 fw = load_chunk(w[i], k, left);
#pragma unroll
                for (int j = 0; j < MT; j++) acc[i][j] = mma<T>(fw, fx[j], acc[i][j]);
            }
#pragma unroll
            for (int j = 0; j < FJ; j++) ta[j] = mma<T>(load_chunk(a[j], k, left), fx[0], ta[j]);
        }
#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
        for (int j = 0; j < MT; j++) red[(wave * (TILES + FJ) + i * MT + j) * 64 + lane] = acc[i][j];
#pragma unroll
    for (int j = 0; j < FJ; j++) red[(wave * (TILES + FJ) + TILES + j) * 64 + lane] = ta[j];
    __syncthreads();
    if (FJ) {   // column m of job (m, rank tile) holds t[m]
        for (int q = tid; q < op.rows * rp; q += NTH) {
            const int m = q / rp, r = q % rp, j = m * rt + r / 16;
            float v = 0;
#pragma unroll
            for (int s = 0; s < NW; s++) v += red[(s * (TILES + FJ) + TILES + j) * 64 + (r % 16 / 4) * 16 + m][r & 3];
            tl[m * rp + r] = r < op.rank ? v : 0.f;
        }
    }
    // results (row m, columns n ..), four neighbours a thread; the items' sums go where the partial sums were
    constexpr int QN = (TILES * 64 + NTH - 1) / NTH;
    f32x4 v[QN];
#pragma unroll
    for (int k = 0; k < QN; k++) {
        const int q = tid + k * NTH;
        v[k] = f32x4{};
        if (q < TILES * 64)
#pragma unroll
            for (int s = 0; s < NW; s++) v[k] += red[(s * (TILES + FJ) + q / 64) * 64 + q % 64];
    }
    __syncthreads();
    float* ex = reinterpret_cast<float*>(smem);   // [row][column][chunk]
    if (items) {
        constexpr int BATCH = 8;
        for (int it = it0; it < per && im0 < wide; it += per <= NTH ? per : NTH) {
            const int c = it % chunks, n = it / chunks;
            const long long at = (long long)min(n0 + n, op.N - 1) * op.rank;
            for (int m = im0; m < op.rows; m += BATCH * wide) {
                u32x4 b[BATCH];
#pragma unroll
                for (int u = 0; u < BATCH; u++) {
                    const int i = max(adapter[min(m + u * wide, op.rows - 1)], 0);
                    if (u == 0 && m == im0 && it == it0) b[u] = b0;
                    else if (m + u * wide < op.rows) b[u] = load_chunk(static_cast<const T*>(op.b) + (long long)i * op.N * op.rank + at, c * CE, op.rank);
                }
#pragma unroll
                for (int u = 0; u < BATCH; u++)
                    if (m + u * wide < op.rows) ex[(m + u * wide) * per + it] = dot_chunk<T>(tl + (m + u * wide) * rp + c * CE, b[u]);
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < QN; k++) {
        const int q = tid + k * NTH, tile = q / 64, l = q % 64, m = (tile % MT) * 16 + (l & 15), nl = (tile / MT) * 16 + (l >> 4) * 4;
        if (q >= TILES * 64 || m >= op.rows || n0 + nl >= op.N) continue;
        const int i = adapter[m];
        if (i >= 0) {
            const float sc = op.scale ? op.scale[i] : 1.f;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                float d = 0;
                if (items) {
                    for (int c = 0; c < chunks; c++) d += ex[m * per + (nl + e) * chunks + c];
                } else {
                    const T* b = static_cast<const T*>(op.b) + ((long long)i * op.N + min(n0 + nl + e, op.N - 1)) * op.rank;
                    for (int r = 0; r < op.rank; r += CE) d += dot_chunk<T>(tl + m * rp + r, load_chunk(b, r, op.rank));
                }
                v[k][e] = fmaf(sc, d, v[k][e]);
            }
        } else if (i == kForeign) {
            v[k] = f32x4{NAN, NAN, NAN, NAN};
        }
        store4<T>(op, m, n0 + nl, v[k]);
    }
}

// ---- tiles -------------------------------------------------------------------------------------------------------------------
// LDS: a ring of stages, each 64 bytes of k (4 chunks) of BM rows of x and BN rows of W.  Chunk c of row r stands at slot
// c ^ (r >> 1 & 3): the 8 lanes that an LDS read serves at a time then hit 8 different 16-byte columns.
// DMA: rows of both operands are 16-byte aligned: global -> LDS without registers, three stages ahead.  Otherwise through registers.
// With and without it, bf16, whole calls: 8192x4096x4096 273 and 310 us, 2048x2048x2048 43.4 and 52.9, 1000x2048x2000 32.2 and 33.7.
// Bound by LDS reads, barriers and their waits beside the matrix instructions where tiles are large (8192x4096x4096: 293 us in a trace,
// 0.94 PFLOP/s, matrix pipes busy 49 % of the time; the library's bare product 1.33), by what each workgroup brings from L2 where they are
// small (1000x2050x1999: 38.4 us, 268 MB, 7 TB/s).
template <int BM, int BN>
constexpr size_t tile_stage_bytes() {
    return (size_t)(BM + BN) * 64;
}
constexpr int kRing = 4;
template <int BM>
constexpr int kOrderBytes = 4 * BM * (int)sizeof(int);

// Small tiles split K over KS groups of waves, each with a ring of its own: their sums are joined before the adapters' term, of
// which each group takes a part of the columns.
template <int BM>
constexpr int kTileGroups = BM == 64 ? 2 : 1;

template <typename T, int BM, int BN, int WM, int WN, bool DMA>
__global__ __launch_bounds__(64 * WM * WN * kTileGroups<BM>, 2) void k_tile(AdapterOp op, const float* part, int splits) {
    constexpr int KS = kTileGroups<BM>, CE = kChunk<T>, NW = WM * WN, NTH = 64 * NW * KS, MI = BM / WM / 16, NI = BN / WN / 16;
    constexpr int NE = NI / KS;   // tiles of columns per wave after the sums are joined
    constexpr int STAGE = (int)tile_stage_bytes<BM, BN>();
    extern __shared__ __attribute__((aligned(16))) char lds[];   // (all of it dynamic: the opt-in covers 160 KiB of that)
    int *raw = reinterpret_cast<int*>(lds), *order = raw + BM, *key = order + BM, *nth = key + BM;
    char* smem = lds + kOrderBytes<BM>;
    const int tid = threadIdx.x, lane = tid & 63, all = __builtin_amdgcn_readfirstlane(tid >> 6), lr = lane & 15, kq = lane >> 4;
    const int wave = all % NW, group = all / NW;
    // tiles of 8 row blocks x all column blocks in turn, so that what runs at one time shares operands in L2; consecutive
    // workgroups go to the 8 XCDs in turn: each takes a contiguous share
    const int ntm = (op.rows + BM - 1) / BM, ntn = (op.N + BN - 1) / BN, nt = ntm * ntn;
    int tile = blockIdx.x;
    {
        const int per = nt / 8, rem = nt % 8, xcd = tile % 8, at = tile / 8;
        tile = xcd * per + min(xcd, rem) + at;
    }
    constexpr int G = 8;
    const int band = tile / (G * ntn), gm = min(G, ntm - band * G), in = tile - band * G * ntn;
    const int m0 = (band * G + in % gm) * BM, n0 = in / gm * BN;
    const int count = min(BM, op.rows - m0);
    order_rows<BM, NTH, false>(op, m0, count, raw, order, key, nth);

    const T* xb = static_cast<const T*>(op.x) + m0 * op.x_stride;
    const T* wb = static_cast<const T*>(op.w) + n0 * op.w_stride;
    f32x4 acc[NI][MI] = {};
    const int wm = (wave % WM) * (BM / WM), wn = (wave / WM) * (BN / WN);
    // whole stages of k: all, this group's [first, first + mine), and the most that a group has
    const int full = op.K / (4 * CE), first = full * group / KS, mine = full * (group + 1) / KS - first, steps = (full + KS - 1) / KS;
    char* ring = smem + group * kRing * STAGE;
    const auto read = [&](const char* st, u32x4 (&fx)[MI], u32x4 (&fw)[NI]) {
#pragma unroll
        for (int j = 0; j < MI; j++) {
            const int r = wm + j * 16 + lr;
            fx[j] = *reinterpret_cast<const u32x4*>(st + r * 64 + ((kq ^ (r >> 1 & 3)) << 4));
        }
#pragma unroll
        for (int i = 0; i < NI; i++) {
            const int r = wn + i * 16 + lr;
            fw[i] = *reinterpret_cast<const u32x4*>(st + (BM + r) * 64 + ((kq ^ (r >> 1 & 3)) << 4));
        }
    };
    const auto multiply = [&](const u32x4 (&fx)[MI], const u32x4 (&fw)[NI]) {
#pragma unroll
        for (int i = 0; i < NI; i++)
#pragma unroll
            for (int j = 0; j < MI; j++) acc[i][j] = mma<T>(fw[i], fx[j], acc[i][j]);
    };
    const auto compute = [&](const char* st) {
        u32x4 fx[MI], fw[NI];
        read(st, fx, fw);
        multiply(fx, fw);
    };
    constexpr int LX = BM / 16 / NW, LW = BN / 16 / NW;   // 16-row pieces of each operand that a wave brings
    static_assert(LX * NW * 16 == BM && LW * NW * 16 == BN, "pieces");
    // piece i of this wave: lane -> (row of the tile, slot); its source row and k chunk
    const int slot = lane & 3;
    if constexpr (DMA) {
        unsigned ox[LX], ow[LW];
        const unsigned lds0 = (unsigned)(unsigned long long)(__attribute__((address_space(3))) char*)ring;
#pragma unroll
        for (int i = 0; i < LX; i++) {
            const int r = (wave * LX + i) * 16 + (lane >> 2);
            ox[i] = (unsigned)(min(order[r], count - 1) * op.x_stride * sizeof(T)) + ((slot ^ (r >> 1 & 3)) << 4);
        }
#pragma unroll
        for (int i = 0; i < LW; i++) {
            const int r = (wave * LW + i) * 16 + (lane >> 2);
            ow[i] = (unsigned)(min(r, op.N - 1 - n0) * op.w_stride * sizeof(T)) + ((slot ^ (r >> 1 & 3)) << 4);
        }
        const char* gx = reinterpret_cast<const char*>(xb) + first * 64ll;
        const char* gw = reinterpret_cast<const char*>(wb) + first * 64ll;
        // written as one statement each, M0 with it: the compiler's own waits for such loads in flight would drain them at
        // every LDS read
        auto issue = [&](int stage) {
            const unsigned dst = lds0 + (stage % kRing) * STAGE;
#pragma unroll
            for (int i = 0; i < LX; i++)
                asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %0, %2" ::"v"(ox[i]), "s"(dst + (wave * LX + i) * 1024), "s"(gx) : "memory");
#pragma unroll
            for (int i = 0; i < LW; i++)
                asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %0, %2" ::"v"(ow[i]), "s"(dst + BM * 64 + (wave * LW + i) * 1024), "s"(gw) : "memory");
            gx += 64;
            gw += 64;
        };
        constexpr int PER = LX + LW;
        // stage s + 1 has arrived in this wave's share (those behind it may be in flight) and this wave has read stage s; then
        // everyone's
        const auto arrive = [&](int s) {
            if (s + 3 < mine) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * PER) : "memory");
            else if (s + 2 < mine) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(PER) : "memory");
            else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        };
        // While the matrix instructions work on stage s from registers, stage s + 1 is read from LDS and stage s + 4 goes where
        // stage s was.
        u32x4 fx[2][MI], fw[2][NI];
        const auto step = [&](int s, u32x4 (&cx)[MI], u32x4 (&cw)[NI], u32x4 (&nx)[MI], u32x4 (&nw)[NI]) {
            arrive(s);
            if (s + kRing < mine) issue(s + kRing);
            if (s + 1 < mine) read(ring + ((s + 1) % kRing) * STAGE, nx, nw);
            if (KS == 1 || s < mine) multiply(cx, cw);
#pragma unroll
            for (int g = 0; g < MI + NI; g++) {   // an LDS read between every few matrix instructions
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, MI * NI * (sizeof(T) == 4 ? 4 : 1) / (MI + NI), 0);
            }
        };
        if (full > 0) {
#pragma unroll
            for (int s = 0; s < kRing; s++)
                if (s < mine) issue(s);
            // (stage 0 of `arrive(-1)`: the ring holds one stage more than from then on)
            if (mine >= kRing) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(3 * PER) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
            read(ring, fx[0], fw[0]);
            for (int s = 0; s < steps; s += 2) {
                step(s, fx[0], fw[0], fx[1], fw[1]);
                if (s + 1 < steps) step(s + 1, fx[1], fw[1], fx[0], fw[0]);
            }
        }
    }
    {
        // Through registers: all of K without DMA, what is left of a stage with it.  By 4-byte words, 16 lanes to the 64 bytes of a
        // row: a 16-byte load that is not aligned to 16 takes the time of four, and here rows need not be aligned to anything.
        constexpr int RX = BM / NW / 4, RW = BN / NW / 4, E = 4 / (int)sizeof(T);   // rows of each operand per lane; elements of a word
        const int word = lane & 15;
        const T *px[RX], *pw[RW];
        int to[RX], tw[RW];     // where the words go in a stage
#pragma unroll
        for (int i = 0; i < RX; i++) {
            const int r = (wave * RX + i) * 4 + (lane >> 4);
            px[i] = xb + min(order[r], count - 1) * op.x_stride + word * E;
            to[i] = r * 64 + (((word >> 2) ^ (r >> 1 & 3)) << 4) + (word & 3) * 4;
        }
#pragma unroll
        for (int i = 0; i < RW; i++) {
            const int r = (wave * RW + i) * 4 + (lane >> 4);
            pw[i] = wb + min(r, op.N - 1 - n0) * op.w_stride + word * E;
            tw[i] = (BM + r) * 64 + (((word >> 2) ^ (r >> 1 & 3)) << 4) + (word & 3) * 4;
        }
        const auto put = [&](char* st, const uint32_t (&vx)[RX], const uint32_t (&vw)[RW]) {
#pragma unroll
            for (int i = 0; i < RX; i++) *reinterpret_cast<uint32_t*>(st + to[i]) = vx[i];
#pragma unroll
            for (int i = 0; i < RW; i++) *reinterpret_cast<uint32_t*>(st + tw[i]) = vw[i];
        };
        if (!DMA && full > 0) {
            constexpr int D = BM == 64 ? 4 : 2;   // stages on their way; behind the last whole one: that one again
            uint32_t vx[D][RX], vw[D][RW];
            const auto fetch = [&](int s, uint32_t (&vx)[RX], uint32_t (&vw)[RW]) {
                const int k = (first + max(min(s, mine - 1), 0)) * 4 * CE;
#pragma unroll
                for (int i = 0; i < RX; i++) __builtin_memcpy(&vx[i], px[i] + k, 4);
#pragma unroll
                for (int i = 0; i < RW; i++) __builtin_memcpy(&vw[i], pw[i] + k, 4);
                __builtin_amdgcn_sched_barrier(0);   // loads in the order of the stages: the waits count them
            };
#pragma unroll
            for (int d = 0; d < D; d++) fetch(d, vx[d], vw[d]);
            constexpr int G = BM == 64 ? 2 : 1;   // stages to a barrier: small tiles have little to do in one
            for (int s = 0; s < steps; s += D)
#pragma unroll
                for (int d = 0; d < D; d += G) {
                    // (a step behind the last stage only turns the barrier)
#pragma unroll
                    for (int g = 0; g < G; g++) put(ring + (d + g) % (2 * G) * STAGE, vx[d + g], vw[d + g]);
#pragma unroll
                    for (int g = 0; g < G; g++) fetch(s + d + g + D, vx[d + g], vw[d + g]);
                    // the fetches stay in flight over the barrier; LDS: the slots that are written next were read a step ago
                    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
                    for (int g = 0; g < G; g++)
                        if (s + d + g < mine) compute(ring + (d + g) % (2 * G) * STAGE);
                }
        }
        if (full * 4 * CE < op.K) {
            const int k = full * 4 * CE, left = op.K - k - word * E;   // elements of the row from this lane's word on
            uint32_t vx[RX], vw[RW];
            const auto rest = [&](const T* p) {
                uint32_t v = 0;
                if (left >= E) __builtin_memcpy(&v, p + k, 4);
                else if (left > 0) __builtin_memcpy(&v, p + k, sizeof(T));   // half of a word: the low one
                return v;
            };
#pragma unroll
            for (int i = 0; i < RX; i++) vx[i] = rest(px[i]);
#pragma unroll
            for (int i = 0; i < RW; i++) vw[i] = rest(pw[i]);
            __syncthreads();   // the stages before have been read
            if (group == 0) put(ring, vx, vw);
            __syncthreads();
            if (group == 0) compute(ring);
        }
    }
    f32x4 sum[NE][MI];
    if constexpr (KS == 2) {
        static_assert(NTH * NE * MI * 16 <= KS * kRing * STAGE, "exchange");
        f32x4* other = reinterpret_cast<f32x4*>(smem) + tid;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NE; i++)
#pragma unroll
            for (int j = 0; j < MI; j++) other[(i * MI + j) * NTH] = group ? acc[i][j] : acc[NE + i][j];
        __syncthreads();
        other += group ? -(NTH / 2) : NTH / 2;
#pragma unroll
        for (int i = 0; i < NE; i++)
#pragma unroll
            for (int j = 0; j < MI; j++) sum[i][j] = (group ? acc[NE + i][j] : acc[i][j]) + other[(i * MI + j) * NTH];
    } else {
#pragma unroll
        for (int i = 0; i < NE; i++)
#pragma unroll
            for (int j = 0; j < MI; j++) sum[i][j] = acc[i][j];
    }
    const int we = wn + group * NE * 16;   // this wave's first column of the tile from here on

    // ---- the adapters' term: t of this tile's rows, in its order -> LDS
    const int rp = padded_rank(op.rank), ts = rp + 4;
    float* tl = reinterpret_cast<float*>(smem);          // [BM][ts]
    __syncthreads();
    for (int q = tid; q < BM * (rp / 4); q += NTH) {
        const int p = q / (rp / 4), r = q % (rp / 4) * 4;
        f32x4 v = {};
        if (key[p] >= 0) v = sum_parts(part, splits, op.rows, m0 + order[p], rp, r);
        *reinterpret_cast<f32x4*>(tl + p * ts + r) = v;
    }
    __syncthreads();
    // With few rows per adapter (by the numbers of both, not by the data: the two ways round differently, and a row's result must
    // not depend on its neighbours) every lane takes the B of its own row; else the matrix instructions take 16 rows at a time.
    // By rows and by matrix instructions, in mixed order: 2000x1024x1024 bf16 rank 16 (tiles of 64) 8 adapters 24.6 and 26.3 us,
    // 12 24.4 and 27.3, 64 30.0 and 42.6; 4096x512x2304 (of 128) 16 adapters 62.4 and 67.2, 32 66.0 and 90.7.
    const bool per_row = op.rank <= 32 && BM <= 8 * op.adapters;
    const auto add_term = [&](auto J) __attribute__((always_inline)) {
        constexpr int j = J.value;
        const int p = wm + j * 16 + lr, own = key[p];
        // bf16: t as the sum of three bf16 numbers, exactly (from 2^-100 on, so that the third is a normal one).  fp16: t scaled by a power of two to a maximum in [2^14, 2^15), as the sum of two fp16 numbers: within 2^-24 of its value down to
        // 2^-15 of the maximum, where their subnormal step, 2^-24, begins to tell.  Below that a third number, 2^24 times larger, takes what
        // they leave (`wide`), down to 2^-38 of the maximum, where the first is not 0 yet.  Rows whose ranks are still further apart (bf16:
        // below 2^-100), and rows with an inf or a NaN, are summed by themselves.  All of this goes by the row's own t alone.
        bool by_itself = per_row, wide = false;
        float back = 1.f, to = 1.f;
        if (sizeof(T) == 2 && !per_row) {
            float mx = 0, mn = INFINITY;
            for (int r = kq * 4; r < rp; r += 16)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float v = fabsf(tl[p * ts + r + e]);
                    mx = v < INFINITY ? fmaxf(mx, v) : INFINITY;
                    mn = v > 0 ? fminf(mn, v) : mn;
                }
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            mn = fminf(mn, __shfl_xor(mn, 16));
            mn = fminf(mn, __shfl_xor(mn, 32));
            if constexpr (__is_same(T, bf16_t)) {
                by_itself = !(mx < INFINITY) || mn < 0x1p-100f;
            } else {
                if (mx > 0) {
                    by_itself = mx > 0x1p100f || mx < 0x1p-80f || mn < mx * 0x1p-38f;
                    wide = mn < mx * 0x1p-15f;
                    const int em = by_itself ? 0 : ilogbf(mx) - 14;
                    back = ldexpf(1.f, em);
                    to = ldexpf(1.f, -em);
                }
            }
        }
        if (by_itself && own >= 0) {
            const float sc = op.scale ? op.scale[own] : 1.f;
            f32x4 d[NE] = {};
            for (int r = 0; r < op.rank; r += CE) {
                float t[CE];
#pragma unroll
                for (int k = 0; k < CE; k++) t[k] = tl[p * ts + r + k];
#pragma unroll
                for (int ni = 0; ni < NE; ni++) {
                    u32x4 c[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int n = min(n0 + we + ni * 16 + kq * 4 + e, op.N - 1);
                        c[e] = load_chunk(static_cast<const T*>(op.b) + ((long long)own * op.N + n) * op.rank, r, op.rank);
                    }
#pragma unroll
                    for (int e = 0; e < 4; e++) d[ni][e] += dot_chunk<T>(t, c[e]);
                }
            }
#pragma unroll
            for (int ni = 0; ni < NE; ni++)
#pragma unroll
                for (int e = 0; e < 4; e++) sum[ni][j][e] = fmaf(sc, d[ni][e], sum[ni][j][e]);
        }
        // per adapter among the 16 rows
        unsigned long long todo = __ballot(own >= 0 && !by_itself);
        while (todo) {
            const int i = __shfl(own, __ffsll(todo) - 1);
            const bool use = own == i && !by_itself;
            todo &= ~__ballot(use);
            const float sc = op.scale ? op.scale[i] : 1.f;
            const auto product = [&](auto Part) __attribute__((always_inline)) {
                constexpr bool kThird = Part.value == 1;
                f32x4 d[NE] = {};
                for (int r0 = 0; r0 < rp; r0 += 16) {
                    // fp32: 16 ranks as they are.  16 bits: a product of 16 ranks of one part of t, then of the same 16 of another: of the
                    // first and second part (t0), and in bf16, which needs three to hold a float, of the third and nothing (t1).
                    const int rb = r0 + (sizeof(T) == 4 ? kq * 4 : (kq & 1) * 8);
                    const bool other = kq >= 2;
                    u32x4 t0, t1;
                    if constexpr (sizeof(T) == 4) {
                        t0 = *reinterpret_cast<const u32x4*>(tl + p * ts + rb);
                    } else {
                        float v[8];
#pragma unroll
                        for (int e = 0; e < 8; e++) v[e] = tl[p * ts + rb + e] * (__is_same(T, bf16_t) ? 1.f : to);
                        if constexpr (__is_same(T, bf16_t)) {
                            const u32x4 a = take_bf16(v), b = take_bf16(v), c = take_bf16(v);
                            t0 = other ? b : a;
                            t1 = other ? u32x4{0, 0, 0, 0} : c;
                        } else {
                            T h[8];
#pragma unroll
                            for (int e = 0; e < 8; e++) {
                                h[e] = from_float<T>(v[e]);
                                if (kThird || other) {
                                    const float rest = v[e] - to_float(h[e]);
                                    h[e] = from_float<T>(rest);
                                    if (kThird) h[e] = from_float<T>(other ? 0.f : (rest - to_float(h[e])) * 0x1p24f);
                                }
                            }
                            __builtin_memcpy(&t0, h, 16);
                        }
                    }
#pragma unroll
                    for (int ni = 0; ni < NE; ni++) {
                        const int n = min(n0 + we + ni * 16 + lr, op.N - 1);
                        u32x4 v = load_chunk(static_cast<const T*>(op.b) + ((long long)i * op.N + n) * op.rank, rb, op.rank);
                        // an inf of B meets the first part of t alone: the others may be 0 or have the other sign
                        if constexpr (__is_same(T, bf16_t)) {
                            const u32x4 f = finite_only<T>(v);
                            d[ni] = mma<T>(f, t1, d[ni]);
                            v = other ? f : v;
                        } else if constexpr (sizeof(T) == 2) {
                            if (kThird || other) v = finite_only<T>(v);
                        }
                        d[ni] = mma<T>(v, t0, d[ni]);
                    }
                }
                if (use && (!kThird || wide)) {
                    const float unit = kThird ? back * 0x1p-24f : back;
#pragma unroll
                    for (int ni = 0; ni < NE; ni++)
#pragma unroll
                        for (int e = 0; e < 4; e++) sum[ni][j][e] = fmaf(sc, d[ni][e] * unit, sum[ni][j][e]);
                }
            };
            product(std::integral_constant<int, 0>{});
            if constexpr (__is_same(T, _Float16))
                if (__ballot(use && wide)) product(std::integral_constant<int, 1>{});
        }
    };
    static_for(add_term, std::make_integer_sequence<int, MI>{});
    // (stores last: a load behind a store would wait for it)
    const auto store = [&](auto J) __attribute__((always_inline)) {
        constexpr int j = J.value;
        const int p = wm + j * 16 + lr;
        if (p < count) {
            const int m = m0 + order[p], own = key[p];
#pragma unroll
            for (int ni = 0; ni < NE; ni++) {
                const int n = n0 + we + ni * 16 + kq * 4;
                if (n < op.N) store4<T>(op, m, n, own == kForeign ? f32x4{NAN, NAN, NAN, NAN} : sum[ni][j]);
            }
        }
    };
    static_for(store, std::make_integer_sequence<int, MI>{});
}

// ---- launch ------------------------------------------------------------------------------------------------------------------
struct Plan {
    bool skinny, fused;
    int mt, nt;          // skinny: tiles of 16 rows of x / of W
    int tile;            // 256, 128, 64
    int splits, block;   // k_shrink: parts of K, rows per workgroup
};
constexpr int kCus = 256;
// Tiles of 64 x 64 that leave half of the chip idle or more, each of which walks all of K alone: k_skinny's workgroups are smaller and
// share K out over their waves.  Tiles against those, bf16 unless said: 720x939x98 (24 tiles) 33.1 and 22.8 us, 256x1024x1024 (64)
// 15.8 and 13.3, 256x2048x1024 fp32 (64) 50.6 and 31.1, 512x4098x1024 (128) 45.4 and 39.3, 512x1024x1024 (128) 16.8 both,
// 256x4096x2048 (128) 31.3 and 34.3, 256x4096x4096 (256) 33.5 and 60.9.  (At 128 tiles the faster one goes by the shape, which the rule
// does not: up to a tenth lost.)
constexpr int kFewTiles = 128;
// Above it, W is streamed for few rows.  That against tiles, W from memory, bf16, 4096 to 11000: 16 rows 30.8 and 38.2 us, 32 rows 32.8
// and 45.6, 48 rows 37.4 and 45.3, 64 rows 43.0 and 45.3; 4096 to 16384, where the last round of workgroups is not full: 32 rows 49.0
// and 52.8, 48 rows 56.9 and 51.5, 64 rows 64.1 and 52.2.  fp32, 4096 to 11000: 32 rows 69.4 and 92.5, 48 rows 104 and 91.9.  (Between 33
// and 64 rows the faster one also goes by the number of outputs, which the rule does not: up to a tenth lost.)
constexpr int kSkinnyRows16 = 48, kSkinnyRows32 = 32;

Plan make_plan(const AdapterOp& op) {
    Plan p{};
    const int rt = padded_rank(op.rank) / 16;
    const int pairs = (op.K * (op.type == kFp32 ? 4 : 2) + 127) / 128;
    const auto tiles = [&](int m, int n) { return (long long)((op.rows + m - 1) / m) * ((op.N + n - 1) / n); };
    const int few_rows = op.type == kFp32 ? kSkinnyRows32 : kSkinnyRows16;
    p.skinny = op.rows <= few_rows || tiles(64, 64) <= kFewTiles;
    // few rows per adapter, whatever their number: smaller blocks order faster and spread further.  Blocks of 16 and of 128 rows:
    // 100x4096x1024 bf16 21.5 and 27.5 us, 720x939x98 fp16 23.6 and 26.8, 1000x2050x1999 43.9 and 43.1, 1024x1024x2048 25.1 and 22.5
    p.block = op.rows < 1024 ? 16 : 128;
    if (p.skinny && op.rows > few_rows) {
        // what a workgroup brings from L2, times the rounds of workgroups on the chip; among equals the fewest workgroups
        long long least = 0;
        for (int mt = 4; mt >= 1; mt--)
            for (int nt = 3; nt >= 1; nt--) {
                const long long cost = (tiles(16 * mt, 16 * nt) + kCus - 1) / kCus * (mt + nt);
                if (!least || cost < least) {
                    least = cost;
                    p.mt = mt;
                    p.nt = nt;
                }
            }
    } else if (p.skinny) {
        p.mt = (op.rows + 15) / 16;
        // rows of W per workgroup: what leaves the fewest rounds of workgroups on the chip; among equals the most, as every
        // workgroup reads x
        auto rounds = [&](int nt) { return ((op.N + 16 * nt - 1) / (16 * nt) + kCus - 1) / kCus * nt; };
        p.nt = 3;
        for (int nt = 2; nt >= 1; nt--)
            if (rounds(nt) < rounds(p.nt)) p.nt = nt;
        // Every workgroup reads the A of all rows: only while that is little.  Fused and not, one row of rank 16 unless said, bf16:
        // 4096 to 11000 21.7 and 22.7 us, 8192 to 8192 31.1 and 40.5; 2048 to 2048, rank 32 10.3 and 10.5; two rows, 1024 to 1024
        // 7.8 and 9.0, 4096 to 4096 16.5 and 13.6; fp32: 162 to 82 5.5 and 8.6, 4096 to 4096 27.3 and 22.4
        const int es = op.type == kFp32 ? 4 : 2, t_tiles = op.rows * rt;
        p.fused = t_tiles <= 2 && ((long long)t_tiles * op.K * es <= 8192 || (t_tiles == 1 && es == 2));
    } else {
        // The larger tile reads less, the smaller one fills the chip: the largest that still does.  Sides 64, 128, 256, bf16:
        // 4096x4096x4096 320, 207, 170 us; 2048x4096x4096 168, 111, 146; 512x4096x4096 59, 74, 149; 16384x2048x128 63, 73, 127.
        // fp32, whose matrix instructions are slow enough for 128: 16384x512x512 118, 95, 168; 2048x2048x2048 161, 164, 523.
        p.tile = op.type != kFp32 && tiles(256, 256) >= kCus ? 256 : tiles(128, 128) >= kCus ? 128 : 64;
    }
    const int blocks = (op.rows + p.block - 1) / p.block;
    // parts of K: a round of k_shrink's workgroups on the chip (8192x1024x1024 bf16: 4 parts 56.5 us, 2 59.8, 8 59.7; 16384x162x82 fp32:
    // 2 parts 29.2 us, 3 31.6, 1 29.4)
    const int s = (kCus * (p.block == 16 ? 2 : 1) + blocks - 1) / blocks;
    p.splits = s < 1 ? 1 : s > 16 ? 16 : s;
    if (p.splits > (pairs + 1) / 2) p.splits = (pairs + 1) / 2;
    if (p.fused) p.splits = 0;
    return p;
}

template <typename T, int MT, int NT, int FJ>
hipError_t launch_skinny(hipStream_t st, const AdapterOp& op, const float* part, int splits) {
    const size_t lds = skinny_lds<MT, NT, FJ>() + 16 * MT * 4 + (size_t)std::min(op.rows, 16 * MT) * padded_rank(op.rank) * 4;
    lds_optin((const void*)k_skinny<T, MT, NT, FJ>);
    const dim3 grid((op.N + 16 * NT - 1) / (16 * NT), (op.rows + 16 * MT - 1) / (16 * MT));
    return launch_kernel(st, grid, dim3(64 * kSkinnyWaves<MT>), lds, k_skinny<T, MT, NT, FJ>, op, part, splits);
}
template <typename T, int MT, int FJ>
hipError_t launch_skinny(hipStream_t st, const AdapterOp& op, const float* part, int splits, int nt) {
    if (nt == 1) return launch_skinny<T, MT, 1, FJ>(st, op, part, splits);
    if (nt == 2) return launch_skinny<T, MT, 2, FJ>(st, op, part, splits);
    return launch_skinny<T, MT, 3, FJ>(st, op, part, splits);
}
template <typename T, int B, int WM, int WN>
hipError_t launch_tile(hipStream_t st, const AdapterOp& op, const float* part, int splits) {
    const int nt = ((op.rows + B - 1) / B) * ((op.N + B - 1) / B);
    const size_t es = sizeof(T), ring = kTileGroups<B> * kRing * tile_stage_bytes<B, B>(), tl = (size_t)B * (padded_rank(op.rank) + 4) * 4;
    const bool dma = ((uintptr_t)op.x | (uintptr_t)op.w) % 16 == 0 && op.x_stride * es % 16 == 0 && op.w_stride * es % 16 == 0 &&
                     (long long)B * op.x_stride * (long long)es < (1ll << 31) && (long long)B * op.w_stride * (long long)es < (1ll << 31);
    const size_t lds = kOrderBytes<B> + (ring > tl ? ring : tl);
    const auto kernel = dma ? k_tile<T, B, B, WM, WN, true> : k_tile<T, B, B, WM, WN, false>;
    lds_optin((const void*)kernel);
    return launch_kernel(st, dim3(nt), dim3(64 * WM * WN * kTileGroups<B>), lds, kernel, op, part, splits);
}
template <typename T, int BR>
hipError_t launch_shrink(hipStream_t st, const AdapterOp& op, float* part, int splits) {
    constexpr int NTH = 64 * kShrinkWaves<BR>;
    const dim3 grid((op.rows + BR - 1) / BR, splits, kShrinkParts<BR>);
    const int rt = padded_rank(op.rank) / 16;
    return launch_kernel(st, grid, dim3(NTH), 0, rt == 1 ? k_shrink<T, 1, BR> : rt == 2 ? k_shrink<T, 2, BR> : rt <= 4 ? k_shrink<T, 4, BR> : k_shrink<T, 8, BR>, op, part, splits);
}

template <typename T>
hipError_t launch_typed(hipStream_t st, const AdapterOp& op, void* workspace) {
    const Plan p = make_plan(op);
    float* part = static_cast<float*>(workspace);
    if (!p.fused) {
        if (hipError_t e = p.block == 16 ? launch_shrink<T, 16>(st, op, part, p.splits) : launch_shrink<T, 128>(st, op, part, p.splits)) return e;
    }
    hipError_t e = hipErrorInvalidConfiguration;
    if (p.skinny) {
        if (p.fused && op.rows * padded_rank(op.rank) == 16) e = launch_skinny<T, 1, 1>(st, op, part, p.splits, p.nt);
        else if (p.fused) e = launch_skinny<T, 1, 2>(st, op, part, p.splits, p.nt);
        else if (p.mt == 1) e = launch_skinny<T, 1, 0>(st, op, part, p.splits, p.nt);
        else if (p.mt == 2) e = launch_skinny<T, 2, 0>(st, op, part, p.splits, p.nt);
        else if (p.mt == 3) e = launch_skinny<T, 3, 0>(st, op, part, p.splits, p.nt);
        else e = launch_skinny<T, 4, 0>(st, op, part, p.splits, p.nt);
    } else if (sizeof(T) == 2 && p.tile == 256) {
        if constexpr (sizeof(T) == 2) e = launch_tile<T, 256, 4, 2>(st, op, part, p.splits);
    } else if (p.tile == 128) {
        e = launch_tile<T, 128, 2, 2>(st, op, part, p.splits);
    } else {
        e = launch_tile<T, 64, 2, 2>(st, op, part, p.splits);
    }
    if (hipError_t o = take_optin_error()) return o;
    return e;
}

}  // namespace

size_t adapter_workspace_bytes(const AdapterOp& op) {
    if (op.rows == 0) return 0;
    const Plan p = make_plan(op);
    return p.fused ? 0 : (size_t)p.splits * op.rows * padded_rank(op.rank) * sizeof(float);
}

hipError_t launch_adapter(hipStream_t st, const AdapterOp& op, void* workspace) {
    switch (op.type) {
        case kFp32: return launch_typed<float>(st, op, workspace);
        case kBf16: return launch_typed<bf16_t>(st, op, workspace);
        default: return launch_typed<_Float16>(st, op, workspace);
    }
}

}  // namespace mz

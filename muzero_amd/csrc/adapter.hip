// mz_adapter_linear: y[m] = x[m] W^T + bias + s_i (x[m] A_i^T) B_i^T with i = index[m], the row's own adapter.
//   k_shrink   t[m] = s_i x[m] A_i^T, fp32, [rows][rank] in the workspace
//   k_project  the product with W on the matrix cores, then t[m] B_i^T and the bias on its accumulators
#include "ops.h"

#include <math.h>

namespace mz {
namespace {

constexpr int W = 64;

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

// ---- t = s x A^T: a wave per (row, rank) -----------------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void k_shrink(AdapterOp op, float* t) {
    const int lane = threadIdx.x & 63;
    const long long job = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int m = (int)(job / op.rank), j = (int)(job % op.rank);
    if (m >= op.rows) return;
    const int i = op.index[m];
    if (i < 0 || i >= op.adapters) return;
    const T* x = static_cast<const T*>(op.x) + m * op.x_stride;
    const T* a = static_cast<const T*>(op.a) + ((long long)i * op.rank + j) * op.K;
    float s = 0;
    for (int k = lane; k < op.K; k += W) s = fmaf(to_float(x[k]), to_float(a[k]), s);
#pragma unroll
    for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
    if (lane == 0) t[(long long)m * op.rank + j] = op.scale ? op.scale[i] * s : s;
}

// ---- the projection --------------------------------------------------------------------------------------------------------
template <typename T, typename O>
__global__ __launch_bounds__(256) void k_project(AdapterOp op, const float* t) {
    constexpr int BM = 64, BN = 64, CH = 8, N16 = 16 / sizeof(T);   // tile rows of x / of W; 16-byte chunks of k per step
    __shared__ u32x4 sx[BM * CH], sw[BN * CH];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int ntn = (op.N + BN - 1) / BN;
    const int m0 = (int)(blockIdx.x / ntn) * BM, n0 = (int)(blockIdx.x % ntn) * BN;
    const int wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
    f32x4 acc[2][2] = {};   // [n tile][m tile]
    for (int k0 = 0; k0 < op.K; k0 += CH * N16) {
        __syncthreads();
        for (int c = tid; c < BM * CH; c += 256) {
            const int r = c / CH, s = c % CH;
            const int m = min(m0 + r, op.rows - 1);
            sx[r * CH + (s ^ (r & 7))] = load_chunk(static_cast<const T*>(op.x) + m * op.x_stride, k0 + s * N16, op.K);
        }
        for (int c = tid; c < BN * CH; c += 256) {
            const int r = c / CH, s = c % CH;
            const int n = min(n0 + r, op.N - 1);
            sw[r * CH + (s ^ (r & 7))] = load_chunk(static_cast<const T*>(op.w) + n * op.w_stride, k0 + s * N16, op.K);
        }
        __syncthreads();
#pragma unroll
        for (int ks = 0; ks < CH / 4; ks++) {
            const int c = ks * 4 + (lane >> 4);
            u32x4 fw[2], fx[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int rw = wn + i * 16 + (lane & 15), rx = wm + i * 16 + (lane & 15);
                fw[i] = sw[rw * CH + (c ^ (rw & 7))];
                fx[i] = sx[rx * CH + (c ^ (rx & 7))];
            }
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int j = 0; j < 2; j++) acc[i][j] = mma<T>(fw[i], fx[j], acc[i][j]);
        }
    }
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const int m = m0 + wm + j * 16 + (lane & 15);
        if (m >= op.rows) continue;
        const int idx = op.index[m];
        const bool some = idx >= 0 && idx < op.adapters;
        const float* tm = t + (long long)m * op.rank;
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int n = n0 + wn + i * 16 + (lane >> 4) * 4 + e;
                if (n >= op.N) continue;
                float v = acc[i][j][e];
                if (some) {
                    const T* b = static_cast<const T*>(op.b) + ((long long)idx * op.N + n) * op.rank;
                    float s = 0;
                    for (int q = 0; q < op.rank; q++) s = fmaf(tm[q], to_float(b[q]), s);
                    v += s;
                } else if (idx != -1) {
                    v = NAN;
                }
                if (op.bias) v += to_float(static_cast<const T*>(op.bias)[n]);
                static_cast<O*>(op.y)[m * op.y_stride + n] = from_float<O>(v);
            }
    }
}

template <typename T, typename O>
hipError_t launch_typed(hipStream_t st, const AdapterOp& op, void* workspace) {
    float* t = static_cast<float*>(workspace);
    k_shrink<T><<<dim3((unsigned)(((long long)op.rows * op.rank + 3) / 4)), dim3(256), 0, st>>>(op, t);
    if (hipError_t e = hipGetLastError()) return e;
    const unsigned nt = (unsigned)((op.rows + 63) / 64) * ((op.N + 63) / 64);
    k_project<T, O><<<dim3(nt), dim3(256), 0, st>>>(op, t);
    return hipGetLastError();
}

}  // namespace

size_t adapter_workspace_bytes(const AdapterOp& op) { return (size_t)op.rows * op.rank * sizeof(float); }

hipError_t launch_adapter(hipStream_t st, const AdapterOp& op, void* workspace) {
    const bool f = op.out_type == kFp32;
    switch (op.type) {
        case kFp32: return launch_typed<float, float>(st, op, workspace);
        case kBf16: return f ? launch_typed<bf16_t, float>(st, op, workspace) : launch_typed<bf16_t, bf16_t>(st, op, workspace);
        default: return f ? launch_typed<_Float16, float>(st, op, workspace) : launch_typed<_Float16, _Float16>(st, op, workspace);
    }
}

}  // namespace mz

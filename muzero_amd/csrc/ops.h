// Stand-alone operators behind the C ABI (include/muzero_hip.h: mz_sample_actions, mz_adapter_linear): launch descriptions and
// launchers.  Arguments have been checked by ops_api.cpp; every pointer is memory of the current device.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <string>
#include <tuple>

namespace mz {

int op_fail(const std::string& msg);   // text for mz_last_error(NULL); returns -1

// Queues a kernel; the status is this launch's own.  (hipGetLastError after <<<>>> also gives what an earlier call of the thread, of
// whatever library, has left behind.)
template <typename... P, typename... A>
hipError_t launch_kernel(hipStream_t st, dim3 grid, dim3 block, size_t lds, void (*kernel)(P...), A... a) {
    std::tuple<P...> held(a...);
    return std::apply(
        [&](P&... p) {
            void* args[] = {&p...};
            return hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, block, args, lds, st);
        },
        held);
}

enum OpType { kFp32 = 0, kBf16 = 1, kF16 = 2 };   // MZ_DTYPE_*

struct SampleOp {
    int rows, actions, type;
    const void* logits;
    long long row_stride;          // elements
    const uint8_t* legal;          // nullptr: every action is legal
    long long legal_stride;
    const double* u;               // [rows]
    double temperature, top_p, min_p;
    int top_k;
    const double* row_temperature; // [rows] each, or nullptr: the scalar
    const int* row_top_k;
    const double* row_top_p;
    const double* row_min_p;
    int* action;                   // [rows]
    float* logprob;                // [rows] or nullptr
    int* kept;                     // [rows] or nullptr
    float* probs;                  // or nullptr
    long long probs_stride;
};
size_t sample_workspace_bytes(const SampleOp& op);
hipError_t launch_sample(hipStream_t st, const SampleOp& op, void* workspace);

struct AdapterOp {
    int rows, K, N, rank, adapters, type, out_type;
    const void* x;
    long long x_stride;
    const void* w;
    long long w_stride;
    const void* bias;
    const void* a;       // [adapters][rank][K]
    const void* b;       // [adapters][N][rank]
    const float* scale;
    const int* index;
    void* y;
    long long y_stride;
};
size_t adapter_workspace_bytes(const AdapterOp& op);
hipError_t launch_adapter(hipStream_t st, const AdapterOp& op, void* workspace);

}  // namespace mz

// C entries of the operators on device tensors (include/muzero_hip.h): every check of the arguments, then the launchers of ops.h.
#include <cmath>
#include <cstdint>
#include <string>

#include "../../include/muzero_hip.h"
#include "ops.h"

using namespace mz;

namespace {

constexpr int kMaxRank = 128;
constexpr int kMaxSampleRows = 1 << 21;     // a workgroup of up to 1024 threads each: below 2^32 threads
constexpr int kMaxSampleActions = 262144;   // 2^18: sample.hip's histogram masses are sums of 2^46 in 64 bits

// The device all operands live on: the first pointer names it, every other one must agree.  What a call writes must not overlap
// anything else of it.
struct Operands {
    int device = -1;
    const char* bad = nullptr;
    std::string why;
    struct Block {   // rows of `width` bytes, `pitch` bytes apart (0: one row)
        const char* name;
        uintptr_t at;
        unsigned __int128 end;
        uintptr_t pitch, width;
        bool written;
    } block[16];
    int blocks = 0;
    void in(const void* p, const char* name, size_t elem, size_t rows, size_t stride, size_t width) { add(p, name, elem, rows, stride * elem, width * elem, false); }
    void out(const void* p, const char* name, size_t elem, size_t rows, size_t stride, size_t width) { add(p, name, elem, rows, stride * elem, width * elem, true); }
    void add(const void* p, const char* name, size_t align, size_t rows, size_t pitch, size_t width, bool written) {
        if (bad || !p) return;
        const uintptr_t at0 = reinterpret_cast<uintptr_t>(p);
        const Block b{name, at0, (unsigned __int128)(rows - 1) * pitch + width + at0, rows > 1 ? pitch : 0, width, written};
        for (int i = 0; i < blocks; i++)
            if ((written || block[i].written) && overlap(block[i], b)) return fail(name, (std::string("overlaps ") + block[i].name).c_str());
        block[blocks++] = b;
        hipPointerAttribute_t at;
        if (hipPointerGetAttributes(&at, p) != hipSuccess) {
            (void)hipGetLastError();
            fail(name, "is not device memory");
        } else if (at.type != hipMemoryTypeDevice && at.type != hipMemoryTypeManaged) {
            fail(name, "is not device memory");
        } else if (reinterpret_cast<uintptr_t>(p) % align) {
            fail(name, "is not aligned to its type");
        } else if (at.type == hipMemoryTypeDevice) {
            if (device < 0) device = at.device;
            else if (device != at.device) fail(name, "is memory of another device");
        }
    }
    static bool overlap(const Block& a, const Block& b) {
        if (a.end <= b.at || b.end <= a.at) return false;
        const uintptr_t pitch = a.pitch ? a.pitch : b.pitch;   // one row may stand in any wide row
        if (pitch == 0 || (a.pitch && b.pitch && a.pitch != b.pitch)) return true;
        const uintptr_t d = (b.at % pitch + pitch - a.at % pitch) % pitch;   // columns of the same wide rows
        return !(d >= a.width && d + b.width <= pitch);
    }
    void fail(const char* name, const char* what) {
        bad = name;
        why = std::string(name) + " " + what;
    }
};

struct DeviceGuard {   // runs on `device`, leaves the caller's device as it was
    int before = -1;
    hipError_t err;
    explicit DeviceGuard(int device) {
        err = hipGetDevice(&before);
        if (err == hipSuccess && before != device) err = hipSetDevice(device);
        else if (err == hipSuccess) before = -1;
    }
    ~DeviceGuard() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

size_t type_bytes(int t) { return t == MZ_DTYPE_FP32 ? 4 : 2; }
bool known_type(int t) { return t == MZ_DTYPE_FP32 || t == MZ_DTYPE_BF16 || t == MZ_DTYPE_F16; }

// Common end of a call: device and stream, workspace, launch.
template <typename F>
int run_op(Operands& o, void* workspace, size_t have, size_t need, void* stream, F launch) {
    if (need) {
        if (!workspace || have < need)
            return op_fail("workspace has " + std::to_string(workspace ? have : 0) + " bytes, needs " + std::to_string(need));
        o.add(workspace, "workspace", 256, 1, need, need, true);
    }
    if (o.bad) return op_fail(o.why);
    int dev = o.device;
    if (dev < 0 && hipGetDevice(&dev) != hipSuccess) return op_fail("no HIP device");   // all operands are managed memory
    DeviceGuard g(dev);
    if (g.err != hipSuccess) return op_fail(std::string("hipSetDevice: ") + hipGetErrorString(g.err));
    if (stream) {
        int sd = -1;
        if (hipStreamGetDevice(static_cast<hipStream_t>(stream), &sd) != hipSuccess) {
            (void)hipGetLastError();
            return op_fail("stream is not a stream");
        }
        if (sd != dev) return op_fail("stream is a stream of another device");
    }
    const hipError_t e = launch(static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return op_fail(std::string("launch: ") + hipGetErrorString(e));
    return 0;
}

const char* check_sample(const mz_sample_args* a) {
    if (!a) return "args is NULL";
    if (a->rows < 0 || a->rows > kMaxSampleRows) return "rows must be 0 .. 2097152";
    if (a->actions < 1 || a->actions > kMaxSampleActions) return "actions must be 1 .. 262144";
    if (!known_type(a->dtype)) return "unknown dtype";
    if (!a->row_temperature && !(a->temperature >= 0 && std::isfinite(a->temperature))) return "temperature must be finite and >= 0";
    if (!a->row_top_k && a->top_k < 0) return "top_k must be >= 0";
    if (!a->row_top_p && !(a->top_p > 0 && a->top_p <= 1)) return "top_p must be in (0, 1]";
    if (!a->row_min_p && !(a->min_p >= 0 && a->min_p <= 1)) return "min_p must be in [0, 1]";
    if (a->row_stride < 0 || (a->legal && a->legal_stride < 0)) return "strides must be >= 0";
    if (a->probs && a->rows > 1 && a->probs_stride < a->actions) return "probs_stride < actions";
    if (a->rows > 0 && (!a->logits || !a->u || !a->action)) return "logits, u and action must not be NULL";
    return nullptr;
}
SampleOp sample_op(const mz_sample_args& a) {
    SampleOp o{};
    o.rows = a.rows;
    o.actions = a.actions;
    o.type = a.dtype;
    o.logits = a.logits;
    o.row_stride = a.row_stride;
    o.legal = a.legal;
    o.legal_stride = a.legal_stride;
    o.u = a.u;
    o.temperature = a.temperature;
    o.top_p = a.top_p;
    o.min_p = a.min_p;
    o.top_k = a.top_k;
    o.row_temperature = a.row_temperature;
    o.row_top_k = a.row_top_k;
    o.row_top_p = a.row_top_p;
    o.row_min_p = a.row_min_p;
    o.action = a.action;
    o.logprob = a.logprob;
    o.kept = a.kept;
    o.probs = a.probs;
    o.probs_stride = a.probs_stride;
    return o;
}

const char* check_adapter(const mz_adapter_args* a) {
    if (!a) return "args is NULL";
    if (a->rows < 0) return "rows < 0";
    if (a->in_features < 1 || a->out_features < 1) return "in_features and out_features must be >= 1";
    if (a->in_features > (1 << 26)) return "in_features must be at most 67108864";   // its bytes fit an int
    if (((long long)a->rows + 255) / 256 * (((long long)a->out_features + 255) / 256) > (1 << 21) || a->out_features > (1 << 26)) return "too many outputs for one call";
    if (a->rank < 1 || a->rank > kMaxRank) return "rank must be 1 .. 128";
    if (a->adapters < 1) return "adapters must be >= 1";
    if (!known_type(a->dtype)) return "unknown dtype";
    if (a->out_dtype != a->dtype && a->out_dtype != MZ_DTYPE_FP32) return "out_dtype must be dtype or fp32";
    if (a->x_stride < 0) return "x_stride must be >= 0";
    if (a->weight_stride < a->in_features) return "weight_stride < in_features";
    if (a->rows > 1 && a->y_stride < a->out_features) return "y_stride < out_features";
    if (a->rows > 0 && (!a->x || !a->weight || !a->a || !a->b || !a->index || !a->y)) return "x, weight, a, b, index and y must not be NULL";
    return nullptr;
}
AdapterOp adapter_op(const mz_adapter_args& a) {
    AdapterOp o{};
    o.rows = a.rows;
    o.K = a.in_features;
    o.N = a.out_features;
    o.rank = a.rank;
    o.adapters = a.adapters;
    o.type = a.dtype;
    o.out_type = a.out_dtype;
    o.x = a.x;
    o.x_stride = a.x_stride;
    o.w = a.weight;
    o.w_stride = a.weight_stride;
    o.bias = a.bias;
    o.a = a.a;
    o.b = a.b;
    o.scale = a.scale;
    o.index = a.index;
    o.y = a.y;
    o.y_stride = a.y_stride;
    return o;
}

// no exception (std::string may throw) crosses the C boundary
template <typename F>
int guarded(F f) {
    try {
        return f();
    } catch (...) {
        return -1;
    }
}

}  // namespace

extern "C" {

size_t mz_sample_workspace_bytes(const mz_sample_args* args) { return check_sample(args) ? 0 : sample_workspace_bytes(sample_op(*args)); }

int mz_sample_actions(const mz_sample_args* args, void* workspace, size_t workspace_bytes, void* stream) {
    return guarded([&] {
        if (const char* e = check_sample(args)) return op_fail(std::string("mz_sample_actions: ") + e);
        const SampleOp op = sample_op(*args);
        if (op.rows == 0) return 0;
        Operands o;
        const size_t n = op.rows, A = op.actions;
        o.in(op.logits, "logits", type_bytes(op.type), n, op.row_stride, A);
        o.in(op.legal, "legal", 1, n, op.legal_stride, A);
        o.in(op.u, "u", 8, n, 1, 1);
        o.in(op.row_temperature, "row_temperature", 8, n, 1, 1);
        o.in(op.row_top_k, "row_top_k", 4, n, 1, 1);
        o.in(op.row_top_p, "row_top_p", 8, n, 1, 1);
        o.in(op.row_min_p, "row_min_p", 8, n, 1, 1);
        o.out(op.action, "action", 4, n, 1, 1);
        o.out(op.logprob, "logprob", 4, n, 1, 1);
        o.out(op.kept, "kept", 4, n, 1, 1);
        o.out(op.probs, "probs", 4, n, op.probs_stride, A);
        return run_op(o, workspace, workspace_bytes, sample_workspace_bytes(op), stream, [&](hipStream_t st) { return launch_sample(st, op, workspace); });
    });
}

size_t mz_adapter_workspace_bytes(const mz_adapter_args* args) { return check_adapter(args) ? 0 : adapter_workspace_bytes(adapter_op(*args)); }

int mz_adapter_linear(const mz_adapter_args* args, void* workspace, size_t workspace_bytes, void* stream) {
    return guarded([&] {
        if (const char* e = check_adapter(args)) return op_fail(std::string("mz_adapter_linear: ") + e);
        const AdapterOp op = adapter_op(*args);
        if (op.rows == 0) return 0;
        const size_t es = type_bytes(op.type);
        Operands o;
        const size_t M = op.rows, K = op.K, N = op.N, n = op.adapters;
        o.in(op.x, "x", es, M, op.x_stride, K);
        o.in(op.w, "weight", es, N, op.w_stride, K);
        o.in(op.bias, "bias", es, 1, N, N);
        o.in(op.a, "a", es, n * op.rank, K, K);
        o.in(op.b, "b", es, n * N, op.rank, op.rank);
        o.in(op.scale, "scale", 4, n, 1, 1);
        o.in(op.index, "index", 4, M, 1, 1);
        o.out(op.y, "y", type_bytes(op.out_type), M, op.y_stride, N);
        return run_op(o, workspace, workspace_bytes, adapter_workspace_bytes(op), stream, [&](hipStream_t st) { return launch_adapter(st, op, workspace); });
    });
}

}  // extern "C"

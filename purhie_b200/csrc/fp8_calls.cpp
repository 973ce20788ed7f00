// The plain calls of the 8-bit linear layers' Python faces (fp8.py), from checks to launch in one step: outputs not given, nothing
// out of the ordinary.  Where a call is anything else (an output given, a tensor that is not as it has to be, a device that is
// not the current one), nothing is done and None comes back, and the face goes through its own checks, which name what is
// wrong.  A decoded token's operators run for a microsecond or two on the device; through ctypes and one torch call for each
// output a call took 10 us of the host's time (quantize 32 x 4096) or 14 (gemm 1 x 6144 x 4096).
//
// The kernels' launchers are handed over by address (set_launchers): this file links against torch and nothing else here does.
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <algorithm>

namespace py = pybind11;

namespace {

typedef int (*QuantizeFn)(const void*, int, long long, void*, float*, int, int, int, cudaStream_t);
typedef int (*NormFn)(const float*, const void*, int, int, long long, const float*, float, const int32_t*, int, int, int, float*, void*, float*, cudaStream_t);
typedef int (*GatedFn)(const void*, int, int, long long, void*, float*, int, int, const float*, cudaStream_t);
typedef int (*PlanFn)(int, int, int, int, int*, int*);
typedef int (*GemmFn)(const void*, const float*, const void*, const float*, void*, int, int, int, int, int, int, float*, int, int*, cudaStream_t);

QuantizeFn g_quantize;
NormFn g_norm;
GatedFn g_gated;
PlanFn g_plan;
GemmFn g_gemm;

constexpr int64_t BLOCK = 128, MOST = 0x7fffffff, MAX_NORM_WIDTH = 32768;
constexpr auto E4M3 = at::kFloat8_e4m3fn;

int64_t blocks(int64_t n) { return (n + BLOCK - 1) / BLOCK; }
// 0 float32, 1 bfloat16, -1 anything else, as the launchers count
int code(const at::Tensor& t) { return t.scalar_type() == at::kFloat ? 0 : t.scalar_type() == at::kBFloat16 ? 1 : -1; }
// contiguous, of this type, on the current device
bool fits(const at::Tensor& t, at::ScalarType type, int device) { return t.is_cuda() && t.get_device() == device && t.scalar_type() == type && t.is_contiguous(); }
bool is(const at::Tensor& t, int64_t a, int64_t b) { return t.dim() == 2 && t.size(0) == a && t.size(1) == b; }
bool size_ok(int64_t n) { return n > 0 && n <= MOST; }
// The stream that a launch goes to: the scope's (`given`, where it is not negative), else the current one.  While this lives it is the
// current one, so that new tensors are of its memory: another stream's would be handed out again there while the launch still
// works on it.
struct LaunchStream {
    cudaStream_t stream;
    c10::cuda::OptionalCUDAStreamGuard guard;
    LaunchStream(int device, int64_t given) : stream(c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream()) {
        if (given < 0 || (cudaStream_t)given == stream) return;
        stream = (cudaStream_t)given;
        guard.reset_stream(c10::cuda::getStreamFromExternal(stream, (c10::DeviceIndex)device));
    }
};
at::Tensor matrix(int64_t rows, int64_t columns, const at::Tensor& like, at::ScalarType type) { return at::empty({rows, columns}, like.options().dtype(type)); }

// What a launch gave: its outputs, or the status that the face turns into the library's error.
py::object outcome(int status, const at::Tensor& a, const at::Tensor& b) {
    if (status != 0) return py::int_(status);
    return py::make_tuple(a, b);
}

// given: the stream of a scope that has one (>= 0), else -1.  Tensors are made and kernels launched without the interpreter's lock, as
// through ctypes and torch: either waits where memory or the device's queue is full, and what it waits for may need another
// thread of Python.
py::object quantize(const at::Tensor& x, int64_t block_rows, int64_t given) {
    if (!x.is_cuda() || x.dim() != 2 || (block_rows != 1 && block_rows != BLOCK)) return py::none();
    const int64_t T = x.size(0), K = x.size(1), apart = x.stride(0);
    const int device = x.get_device(), type = code(x);
    if (device != c10::cuda::current_device() || type < 0 || !size_ok(T) || !size_ok(K) || (x.stride(1) != 1 && K > 1) || (T > 1 && apart < K)) return py::none();
    at::Tensor q, scales;
    int status;
    {
        py::gil_scoped_release unlocked;
        LaunchStream launch(device, given);
        q = matrix(T, K, x, E4M3);
        scales = matrix(block_rows == 1 ? T : blocks(T), blocks(K), x, at::kFloat);
        status = g_quantize(x.data_ptr(), type, T > 1 ? apart : K, q.data_ptr(), (float*)scales.data_ptr(), (int)T, (int)K, (int)block_rows, launch.stream);
    }
    return outcome(status, q, scales);
}

py::object add_rmsnorm(const at::Tensor& x, const std::optional<at::Tensor>& add, const at::Tensor& weight, double eps, int64_t parts, bool write_x,
                       const std::optional<at::Tensor>& x_out, int64_t given) {
    if (!x.is_cuda() || x.dim() != 2) return py::none();
    const int64_t T = x.size(0), E = x.size(1);
    const int device = x.get_device();
    if (device != c10::cuda::current_device() || !size_ok(T) || E < 1 || E > MAX_NORM_WIDTH || !(eps >= 0.0) || parts < 1 || parts > MOST || !fits(x, at::kFloat, device) ||
        !fits(weight, at::kFloat, device) || weight.dim() != 1 || weight.size(0) != E)
        return py::none();
    int type = 0;
    if (add) {
        type = code(*add);
        const bool whole = add->dim() == 2 && parts == 1, cut = add->dim() == 3 && add->size(0) == parts;
        if (type < 0 || !(whole || cut) || add->size(-2) != T || add->size(-1) != E || !fits(*add, add->scalar_type(), device)) return py::none();
    }
    void* keep = nullptr;
    if (x_out) {
        if (!fits(*x_out, at::kFloat, device) || !is(*x_out, T, E)) return py::none();
        keep = x_out->data_ptr();
    } else if (write_x && add) {
        keep = x.data_ptr();
    }
    at::Tensor q, scales;
    int status;
    {
        py::gil_scoped_release unlocked;
        LaunchStream launch(device, given);
        q = matrix(T, E, x, E4M3);
        scales = matrix(T, blocks(E), x, at::kFloat);
        status = g_norm((const float*)x.data_ptr(), add ? add->data_ptr() : nullptr, type, (int)parts, T * E, (const float*)weight.data_ptr(), (float)eps, nullptr, (int)T, (int)T,
                        (int)E, (float*)keep, q.data_ptr(), (float*)scales.data_ptr(), launch.stream);
    }
    return outcome(status, q, scales);
}

py::object gated(const at::Tensor& gate_up, int64_t parts, int64_t given) {
    const int64_t dim = parts == 1 ? 2 : 3;
    if (!gate_up.is_cuda() || gate_up.dim() != dim || parts < 1 || parts > MOST || (parts > 1 && gate_up.size(0) != parts)) return py::none();
    const int64_t T = gate_up.size(-2), width = gate_up.size(-1), F = width / 2;
    const int device = gate_up.get_device(), type = code(gate_up);
    if (device != c10::cuda::current_device() || type < 0 || !size_ok(T) || !size_ok(width) || width % 2 || !gate_up.is_contiguous()) return py::none();
    at::Tensor q, scales;
    int status;
    {
        py::gil_scoped_release unlocked;
        LaunchStream launch(device, given);
        q = matrix(T, F, gate_up, E4M3);
        scales = matrix(T, blocks(F), gate_up, at::kFloat);
        status = g_gated(gate_up.data_ptr(), type, (int)parts, T * width, q.data_ptr(), (float*)scales.data_ptr(), (int)T, (int)F, nullptr, launch.stream);
    }
    return outcome(status, q, scales);
}

// The whole product, cut as the plan says; bf16: of the output.
py::object gemm(const at::Tensor& x, const at::Tensor& xs, const at::Tensor& w, const at::Tensor& ws, bool bf16, bool early_w, int64_t given) {
    if (!x.is_cuda() || x.dim() != 2 || w.dim() != 2) return py::none();
    const int64_t M = x.size(0), K = x.size(1), N = w.size(0), kb = blocks(K);
    const int device = x.get_device();
    if (device != c10::cuda::current_device() || !size_ok(M) || !size_ok(K) || !size_ok(N) || w.size(1) != K || !fits(x, E4M3, device) || !fits(w, E4M3, device) ||
        !fits(xs, at::kFloat, device) || !fits(ws, at::kFloat, device) || !is(xs, M, kb) || !is(ws, blocks(N), kb))
        return py::none();
    int tile = 0, splits = 0;
    if (const int status = g_plan((int)M, (int)N, (int)K, 1, &tile, &splits)) return py::int_(status);
    at::Tensor out, parts;
    int status;
    {
        py::gil_scoped_release unlocked;
        LaunchStream launch(device, given);
        out = matrix(M, N, x, bf16 ? at::kBFloat16 : at::kFloat);
        if (splits > 1) parts = at::empty({splits, M, N}, x.options().dtype(at::kFloat));
        status = g_gemm(x.data_ptr(), (const float*)xs.data_ptr(), w.data_ptr(), (const float*)ws.data_ptr(), out.data_ptr(), bf16 ? 1 : 0, (int)M, (int)N, (int)K, tile, splits,
                        splits > 1 ? (float*)parts.data_ptr() : nullptr, early_w ? 1 : 0, nullptr, launch.stream);
    }
    if (status != 0) return py::int_(status);
    return py::cast(out);
}

void set_launchers(size_t quantize_fn, size_t norm_fn, size_t gated_fn, size_t plan_fn, size_t gemm_fn) {
    g_quantize = (QuantizeFn)quantize_fn;
    g_norm = (NormFn)norm_fn;
    g_gated = (GatedFn)gated_fn;
    g_plan = (PlanFn)plan_fn;
    g_gemm = (GemmFn)gemm_fn;
}

}  // namespace

PYBIND11_MODULE(fp8_calls, m) {
    m.def("set_launchers", &set_launchers);
    m.def("quantize", &quantize);
    m.def("add_rmsnorm", &add_rmsnorm);
    m.def("gated", &gated);
    m.def("gemm", &gemm);
}

// PyTorch binding of the reproducible operations: the compiled counterpart of the reference's
// repro_torch/src/bindings.cpp:43-175,286-297 (_backend.gemm, exact_sum, conv2d,
// conv2d_grad_weight, conv2d_grad_input, scan_finite), with the same names, arguments, checks
// and results; and the vocabulary loss, the residual norms, attention, the bias of relative positions and dropout (with their
// autograd nodes) and the AdamW steps.
//
// A GPU tensor runs on the MI355X library (librepro_gemm.so, through its C ABI) on PyTorch's
// current HIP stream of the tensor's device, with the workspace taken from PyTorch's caching
// allocator on that stream: each call has its own workspace, which the allocator hands to no
// other stream's work while this call's kernels may still use it. A CPU tensor runs the CPU
// implementation of the same definition (include/repro_*_cpu.h), which gives the same bits.
// Errors from the library raise the package's ReproGemmError (its .code is the hipError_t);
// argument errors raise ValueError.
#include <torch/extension.h>

#include <torch/csrc/autograd/functions/basic_ops.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <stdexcept>
#include <string>
#include <vector>

#include "repro_adamw.h"
#include "repro_adamw_cpu.h"
#include "repro_attention.h"
#include "repro_attention_cpu.h"
#include "repro_conv.h"
#include "repro_conv_cpu.h"
#include "repro_dropout.h"
#include "repro_dropout_cpu.h"
#include "repro_gemm.h"
#include "repro_gemm_cpu.h"
#include "repro_loss.h"
#include "repro_loss_cpu.h"
#include "repro_norm.h"
#include "repro_norm_cpu.h"
#include "repro_sum.h"
#include "repro_sum_cpu.h"

namespace {

using torch::Tensor;

// A non-zero hipError_t from the library, raised in Python as error_class(code, what).
// (A std::exception: the autograd engine's threads hand on no others.)
struct LibraryError : std::exception {
    int code;
    std::string message;
    LibraryError(int c, const char* w) : code(c), message(w) {}
    const char* what() const noexcept override { return message.c_str(); }
};
PyObject* g_error_class = nullptr;  // set once by the package (set_error_class)

void check(int code, const char* what) {
    if (code != 0) throw LibraryError(code, what);
}

void need(bool ok, const std::string& what) {
    if (!ok) throw std::invalid_argument(what);
}

void require_f32(const Tensor& t, const char* name) {
    need(t.scalar_type() == torch::kFloat32, std::string(name) + " must be float32");
}

// Both tensors on the GPU (true), both on the CPU (false), anything else is an error.
bool on_gpu(const Tensor& a, const Tensor& b, const char* op) {
    need(a.device() == b.device(), std::string(op) + ": tensors must be on the same device");
    need(a.is_cuda() || a.is_cpu(), std::string(op) + ": tensors must be on the CPU or a GPU");
    return a.is_cuda();
}

// Lets other Python threads run while the CPU computes, where this thread has the interpreter (a backward
// pass of the binding's own functions has not).
struct Unlocked {
    c10::optional<py::gil_scoped_release> released;
    Unlocked() {
        if (PyGILState_Check()) released.emplace();
    }
};

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

Tensor workspace_like(size_t bytes, const Tensor& t) {
    return torch::empty({(int64_t)std::max<size_t>(bytes, 1)}, t.options().dtype(torch::kUInt8));
}

// A layer's bias (or none) that a library call can add in its own launches: n contiguous floats on
// the operands' device. Any other (a broadcastable shape, another type or stride, a lazily negated
// view, whose memory holds the opposite values) is added by a PyTorch operation.
const float* fusible_bias(const c10::optional<Tensor>& bias, const Tensor& a, int64_t n) {
    if (!bias.has_value()) return nullptr;
    const Tensor& b = *bias;
    const bool ok = b.scalar_type() == torch::kFloat32 && b.device() == a.device() && b.dim() == 1 &&
                    b.size(0) == n && b.is_contiguous() && !b.is_neg();
    return ok ? b.data_ptr<float>() : nullptr;
}

// C[M, N] = op(A) op(B) (bindings.cpp:43-66), with the planner's options exposed: split_k,
// the block tile and the algorithm change the speed, never a bit; they apply to GPU tensors.
// out, when given, must be a contiguous float32 tensor of M*N elements on A's device.
// bias, when given, is added to the rows of C, one rounding per output (an out is not given then).
Tensor gemm_run(Tensor A, Tensor B, int M, int N, int K, bool ta, bool tb, int S, int split_k,
                int tile_m, int tile_n, int algo, c10::optional<Tensor> out,
                c10::optional<Tensor> bias) {
    require_f32(A, "A");
    require_f32(B, "B");
    const bool gpu = on_gpu(A, B, "gemm");
    A = A.contiguous();
    B = B.contiguous();
    need(M > 0 && N > 0 && K > 0, "gemm: sizes must be positive");
    need(A.numel() == (int64_t)M * K && B.numel() == (int64_t)N * K, "gemm: shape mismatch");
    Tensor C;
    if (out.has_value()) {
        C = *out;
        need(C.scalar_type() == torch::kFloat32, "gemm: out must be float32");
        need(C.device() == A.device(), "gemm: out must be on the inputs' device");
        need(C.is_contiguous() && C.numel() == (int64_t)M * N, "gemm: out must be contiguous with M*N elements");
    } else {
        C = torch::empty({M, N}, A.options());
    }
    if (gpu) {
        c10::DeviceGuard guard(A.device());
        rg_config cfg;
        rg_config_init(&cfg);
        cfg.slices = S;
        cfg.trans_a = ta ? 1 : 0;
        cfg.trans_b = tb ? 1 : 0;
        cfg.split_k = split_k;
        cfg.tile_m = tile_m;
        cfg.tile_n = tile_n;
        cfg.algo = algo;
        rg_plan plan;
        check(rg_make_plan(M, N, K, &cfg, &plan), "gemm plan");
        Tensor ws = workspace_like(plan.workspace_bytes, A);
        if (const float* b = fusible_bias(bias, A, N)) {
            check(rg_gemm_bias_fp32_ws(A.data_ptr<float>(), B.data_ptr<float>(), b, C.data_ptr<float>(),
                                       M, N, K, &cfg, ws.data_ptr(), (size_t)ws.numel(), stream_of(A)),
                  "gemm");
            return C;
        }
        check(rg_gemm_fp32_ws(A.data_ptr<float>(), B.data_ptr<float>(), C.data_ptr<float>(), M, N, K,
                              &cfg, ws.data_ptr(), (size_t)ws.numel(), stream_of(A), nullptr),
              "gemm");
        return bias.has_value() ? C + *bias : C;
    }
    need(S >= 1 && S <= 3, "gemm: slices must be 1..3");
    const float* a = A.data_ptr<float>();
    const float* b = B.data_ptr<float>();
    float* c = C.data_ptr<float>();
    py::gil_scoped_release nogil;
    repro_gemm::cpu_gemm(a, b, c, M, N, K, ta, tb, S);
    return bias.has_value() ? C + *bias : C;
}

Tensor gemm_ex(Tensor A, Tensor B, int M, int N, int K, bool ta, bool tb, int S, int split_k,
               int tile_m, int tile_n, int algo, c10::optional<Tensor> out) {
    return gemm_run(std::move(A), std::move(B), M, N, K, ta, tb, S, split_k, tile_m, tile_n, algo,
                    std::move(out), c10::nullopt);
}

// y[M, N] = x[M, K] w[N, K]^T, plus bias (or None).
Tensor linear(Tensor x, Tensor w, c10::optional<Tensor> bias, int M, int N, int K, int S) {
    return gemm_run(std::move(x), std::move(w), M, N, K, false, true, S, 1, 16, 16, RG_ALGO_AUTO,
                    c10::nullopt, std::move(bias));
}

Tensor gemm(Tensor A, Tensor B, int M, int N, int K, bool ta, bool tb, int S) {
    return gemm_run(std::move(A), std::move(B), M, N, K, ta, tb, S, 1, 16, 16, RG_ALGO_AUTO, c10::nullopt,
                    c10::nullopt);
}

// out[b] = exact sum over a, c of x[a, b, c], rounded once; divided by A * C if mean
// (bindings.cpp:69-91).
// flag, when given, is also lowered to op_id if x holds a NaN or infinity (GPU tensors only).
Tensor sum_run(Tensor x, int A, int B, int C, bool mean, c10::optional<Tensor> flag, int op_id) {
    require_f32(x, "x");
    need(x.is_cuda() || x.is_cpu(), "sum: x must be on the CPU or a GPU");
    x = x.contiguous();
    need(A > 0 && B > 0 && C > 0, "sum: sizes must be positive");
    need(x.numel() == (int64_t)A * B * C, "sum: shape mismatch");
    Tensor out = torch::empty({B}, x.options());
    if (x.is_cuda()) {
        c10::DeviceGuard guard(x.device());
        rg_sum_config cfg;
        rg_sum_config_init(&cfg);
        cfg.mean = mean ? 1 : 0;
        rg_sum_plan plan;
        check(rg_make_sum_plan(A, B, C, &cfg, &plan), "sum plan");
        Tensor ws = workspace_like(plan.workspace_bytes, x);
        check(rg_sum_watch_fp32_ws(x.data_ptr<float>(), out.data_ptr<float>(), A, B, C, &cfg,
                                   ws.data_ptr(), (size_t)ws.numel(),
                                   flag.has_value() ? flag->data_ptr<int>() : nullptr, op_id,
                                   stream_of(x)),
              "sum");
        return out;
    }
    const float* p = x.data_ptr<float>();
    float* o = out.data_ptr<float>();
    py::gil_scoped_release nogil;
    repro_sum::cpu_sum(p, o, A, B, C, mean);
    return out;
}

Tensor exact_sum(Tensor x, int A, int B, int C, bool mean) {
    return sum_run(std::move(x), A, B, C, mean, c10::nullopt, 0);
}

void require_flag(const Tensor& flag, const Tensor& x, const char* op) {
    need(flag.scalar_type() == torch::kInt32 && flag.numel() >= 1,
         std::string(op) + ": flag must be an int32 tensor");
    need(on_gpu(x, flag, op), std::string(op) + ": tensors must be on a GPU");
}

// exact_sum and scan_finite of one GPU tensor in one read of it.
Tensor exact_sum_watch(Tensor x, int A, int B, int C, Tensor flag, int op_id) {
    require_f32(x, "x");
    require_flag(flag, x, "exact_sum_watch");
    return sum_run(std::move(x), A, B, C, false, std::move(flag), op_id);
}

repro_conv::ConvShape shape_of(const std::vector<int64_t>& x_shape, int F, int KH, int KW, int SY,
                               int SX, int PY, int PX) {
    need(x_shape.size() == 4, "conv: the input must be [N][C][H][W]");
    repro_conv::ConvShape g;
    g.N = (int)x_shape[0];
    g.C = (int)x_shape[1];
    g.H = (int)x_shape[2];
    g.W = (int)x_shape[3];
    g.F = F;
    g.KH = KH;
    g.KW = KW;
    g.SY = SY;
    g.SX = SX;
    g.PY = PY;
    g.PX = PX;
    return g;
}

typedef int (*ConvWorkspaceFn)(const rg_conv_shape*, int, size_t*);

// One convolution pass on the GPU: plan, per-call workspace, launch on the current stream.
template <class Run>
void conv_gpu(ConvWorkspaceFn ws_fn, Run run, const Tensor& a, const Tensor& b, Tensor& out,
              const repro_conv::ConvShape& g, int S, const char* what) {
    c10::DeviceGuard guard(a.device());
    const rg_conv_shape s = g.to_c();
    size_t bytes = 0;
    check(ws_fn(&s, S, &bytes), "conv plan");
    Tensor ws = workspace_like(bytes, a);
    check(run(a.data_ptr<float>(), b.data_ptr<float>(), out.data_ptr<float>(), &s, S, ws.data_ptr(),
              (size_t)ws.numel(), stream_of(a)),
          what);
}

// out[N][F][OH][OW] from x[N][C][H][W] and w[F][C][KH][KW] (bindings.cpp:112-131).
// bias, when given, is added to the channels of out, one rounding per output.
Tensor conv2d_bias(Tensor x, Tensor w, c10::optional<Tensor> bias, int SY, int SX, int PY, int PX,
                   int S) {
    require_f32(x, "x");
    require_f32(w, "weight");
    const bool gpu = on_gpu(x, w, "conv2d");
    x = x.contiguous();
    w = w.contiguous();
    need(x.dim() == 4 && w.dim() == 4, "conv2d: x and weight must be 4-D");
    need(w.size(1) == x.size(1), "conv2d: weight channels do not match the input");
    auto g = shape_of(x.sizes().vec(), (int)w.size(0), (int)w.size(2), (int)w.size(3), SY, SX, PY, PX);
    need(repro_conv::cpu_shape_valid(g, S), "conv2d: invalid shape");
    Tensor out = torch::empty({g.N, g.F, g.OH(), g.OW()}, x.options());
    if (gpu) {
        const float* b = fusible_bias(bias, x, g.F);
        const auto fused = [b](const float* px, const float* pw, float* po, const rg_conv_shape* s,
                               int S, void* ws, size_t bytes, void* stream) {
            return rg_conv2d_bias_ws(px, pw, b, po, s, S, ws, bytes, stream);
        };
        if (b != nullptr) {
            conv_gpu(rg_conv2d_workspace, fused, x, w, out, g, S, "conv");
            return out;
        }
        conv_gpu(rg_conv2d_workspace, rg_conv2d_ws, x, w, out, g, S, "conv");
        return bias.has_value() ? out + bias->view({1, -1, 1, 1}) : out;
    }
    const float *px = x.data_ptr<float>(), *pw = w.data_ptr<float>();
    float* po = out.data_ptr<float>();
    py::gil_scoped_release nogil;
    repro_conv::cpu_conv2d(px, pw, po, g, S);
    return bias.has_value() ? out + bias->view({1, -1, 1, 1}) : out;
}

Tensor conv2d(Tensor x, Tensor w, int SY, int SX, int PY, int PX, int S) {
    return conv2d_bias(std::move(x), std::move(w), c10::nullopt, SY, SX, PY, PX, S);
}

// dW[F][C][KH][KW] from dY[N][F][OH][OW] and x (bindings.cpp:133-152).
Tensor conv2d_grad_weight(Tensor dy, Tensor x, int KH, int KW, int SY, int SX, int PY, int PX, int S) {
    require_f32(dy, "dy");
    require_f32(x, "x");
    const bool gpu = on_gpu(dy, x, "conv2d_grad_weight");
    dy = dy.contiguous();
    x = x.contiguous();
    need(x.dim() == 4 && dy.dim() == 4, "conv2d_grad_weight: dy and x must be 4-D");
    auto g = shape_of(x.sizes().vec(), (int)dy.size(1), KH, KW, SY, SX, PY, PX);
    need(repro_conv::cpu_shape_valid(g, S), "conv2d_grad_weight: invalid shape");
    need(dy.size(0) == g.N && dy.size(2) == g.OH() && dy.size(3) == g.OW(),
         "conv2d_grad_weight: dy shape does not match the convolution");
    Tensor dw = torch::empty({g.F, g.C, KH, KW}, x.options());
    if (gpu) {
        conv_gpu(rg_conv2d_grad_weight_workspace, rg_conv2d_grad_weight_ws, dy, x, dw, g, S, "conv weight grad");
        return dw;
    }
    const float *pd = dy.data_ptr<float>(), *px = x.data_ptr<float>();
    float* po = dw.data_ptr<float>();
    py::gil_scoped_release nogil;
    repro_conv::cpu_conv2d_grad_weight(pd, px, po, g, S);
    return dw;
}

// dX[N][C][H][W] (x_shape) from dY[N][F][OH][OW] and w (bindings.cpp:154-175).
Tensor conv2d_grad_input(Tensor dy, Tensor w, std::vector<int64_t> x_shape, int SY, int SX, int PY,
                         int PX, int S) {
    require_f32(dy, "dy");
    require_f32(w, "weight");
    const bool gpu = on_gpu(dy, w, "conv2d_grad_input");
    dy = dy.contiguous();
    w = w.contiguous();
    need(dy.dim() == 4 && w.dim() == 4, "conv2d_grad_input: dy and weight must be 4-D");
    auto g = shape_of(x_shape, (int)w.size(0), (int)w.size(2), (int)w.size(3), SY, SX, PY, PX);
    need(repro_conv::cpu_shape_valid(g, S), "conv2d_grad_input: invalid shape");
    need(w.size(1) == g.C && dy.size(0) == g.N && dy.size(1) == g.F && dy.size(2) == g.OH() &&
             dy.size(3) == g.OW(),
         "conv2d_grad_input: shapes do not match the convolution");
    Tensor dx = torch::empty(x_shape, dy.options());
    if (gpu) {
        conv_gpu(rg_conv2d_grad_input_workspace, rg_conv2d_grad_input_ws, dy, w, dx, g, S, "conv input grad");
        return dx;
    }
    const float *pd = dy.data_ptr<float>(), *pw = w.data_ptr<float>();
    float* po = dx.data_ptr<float>();
    py::gil_scoped_release nogil;
    repro_conv::cpu_conv2d_grad_input(pd, pw, po, g, S);
    return dx;
}

// Lowers flag[0] to op_id if x holds a NaN or infinity, without synchronising
// (bindings.cpp:286-297).
void scan_finite(Tensor x, Tensor flag, int op_id) {
    require_f32(x, "x");
    need(flag.scalar_type() == torch::kInt32 && flag.numel() >= 1, "scan_finite: flag must be an int32 tensor");
    const bool gpu = on_gpu(x, flag, "scan_finite");
    x = x.contiguous();
    if (gpu) {
        c10::DeviceGuard guard(x.device());
        check(rg_scan_finite(x.data_ptr<float>(), flag.data_ptr<int>(), (size_t)x.numel(), op_id, stream_of(x)),
              "finite scan");
        return;
    }
    const float* p = x.data_ptr<float>();
    int* f = flag.data_ptr<int>();
    const int64_t n = x.numel();
    for (int64_t i = 0; i < n; ++i) {
        if ((repro_gemm::float_to_bits(p[i]) & 0x7F800000u) == 0x7F800000u) {
            if (op_id < *f) *f = op_id;
            return;
        }
    }
}

// scan_finite of two GPU tensors in one launch.
void scan_finite_pair(Tensor x, int op_x, Tensor y, int op_y, Tensor flag) {
    require_f32(x, "x");
    require_f32(y, "x");
    require_flag(flag, x, "scan_finite");
    require_flag(flag, y, "scan_finite");
    x = x.contiguous();
    y = y.contiguous();
    c10::DeviceGuard guard(x.device());
    check(rg_scan_finite_pair(x.data_ptr<float>(), (size_t)x.numel(), op_x, y.data_ptr<float>(),
                              (size_t)y.numel(), op_y, flag.data_ptr<int>(), stream_of(x)),
          "finite scan");
}

// ---- AdamW ----

rg_adamw_config adamw_config(double lr, double beta1, double beta2, double eps, double weight_decay, int64_t step) {
    need(lr >= 0 && eps >= 0 && weight_decay >= 0, "adamw: lr, eps and weight_decay must not be negative");
    need(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1, "adamw: betas must be in [0, 1)");
    need(step >= 1, "adamw: step must be at least 1");
    rg_adamw_config c;
    rg_adamw_config_init(&c);
    c.lr = lr;
    c.beta1 = beta1;
    c.beta2 = beta2;
    c.eps = eps;
    c.weight_decay = weight_decay;
    c.step = step;
    return c;
}

repro_adamw::Scalars adamw_scalars(const rg_adamw_config& c) {
    return repro_adamw::make_scalars(c.lr, c.beta1, c.beta2, c.eps, c.weight_decay, c.step);
}

// The tensors of a Python list or tuple, which holds them while the call runs (taking a few hundred of them as a
// vector, with its reference counts, and building every check's message took longer than the step).
struct Listed {
    py::object held;
    std::vector<const Tensor*> t;
    Listed(const py::handle& list, const char* name) {
        held = py::reinterpret_steal<py::object>(PySequence_Fast(list.ptr(), "adamw takes lists of tensors"));
        if (!held) throw py::error_already_set();
        const Py_ssize_t n = PySequence_Fast_GET_SIZE(held.ptr());
        PyObject** items = PySequence_Fast_ITEMS(held.ptr());
        t.reserve(n);
        for (Py_ssize_t i = 0; i < n; ++i) {
            if (!THPVariable_Check(items[i])) need(false, std::string("adamw: ") + name + " must be tensors");
            t.push_back(&THPVariable_Unpack(items[i]));
        }
    }
    size_t size() const { return t.size(); }
    const Tensor& operator[](size_t i) const { return *t[i]; }
};

// The step goes through a tensor's memory in its own order, so all of a value's tensors must be
// dense, without overlaps and laid out alike.
void need_alike(const Tensor& p, const Tensor& t, const char* name) {
    if (t.scalar_type() == torch::kFloat32 && t.device() == p.device() && t.sizes() == p.sizes() && !t.is_neg() &&
        (p.is_contiguous() ? t.is_contiguous() : t.strides() == p.strides()))
        return;
    need(false, std::string("adamw: ") + name + " must be float32, on its parameter's device, with its shape and strides" +
                    (t.is_neg() ? " (and no lazily negated view)" : ""));
}

// The first parameter's device kind (true: GPU); every parameter float32, dense and on that device.
bool adamw_parameters(const Listed& params, const Listed& grads) {
    need(params.size() == grads.size(), "adamw: as many gradients as parameters");
    for (size_t i = 0; i < params.size(); ++i) {
        const Tensor& p = params[i];
        if (p.device() != params[0].device()) need(false, "adamw: parameters must be on one device");
        if (!p.is_cuda() && !p.is_cpu()) need(false, "adamw: parameters must be on the CPU or a GPU");
        if (!p.is_non_overlapping_and_dense()) need(false, "adamw: parameters must be dense");
        need_alike(p, p, "a parameter");
        need_alike(p, grads[i], "a gradient");
    }
    return params.size() > 0 && params[0].is_cuda();
}

// Nothing that a step writes may overlap: threads of a launch would read and write the same values. Neighbours in a list
// and what belongs to one parameter are compared, which the loop over the tensors does by the way: that finds one
// buffer given for several. (Sorting all addresses finds the rest and took 10 to 22 us for 300 tensors, of 34 to 51.)
struct Range {
    uintptr_t first = 0, end = 0;
    Range() = default;
    Range(const void* p, int64_t bytes) : first(reinterpret_cast<uintptr_t>(p)), end(first + (uintptr_t)bytes) {}
    bool apart(const Range& b) const { return first >= b.end || b.first >= end; }
};
const char* const OVERLAP = "adamw: parameters and moments must not overlap";
// Whether a list's tensors, taken one after another, are apart from the one before.
struct Neighbours {
    Range last;
    bool apart = true;
    Range next(const void* p, int64_t bytes) {
        const Range r(p, bytes);
        apart &= r.apart(last);
        if (bytes > 0) last = r;
        return r;
    }
};

// What autograd has saved of a tensor is not its value any more.
void changed(const Listed& list) {
    for (const Tensor* t : list.t)
        if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

void adamw_step(py::handle params_, py::handle grads_, py::handle m_, py::handle v_, double lr, double beta1,
                double beta2, double eps, double weight_decay, int64_t step) {
    const rg_adamw_config cfg = adamw_config(lr, beta1, beta2, eps, weight_decay, step);
    const Listed params(params_, "parameters"), grads(grads_, "gradients"), m(m_, "moments"), v(v_, "moments");
    const bool gpu = adamw_parameters(params, grads);
    need(m.size() == params.size() && v.size() == params.size(), "adamw: as many moments as parameters");
    std::vector<rg_adamw_tensor> list(params.size());
    Neighbours at_p, at_m, at_v;
    bool apart = true;
    for (size_t i = 0; i < params.size(); ++i) {
        need_alike(params[i], m[i], "a first moment");
        need_alike(params[i], v[i], "a second moment");
        list[i] = {params[i].data_ptr<float>(), grads[i].data_ptr<float>(), m[i].data_ptr<float>(),
                   v[i].data_ptr<float>(), (long long)params[i].numel()};
        const Range p = at_p.next(list[i].p, 4 * list[i].n), q = at_m.next(list[i].m, 4 * list[i].n),
                    r = at_v.next(list[i].v, 4 * list[i].n);
        apart &= p.apart(q) & p.apart(r) & q.apart(r);
    }
    if (list.empty()) return;
    need(apart && at_p.apart && at_m.apart && at_v.apart, OVERLAP);
    for (const Listed* changing : {&params, &m, &v}) changed(*changing);
    if (gpu) {
        c10::DeviceGuard guard(params[0].device());
        check(rg_adamw_fp32(list.data(), (int)list.size(), &cfg, stream_of(params[0])), "adamw");
        return;
    }
    const repro_adamw::Scalars s = adamw_scalars(cfg);
    Unlocked unlocked;
    for (const rg_adamw_tensor& t : list) repro_adamw::cpu_adamw(t.p, t.g, t.m, t.v, t.n, s);
}

int64_t adamw8_blocks(int64_t n) { return (n + RG_ADAMW8_BLOCK - 1) / RG_ADAMW8_BLOCK; }

void need_codes(const Tensor& t, const Tensor& p, int64_t n, const char* name) {
    if (t.scalar_type() == torch::kUInt8 && t.is_contiguous() && t.device() == p.device() && t.numel() == n &&
        (reinterpret_cast<uintptr_t>(t.data_ptr()) & 3) == 0)
        return;
    need(false, std::string("adamw: ") + name + " must be contiguous uint8 of " + std::to_string(n) +
                    " values, at a multiple of 4 bytes, on the parameters' device");
}

void need_exponents(const Tensor& t, const Tensor& p, int64_t n) {
    if (!(t.scalar_type() == torch::kUInt8 && t.is_contiguous() && t.device() == p.device() && t.numel() == n))
        need(false, "adamw: exponents must be contiguous uint8, one a block, on the parameters' device");
}

// The moments' codes and exponents: one tensor of each for all parameters (each parameter at whole
// blocks, in order), or one for each parameter.
void adamw8_step(py::handle params_, py::handle grads_, py::handle m_, py::handle m_exp_, py::handle v_,
                 py::handle v_exp_, bool flat, double lr, double beta1, double beta2, double eps, double weight_decay,
                 int64_t step) {
    const rg_adamw_config cfg = adamw_config(lr, beta1, beta2, eps, weight_decay, step);
    const Listed params(params_, "parameters"), grads(grads_, "gradients"), m(m_, "moments"), m_exp(m_exp_, "exponents"),
        v(v_, "moments"), v_exp(v_exp_, "exponents");
    const bool gpu = adamw_parameters(params, grads);
    const size_t states = flat ? 1 : params.size();
    need(m.size() == states && m_exp.size() == states && v.size() == states && v_exp.size() == states,
         "adamw: as many moments as parameters");
    if (params.size() == 0) return;
    const auto need_state = [&](size_t k, int64_t blocks) {
        need_codes(m[k], params[0], blocks * RG_ADAMW8_BLOCK, "the first moments");
        need_codes(v[k], params[0], blocks * RG_ADAMW8_BLOCK, "the second moments");
        need_exponents(m_exp[k], params[0], blocks);
        need_exponents(v_exp[k], params[0], blocks);
    };
    int64_t total = 0;
    for (const Tensor* p : params.t) total += adamw8_blocks(p->numel());
    if (flat) need_state(0, total);
    int64_t at = 0;
    std::vector<rg_adamw8_tensor> list(params.size());
    Neighbours at_p, at_m, at_m_exp, at_v, at_v_exp;
    bool apart = true;
    for (size_t i = 0; i < params.size(); ++i) {
        const int64_t blocks = adamw8_blocks(params[i].numel());
        if (!flat) need_state(i, blocks);
        const size_t k = flat ? 0 : i;
        list[i] = {params[i].data_ptr<float>(), grads[i].data_ptr<float>(),
                   m[k].data_ptr<uint8_t>() + at * RG_ADAMW8_BLOCK, m_exp[k].data_ptr<uint8_t>() + at,
                   v[k].data_ptr<uint8_t>() + at * RG_ADAMW8_BLOCK, v_exp[k].data_ptr<uint8_t>() + at,
                   (long long)params[i].numel()};
        at_p.next(list[i].p, 4 * list[i].n);
        if (flat) at += blocks;
        if (flat && i > 0) continue;
        const int64_t held = flat ? total : blocks;
        apart &= at_m.next(list[i].m, held * RG_ADAMW8_BLOCK).apart(at_v.next(list[i].v, held * RG_ADAMW8_BLOCK));
        apart &= at_m_exp.next(list[i].m_exp, held).apart(at_v_exp.next(list[i].v_exp, held));
    }
    need(apart && at_p.apart && at_m.apart && at_m_exp.apart && at_v.apart && at_v_exp.apart, OVERLAP);
    for (const Listed* changing : {&params, &m, &m_exp, &v, &v_exp}) changed(*changing);
    if (gpu) {
        c10::DeviceGuard guard(params[0].device());
        check(rg_adamw8_fp32(list.data(), (int)list.size(), &cfg, stream_of(params[0])), "adamw8");
        return;
    }
    const repro_adamw::Scalars s = adamw_scalars(cfg);
    Unlocked unlocked;
    int64_t first = 0;
    for (const rg_adamw8_tensor& t : list) {
        repro_adamw::cpu_adamw8(t.p, t.g, t.m, t.m_exp, t.v, t.v_exp, t.n, first, s);
        first += adamw8_blocks(t.n);
    }
}

std::vector<Tensor> adamw8_values(const Tensor& m, const Tensor& m_exp, const Tensor& v, const Tensor& v_exp) {
    const int64_t blocks = m_exp.numel();
    need(m.is_cuda() || m.is_cpu(), "adamw: tensors must be on the CPU or a GPU");
    need_codes(m, m, blocks * RG_ADAMW8_BLOCK, "the first moments");
    need_codes(v, m, blocks * RG_ADAMW8_BLOCK, "the second moments");
    need_exponents(m_exp, m, blocks);
    need_exponents(v_exp, m, blocks);
    Tensor mo = torch::empty({blocks * RG_ADAMW8_BLOCK}, m.options().dtype(torch::kFloat32));
    Tensor vo = torch::empty_like(mo);
    if (m.is_cuda()) {
        c10::DeviceGuard guard(m.device());
        check(rg_adamw8_values(m.data_ptr<uint8_t>(), m_exp.data_ptr<uint8_t>(), v.data_ptr<uint8_t>(),
                               v_exp.data_ptr<uint8_t>(), mo.data_ptr<float>(), vo.data_ptr<float>(), blocks,
                               stream_of(m)),
              "adamw8 values");
    } else {
        repro_adamw::cpu_adamw8_values(m.data_ptr<uint8_t>(), m_exp.data_ptr<uint8_t>(), mo.data_ptr<float>(), blocks, true);
        repro_adamw::cpu_adamw8_values(v.data_ptr<uint8_t>(), v_exp.data_ptr<uint8_t>(), vo.data_ptr<float>(), blocks, false);
    }
    return {mo, vo};
}

// ---- norms ----

using OptTensor = c10::optional<Tensor>;

// A float32 tensor of `numel` values on x's device, contiguous; undefined where there is none.
Tensor norm_operand(const OptTensor& t, const Tensor& x, int64_t numel, const char* name) {
    if (!t.has_value()) return Tensor();
    if (t->scalar_type() != torch::kFloat32 || t->device() != x.device() || t->numel() != numel)
        need(false, std::string("norm: ") + name + " must be float32, on x's device, with " + std::to_string(numel) + " values");
    return t->resolve_neg().contiguous();
}

const float* data_or_null(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
float* out_or_null(Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }

rg_norm_config norm_config(const Tensor& x, const OptTensor& gate, bool rms, bool post, double eps, double scale) {
    require_f32(x, "x");
    need(x.is_cuda() || x.is_cpu(), "norm: tensors must be on the CPU or a GPU");
    need(x.dim() >= 1 && x.size(-1) >= 1, "norm: x must be [..., values]");
    need(x.size(-1) <= RG_NORM_MAX_D, "norm: a row must have at most 16384 values");
    static_assert(RG_NORM_MAX_D == 16384, "the message above");
    need(eps >= 0, "norm: eps must not be negative");
    rg_norm_config c;
    rg_norm_config_init(&c);
    c.D = (int)x.size(-1);
    c.N = x.numel() / c.D;
    c.rms = rms ? 1 : 0;
    c.post = post ? 1 : 0;
    c.eps = (float)eps;
    c.scale = (float)scale;
    if (gate.has_value() && c.N > 0) {
        const int64_t rows = gate->numel() / c.D;
        need(rows >= 1 && gate->numel() == rows * c.D && rows <= c.N && c.N % rows == 0,
             "norm: the gate's rows must divide x's");
        c.gate_rows = rows;
    }
    return c;
}

// Lowers a CPU's flag, where there is one.
void report(const OptTensor& flag, bool bad, int op_id) {
    if (bad && flag.has_value()) flag->data_ptr<int>()[0] = std::min(flag->data_ptr<int>()[0], op_id);
}

// x, f [..., D] -> {r (undefined without f), y, stats (undefined unless wanted)}
std::vector<OptTensor> residual_norm(Tensor x, OptTensor f_, OptTensor gate_, OptTensor post_weight_, OptTensor post_bias_,
                                     OptTensor weight_, OptTensor bias_, bool rms, bool post, double eps, double scale,
                                     bool want_stats, OptTensor flag, int op_id) {
    rg_norm_config c = norm_config(x, gate_, rms, post, eps, scale);
    x = x.resolve_neg().contiguous();
    const int64_t D = c.D;
    const Tensor f = norm_operand(f_, x, x.numel(), "f");
    const Tensor gate = norm_operand(gate_, x, gate_.has_value() ? gate_->numel() : 0, "the gate");
    const Tensor pw = norm_operand(post_weight_, x, D, "post_weight"), pb = norm_operand(post_bias_, x, D, "post_bias");
    const Tensor w = norm_operand(weight_, x, D, "weight"), b = norm_operand(bias_, x, D, "bias");
    need(f.defined() || (!gate.defined() && !post), "norm: a gate or a post norm needs f");
    need(post || (!pw.defined() && !pb.defined()), "norm: post_weight and post_bias need the post norm");
    Tensor y = torch::empty_like(x), r, stats;
    if (f.defined()) r = torch::empty_like(x);
    if (want_stats) stats = torch::empty({c.N, 4}, x.options());
    if (x.is_cuda()) {
        c10::DeviceGuard guard(x.device());
        if (flag.has_value()) require_flag(*flag, x, "residual_norm");
        check(rg_residual_norm_fp32(&c, x.data_ptr<float>(), data_or_null(f), c.N > 0 ? data_or_null(gate) : nullptr,
                                    data_or_null(pw), data_or_null(pb), data_or_null(w), data_or_null(b),
                                    out_or_null(r), y.data_ptr<float>(), out_or_null(stats),
                                    flag.has_value() ? flag->data_ptr<int>() : nullptr, op_id, stream_of(x)),
              "residual norm");
    } else {
        Unlocked unlocked;
        bool bad = false;
        repro_norm::cpu_residual_norm(c, x.data_ptr<float>(), data_or_null(f), data_or_null(gate), data_or_null(pw),
                                      data_or_null(pb), data_or_null(w), data_or_null(b), out_or_null(r),
                                      y.data_ptr<float>(), out_or_null(stats), &bad);
        report(flag, bad, op_id);
    }
    const auto opt = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
    return {opt(r), opt(y), opt(stats)};
}

// {dx, df, dgate, dpost_weight, dpost_bias, dweight, dbias}, those that `want` asks for.
std::vector<OptTensor> residual_norm_grad(OptTensor dr_, OptTensor dy_, Tensor r, OptTensor f_, OptTensor gate_,
                                          OptTensor post_weight_, OptTensor post_bias_, OptTensor weight_, Tensor stats,
                                          bool rms, bool post, double eps, double scale, std::vector<bool> want,
                                          OptTensor flag, int op_id) {
    rg_norm_config c = norm_config(r, gate_, rms, post, eps, scale);
    need(want.size() == 7, "norm: seven gradients");
    need(r.is_contiguous(), "norm: r must be contiguous");
    const int64_t D = c.D;
    const Tensor dr = norm_operand(dr_, r, r.numel(), "dr"), dy = norm_operand(dy_, r, r.numel(), "dy");
    const Tensor f = norm_operand(f_, r, r.numel(), "f");
    const Tensor gate = norm_operand(gate_, r, gate_.has_value() ? gate_->numel() : 0, "the gate");
    const Tensor pw = norm_operand(post_weight_, r, D, "post_weight"), pb = norm_operand(post_bias_, r, D, "post_bias");
    const Tensor w = norm_operand(weight_, r, D, "weight");
    need(stats.scalar_type() == torch::kFloat32 && stats.device() == r.device() && stats.is_contiguous() &&
             stats.numel() == 4 * c.N,
         "norm: stats must be the forward pass's");
    need(dr.defined() || dy.defined(), "norm: a gradient of r or y is needed");
    const auto rows = r.options();
    const auto maybe = [&](int i, at::IntArrayRef shape) { return want[i] ? torch::empty(shape, rows) : Tensor(); };
    Tensor dx = maybe(0, r.sizes()), df = maybe(1, r.sizes());
    Tensor dgate = want[2] ? torch::empty(gate.sizes(), rows) : Tensor();
    Tensor dpw = maybe(3, {D}), dpb = maybe(4, {D}), dw = maybe(5, {D}), db = maybe(6, {D});
    if (!dy.defined()) {  // y was not used: its weight's gradients are zero
        for (Tensor* t : {&dw, &db})
            if (t->defined()) t->zero_();
    }
    Tensor kernel_dw = dy.defined() ? dw : Tensor(), kernel_db = dy.defined() ? db : Tensor();
    if (c.N == 0) {
        for (Tensor* t : {&dgate, &dpw, &dpb, &dw, &db})
            if (t->defined()) t->zero_();
    } else if (r.is_cuda()) {
        c10::DeviceGuard guard(r.device());
        if (flag.has_value()) require_flag(*flag, r, "residual_norm_grad");
        const bool sums = dgate.defined() || dpw.defined() || dpb.defined() || kernel_dw.defined() || kernel_db.defined();
        size_t bytes = 0;
        check(rg_residual_norm_grad_workspace(&c, sums ? 1 : 0, &bytes), "norm gradient plan");
        Tensor ws = workspace_like(bytes, r);
        check(rg_residual_norm_grad_fp32(&c, data_or_null(dr), data_or_null(dy), r.data_ptr<float>(), data_or_null(f),
                                         data_or_null(gate), data_or_null(pw), data_or_null(pb), data_or_null(w),
                                         stats.data_ptr<float>(), out_or_null(dx), out_or_null(df), out_or_null(dgate),
                                         out_or_null(dpw), out_or_null(dpb), out_or_null(kernel_dw),
                                         out_or_null(kernel_db), ws.data_ptr(), (size_t)ws.numel(),
                                         flag.has_value() ? flag->data_ptr<int>() : nullptr, op_id, stream_of(r)),
              "norm gradient");
    } else {
        Unlocked unlocked;
        bool bad = false;
        repro_norm::cpu_residual_norm_grad(c, data_or_null(dr), data_or_null(dy), r.data_ptr<float>(), data_or_null(f),
                                           data_or_null(gate), data_or_null(pw), data_or_null(pb), data_or_null(w),
                                           stats.data_ptr<float>(), out_or_null(dx), out_or_null(df),
                                           out_or_null(dgate), out_or_null(dpw), out_or_null(dpb),
                                           out_or_null(kernel_dw), out_or_null(kernel_db), &bad);
        report(flag, bad, op_id);
    }
    const auto opt = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
    return {opt(dx), opt(df), opt(dgate), opt(dpw), opt(dpb), opt(dw), opt(db)};
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Gradients that are not differentiable themselves: where a graph of the backward pass is wanted, using it
// raises an error (and is not left out of it silently).
void differentiable_once(variable_list& grads, const char* op) {
    if (!at::GradMode::is_enabled()) return;
    for (Tensor& g : grads) {
        if (!g.defined()) continue;
        torch::autograd::DelayedError error(std::string(op) + " is differentiable only once", 1);
        g = error.apply({g.detach().requires_grad_()})[0];
    }
}

OptTensor opt_of(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
Tensor or_undefined(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }

// Where a module reports a NaN or infinity: an int32 cell of x's device (or nowhere) and the numbers of its
// labels for the input and the gradient.
struct Watch {
    OptTensor cell;
    int64_t input, gradient;
};

// Autograd in the binding (from Python, a norm's two passes took 130 us of host time, of the kernels' 46).
// The operands are x, f, gate, post_weight, post_bias, weight, bias.
struct NormFunction : torch::autograd::Function<NormFunction> {
    static variable_list forward(AutogradContext* ctx, Tensor x, OptTensor f, OptTensor gate, OptTensor post_weight,
                                 OptTensor post_bias, OptTensor weight, OptTensor bias, bool rms, bool post, double eps,
                                 double scale, Watch watch, std::vector<bool> want) {
        bool any = false;
        for (const bool w : want) any = any || w;
        auto out = residual_norm(x, f, gate, post_weight, post_bias, weight, bias, rms, post, eps, scale, any, watch.cell,
                                 (int)watch.input);
        if (any) {
            ctx->save_for_backward({f.has_value() ? *out[0] : x, or_undefined(f), or_undefined(gate), or_undefined(post_weight),
                                    or_undefined(post_bias), or_undefined(weight), *out[2]});
            ctx->saved_data["settings"] = std::make_tuple(rms, post, eps, scale);
            ctx->saved_data["cell"] = watch.cell;
            ctx->saved_data["label"] = watch.gradient;
            ctx->saved_data["want"] = c10::List<bool>({want[0], want[1], want[2], want[3], want[4], want[5], want[6]});
        }
        ctx->set_materialize_grads(false);
        if (f.has_value()) return {*out[0], *out[1]};
        return {*out[1]};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const Tensor dr = grads.size() > 1 ? grads[0] : Tensor(), dy = grads.back();
        variable_list result(13);
        if (!dr.defined() && !dy.defined()) return result;
        const variable_list s = ctx->get_saved_variables();
        const auto settings = ctx->saved_data["settings"].toTuple();
        const auto list = ctx->saved_data["want"].toBoolList();
        const std::vector<bool> want(list.begin(), list.end());
        const auto out = residual_norm_grad(
            opt_of(dr), opt_of(dy), s[0].resolve_neg().contiguous(), opt_of(s[1]), opt_of(s[2]), opt_of(s[3]), opt_of(s[4]),
            opt_of(s[5]), s[6], settings->elements()[0].toBool(), settings->elements()[1].toBool(),
            settings->elements()[2].toDouble(), settings->elements()[3].toDouble(), want,
            ctx->saved_data["cell"].toOptional<Tensor>(), (int)ctx->saved_data["label"].toInt());
        for (int i = 0; i < 7; ++i) result[i] = or_undefined(out[i]);
        differentiable_once(result, "residual_norm");
        return result;
    }
};

// Whether the gate's leading sizes, without 1s at their end, are x's first ones (1s of x that the gate has not are passed
// over), so that every row has a place among the gate's; or x is rows without further structure, which
// the gate takes in runs. Other gates would be read one way by their count and another by broadcasting.
bool gate_lines_up(const Tensor& gate, const Tensor& x) {
    const auto g = gate.sizes(), s = x.sizes();
    size_t n = g.size() - 1, at = 0;
    while (n > 0 && g[n - 1] == 1) --n;
    if (s.size() == 2 && n <= 1) return true;
    for (size_t i = 0; i < n; ++i, ++at) {
        while (at + 1 < s.size() && s[at] == 1 && g[i] != 1) ++at;
        if (at + 1 >= s.size() || s[at] != g[i]) return false;
    }
    return true;
}

// (y) or (r, y), differentiable; x and f of any leading dimensions.
variable_list norm_apply(const Tensor& x, const OptTensor& f, const OptTensor& gate, const OptTensor& post_weight,
                         const OptTensor& post_bias, const OptTensor& weight, const OptTensor& bias, bool rms, bool post,
                         double eps, double scale, const OptTensor& cell, int64_t input_label, int64_t gradient_label) {
    need(x.dim() >= 1 && x.size(-1) >= 1, "norm: x must be [..., values]");
    need(!f.has_value() || f->sizes() == x.sizes(), "norm: f must have x's shape");
    const int64_t d = x.size(-1);
    need(!gate.has_value() || (gate->dim() >= 1 && gate->size(-1) == d), "norm: the gate's last dimension must be x's");
    need(!gate.has_value() || gate_lines_up(*gate, x), "norm: the gate's leading sizes must be x's first ones");
    const std::pair<const OptTensor*, const char*> vectors[] = {
        {&weight, "weight"}, {&bias, "bias"}, {&post_weight, "post_weight"}, {&post_bias, "post_bias"}};
    for (const auto& v : vectors)
        if (v.first->has_value() && !((*v.first)->dim() == 1 && (*v.first)->size(0) == d))
            need(false, std::string("norm: ") + v.second + " must be [" + std::to_string(d) + "]");
    std::vector<bool> want = {at::GradMode::is_enabled() && x.requires_grad()};
    for (const OptTensor* t : {&f, &gate, &post_weight, &post_bias, &weight, &bias})
        want.push_back(at::GradMode::is_enabled() && t->has_value() && (*t)->requires_grad());
    return NormFunction::apply(x, f, gate, post_weight, post_bias, weight, bias, rms, post,
                               eps, scale, Watch{cell, input_label, gradient_label}, want);
}

// ---- cross entropy of a vocabulary projection ----

// {loss, dx, dweight}: x [..., D], weight [V, D], target [...]; a factor for each token or none; what is wanted.
std::vector<OptTensor> linear_cross_entropy(Tensor x, Tensor weight, Tensor target, OptTensor factors_, int S,
                                            int reduction, int64_t ignore_index, bool want_loss, bool want_dx,
                                            bool want_dw) {
    require_f32(x, "x");
    require_f32(weight, "weight");
    const bool gpu = on_gpu(x, weight, "linear_cross_entropy");
    need(target.device() == x.device(), "linear_cross_entropy: tensors must be on the same device");
    need(target.scalar_type() == torch::kInt64, "linear_cross_entropy: target must be int64");
    need(x.dim() >= 1 && weight.dim() == 2 && x.size(-1) == weight.size(1) && target.sizes() == x.sizes().slice(0, x.dim() - 1),
         "linear_cross_entropy: x must be [..., size], weight [words, size], target [...]");
    need(x.size(-1) >= 1 && weight.size(0) >= 1, "linear_cross_entropy: sizes must be positive");
    need(target.numel() <= RG_LOSS_MAX_TOKENS && x.size(-1) <= RG_LOSS_MAX_SIZE && weight.size(0) <= RG_LOSS_MAX_WORDS,
         "linear_cross_entropy: too many tokens, values or words");
    need(S >= 1 && S <= 3, "linear_cross_entropy: slices must be 1..3");
    need(reduction >= RG_LOSS_MEAN && reduction <= RG_LOSS_NONE, "linear_cross_entropy: unknown reduction");
    x = x.resolve_neg().contiguous();
    weight = weight.resolve_neg().contiguous();
    target = target.contiguous();
    Tensor factors;
    if (factors_.has_value()) {
        factors = factors_->resolve_neg().contiguous();
        require_f32(factors, "factors");
        need(factors.device() == x.device() && factors.numel() == target.numel(), "linear_cross_entropy: one factor for each token");
    }
    rg_loss_config c;
    rg_loss_config_init(&c);
    c.N = target.numel();
    c.D = (int)x.size(-1);
    c.V = (int)weight.size(0);
    c.slices = S;
    c.reduction = reduction;
    c.ignore_index = ignore_index;
    Tensor loss, dx, dw;
    if (want_loss) loss = torch::empty(reduction == RG_LOSS_NONE ? target.sizes() : at::IntArrayRef(), x.options());
    if (want_dx) dx = torch::empty_like(x);
    if (want_dw) dw = torch::empty_like(weight);
    const auto* t = target.data_ptr<int64_t>();
    if (gpu) {
        c10::DeviceGuard guard(x.device());
        size_t bytes = 0;
        check(rg_linear_cross_entropy_workspace(&c, want_dx, want_dw, &bytes), "linear cross entropy plan");
        Tensor ws = workspace_like(bytes, x);
        check(rg_linear_cross_entropy(&c, x.data_ptr<float>(), weight.data_ptr<float>(),
                                      reinterpret_cast<const long long*>(t), data_or_null(factors), out_or_null(loss),
                                      out_or_null(dx), out_or_null(dw), ws.data_ptr(), (size_t)ws.numel(), stream_of(x)),
              "linear cross entropy");
    } else {
        Unlocked unlocked;
        repro_loss::cpu_linear_cross_entropy(c, x.data_ptr<float>(), weight.data_ptr<float>(), t, data_or_null(factors),
                                             out_or_null(loss), out_or_null(dx), out_or_null(dw));
    }
    const auto opt = [](const Tensor& v) { return v.defined() ? OptTensor(v) : OptTensor(); };
    return {opt(loss), opt(dx), opt(dw)};
}

// Both (either may be undefined, both contiguous) times factor[0]; no write on a GPU where that is 1.
void scale(const Tensor& a, const Tensor& b, const Tensor& factor) {
    const Tensor& t = a.defined() ? a : b;
    if (!t.defined()) return;
    if (t.is_cuda()) {
        c10::DeviceGuard guard(t.device());
        check(rg_scale_fp32(a.defined() ? a.data_ptr<float>() : nullptr, a.defined() ? a.numel() : 0,
                            b.defined() ? b.data_ptr<float>() : nullptr, b.defined() ? b.numel() : 0,
                            factor.data_ptr<float>(), stream_of(t)),
              "scale");
        return;
    }
    at::NoGradGuard no_grad;
    for (const Tensor* g : {&a, &b})
        if (g->defined()) g->mul_(factor);
}

// The loss, differentiable. With the sum or the mean, the forward pass leaves the gradients in the context
// for the first backward pass to scale and hand out; a later one, and one without a reduction, computes them.
struct LossFunction : torch::autograd::Function<LossFunction> {
    static Tensor forward(AutogradContext* ctx, Tensor x, Tensor weight, Tensor target, int64_t S, int64_t reduction,
                          int64_t ignore_index, OptTensor cell, int64_t label, bool want_x, bool want_w) {
        const bool early = reduction != RG_LOSS_NONE;
        auto out = linear_cross_entropy(x, weight, target, OptTensor(), (int)S, (int)reduction, ignore_index, true,
                                        want_x && early, want_w && early);
        if (want_x || want_w) {
            ctx->save_for_backward({x, weight, target});
            ctx->saved_data["settings"] = std::make_tuple(S, reduction, ignore_index, want_x, want_w);
            ctx->saved_data["cell"] = cell;
            ctx->saved_data["label"] = label;
            ctx->saved_data["ready"] = early;
            if (early) {
                ctx->saved_data["dx"] = out[1];
                ctx->saved_data["dw"] = out[2];
            }
        }
        return *out[0];
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list s = ctx->get_saved_variables();
        const auto settings = ctx->saved_data["settings"].toTuple();
        const auto& e = settings->elements();
        const int S = (int)e[0].toInt(), reduction = (int)e[1].toInt();
        const int64_t ignore_index = e[2].toInt();
        const bool want_x = e[3].toBool(), want_w = e[4].toBool();
        variable_list result(10);
        const auto cell = ctx->saved_data["cell"].toOptional<Tensor>();
        if (cell.has_value()) scan_finite(grads[0].resolve_neg(), *cell, (int)ctx->saved_data["label"].toInt());
        OptTensor dx, dw;
        if (ctx->saved_data["ready"].toBool()) {
            dx = ctx->saved_data["dx"].toOptional<Tensor>();
            dw = ctx->saved_data["dw"].toOptional<Tensor>();
            ctx->saved_data["ready"] = false;
            ctx->saved_data.erase("dx");
            ctx->saved_data.erase("dw");
        } else {
            auto out = linear_cross_entropy(s[0], s[1], s[2], reduction == RG_LOSS_NONE ? OptTensor(grads[0]) : OptTensor(),
                                            S, reduction, ignore_index, false, want_x, want_w);
            dx = out[1];
            dw = out[2];
        }
        result[0] = or_undefined(dx);
        result[1] = or_undefined(dw);
        if (reduction != RG_LOSS_NONE) scale(result[0], result[1], grads[0].resolve_neg().contiguous());
        differentiable_once(result, "linear_cross_entropy");
        return result;
    }
};

// cell and label: where the gradient that arrives reports a NaN or infinity, or nowhere.
Tensor loss_apply(const Tensor& x, const Tensor& weight, const Tensor& target, int64_t S, int64_t reduction,
                  int64_t ignore_index, const OptTensor& cell, int64_t label) {
    const bool grad = at::GradMode::is_enabled();
    return LossFunction::apply(x, weight, target, S, reduction, ignore_index, cell, label, grad && x.requires_grad(),
                               grad && weight.requires_grad());
}

// A leaf keeps the stream that the first graph over it was made on for as long as such a graph lives, and a backward pass
// waits for that stream; one that is being captured cannot wait for a stream outside of its capture, and PyTorch ends the process
// over it. So the forward pass is refused there, where an operand is such a leaf itself.
bool capturing(const Tensor& t, const char* op) {
    if (!at::GradMode::is_enabled() || !t.is_cuda()) return false;
    const hipStream_t stream = c10::hip::getCurrentHIPStream(t.get_device()).stream();
    if (!stream) return false;  // (the default stream cannot be captured)
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    check((int)hipStreamIsCapturing(stream, &status), op);
    return status != hipStreamCaptureStatusNone;
}
void need_capturable(const std::vector<const Tensor*>& operands, const char* op) {
    if (!at::GradMode::is_enabled()) return;
    for (const Tensor* t : operands) {
        if (!t->defined() || !t->is_cuda() || !t->requires_grad() || !t->is_leaf()) continue;
        const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
        if (!node || !node->stream().has_value()) continue;
        if (node->stream()->id() == c10::hip::getCurrentHIPStream(t->get_device()).unwrap().id()) continue;
        need(!capturing(*t, op), std::string(op) + ": a graph over an operand that was made outside of this capture is still alive; free it "
                                                   "before, or capture under torch.no_grad() where no backward pass is wanted");
    }
}

// ---- dropout ----

// A seed: a number, or an int64 tensor of one element on the operands' device, which is read when the kernels run.
struct Seed {
    uint64_t value;
    Tensor at;
};

Seed seed_of(uint64_t value, const OptTensor& at, const Tensor& x, const char* op) {
    if (!at.has_value()) return Seed{value, Tensor()};
    need(at->scalar_type() == torch::kInt64 && at->numel() == 1 && at->device() == x.device(),
         std::string(op) + ": a seed must be a number or an int64 tensor of one element on the operands' device");
    if (x.is_cpu()) return Seed{(uint64_t)at->data_ptr<int64_t>()[0], Tensor()};
    return Seed{0, at->contiguous()};
}
const unsigned long long* seed_data(const Tensor& at) {
    return at.defined() ? reinterpret_cast<const unsigned long long*>(at.data_ptr<int64_t>()) : nullptr;
}

void need_probability(double p, const char* op) {
    need(p >= 0.0 && p < 1.0, std::string(op) + ": the probability to drop must be in [0, 1)");
}

// used, when defined, receives the seed that was read.
Tensor dropout_run(const Tensor& x_, double p, const Seed& seed, const Tensor& used) {
    const Tensor x = x_.resolve_neg().contiguous();
    Tensor y = torch::empty_like(x);
    if (x.is_cuda()) {
        c10::DeviceGuard guard(x.device());
        check(rg_dropout_fp32(x.data_ptr<float>(), y.data_ptr<float>(), (size_t)x.numel(), p, seed.value, seed_data(seed.at),
                              const_cast<unsigned long long*>(seed_data(used)), stream_of(x)),
              "dropout");
    } else {
        Unlocked unlocked;
        repro_dropout::cpu_dropout(x.data_ptr<float>(), y.data_ptr<float>(), (size_t)x.numel(), p, seed.value);
    }
    return y;
}

struct DropoutFunction : torch::autograd::Function<DropoutFunction> {
    static Tensor forward(AutogradContext* ctx, Tensor x, double p, int64_t seed, OptTensor at, bool want) {
        const Seed s = seed_of((uint64_t)seed, at, x, "dropout");
        Tensor used;
        if (want && s.at.defined()) used = torch::empty({1}, s.at.options());
        const Tensor y = dropout_run(x, p, s, used);
        if (want) {
            if (used.defined()) ctx->saved_data["used"] = used;
            ctx->saved_data["seed"] = (int64_t)s.value;
            ctx->saved_data["p"] = p;
        }
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        Seed s{(uint64_t)ctx->saved_data["seed"].toInt(), Tensor()};
        if (ctx->saved_data.count("used")) s.at = ctx->saved_data["used"].toTensor();
        variable_list result(5);
        result[0] = dropout_run(grads[0], ctx->saved_data["p"].toDouble(), s, Tensor());
        differentiable_once(result, "dropout");
        return result;
    }
};

Tensor dropout_apply(const Tensor& x, double p, uint64_t seed, const OptTensor& at) {
    require_f32(x, "x");
    need(x.is_cuda() || x.is_cpu(), "dropout: tensors must be on the CPU or a GPU");
    need_probability(p, "dropout");
    seed_of(seed, at, x, "dropout");
    need_capturable({&x}, "dropout");
    return DropoutFunction::apply(x, p, (int64_t)seed, at, at::GradMode::is_enabled() && x.requires_grad());
}

// ---- attention ----

// [B, T, heads, D] with its values next to each other; any other strides stay.
Tensor attention_operand(const Tensor& t_) {
    const Tensor t = t_.resolve_neg();
    return (t.size(-1) == 1 || t.stride(-1) == 1) && (t.size(1) <= 1 || t.stride(1) <= RG_ATTENTION_MAX_ROW) ? t : t.contiguous();
}
void set_strides(long long* to, const Tensor& t) {
    for (int n = 0; n < 3; ++n) to[n] = t.size(n) > 1 ? t.stride(n) : 0;
}

struct AttentionSettings {
    double scale;
    bool causal;
    int64_t query_start;
    double dropout;
    int64_t seed;
};

rg_attention_config attention_config(const Tensor& q, const Tensor& k, const Tensor& v, const AttentionSettings& s) {
    rg_attention_config c;
    rg_attention_config_init(&c);
    c.B = q.size(0);
    c.Tq = q.size(1);
    c.H = (int)q.size(2);
    c.D = (int)q.size(3);
    c.Tk = k.size(1);
    c.KVH = (int)k.size(2);
    c.causal = s.causal ? 1 : 0;
    c.query_start = s.query_start;
    c.scale = s.scale;
    c.dropout = s.dropout;
    c.seed = (unsigned long long)s.seed;
    set_strides(c.q_stride, q);
    set_strides(c.k_stride, k);
    set_strides(c.v_stride, v);
    return c;
}
// The packed mask's strides; [items, heads, queries, words], sizes 1 shared.
void set_mask(rg_attention_config& c, const Tensor& words) {
    if (!words.defined()) return;
    const long long row = words.size(3);
    const long long strides[3] = {row * words.size(1) * words.size(2), row * words.size(2), row};
    for (int n = 0; n < 3; ++n) c.mask_stride[n] = words.size(n) > 1 ? strides[n] : 0;
}
const unsigned long long* words_or_null(const Tensor& t) {
    return t.defined() ? reinterpret_cast<const unsigned long long*>(t.data_ptr<int64_t>()) : nullptr;
}
const long long* lengths_or_null(const Tensor& t) {
    return t.defined() ? reinterpret_cast<const long long*>(t.data_ptr<int64_t>()) : nullptr;
}

// The mask (bool, broadcast to [B, H, Tq, Tk]) as words of 64 keys.
Tensor packed_mask(const Tensor& mask_, const Tensor& q, int64_t Tk) {
    need(mask_.scalar_type() == torch::kBool && mask_.device() == q.device() && mask_.dim() <= 4,
         "attention: the mask must be bool, on the operands' device, with at most 4 dimensions");
    Tensor mask = mask_;
    while (mask.dim() < 4) mask = mask.unsqueeze(0);
    const int64_t want[4] = {q.size(0), q.size(2), q.size(1), Tk};
    for (int n = 0; n < 4; ++n)
        need(mask.size(n) == want[n] || mask.size(n) == 1, "attention: the mask must broadcast to [batch, heads, queries, keys]");
    const long long stride[3] = {mask.stride(0), mask.stride(1), mask.stride(2)};
    const long long key_stride = mask.size(3) == Tk ? mask.stride(3) : 0;
    Tensor words = torch::empty({mask.size(0), mask.size(1), mask.size(2), (Tk + 63) / 64}, q.options().dtype(torch::kInt64));
    const auto* from = reinterpret_cast<const unsigned char*>(mask.data_ptr<bool>());
    auto* to = reinterpret_cast<unsigned long long*>(words.data_ptr<int64_t>());
    if (words.numel() == 0) return words;
    if (q.is_cuda()) {
        c10::DeviceGuard guard(q.device());
        check(rg_attention_pack_mask(from, mask.size(0), mask.size(1), mask.size(2), Tk, stride, key_stride, to, stream_of(q)),
              "attention mask");
    } else {
        Unlocked unlocked;
        repro_attention::cpu_pack_mask(from, mask.size(0), mask.size(1), mask.size(2), Tk, stride, key_stride, to);
    }
    return words;
}

// The operands are q, k, v and the relative bias; lengths and words prepared by attention_apply.
struct AttentionFunction : torch::autograd::Function<AttentionFunction> {
    static Tensor forward(AutogradContext* ctx, Tensor q_, Tensor k_, Tensor v_, OptTensor bias_, OptTensor lengths,
                          OptTensor words_, AttentionSettings s, OptTensor seed_at, bool want, bool want_bias) {
        const Tensor q = attention_operand(q_), k = attention_operand(k_), v = attention_operand(v_);
        const Tensor bias = bias_.has_value() ? bias_->resolve_neg().contiguous() : Tensor();
        const Tensor words = or_undefined(words_), keys = or_undefined(lengths);
        const Seed seed = seed_of((uint64_t)s.seed, seed_at, q, "attention");
        s.seed = (int64_t)seed.value;
        rg_attention_config c = attention_config(q, k, v, s);
        set_mask(c, words);
        Tensor y = torch::empty(q.sizes(), q.options()), stats, used;
        if (want) stats = torch::empty({c.B, c.H, c.Tq, 2}, q.options());
        if (want && seed.at.defined()) used = torch::empty({1}, seed.at.options());
        if (q.is_cuda()) {
            c10::DeviceGuard guard(q.device());
            size_t bytes = 0;
            check(rg_attention_workspace(&c, words.defined(), &bytes), "attention plan");
            Tensor ws;
            if (bytes > 0) ws = workspace_like(bytes, q);
            check(rg_attention_fp32(&c, q.data_ptr<float>(), k.data_ptr<float>(), v.data_ptr<float>(), lengths_or_null(keys),
                                    words_or_null(words), data_or_null(bias), seed_data(seed.at),
                                    const_cast<unsigned long long*>(seed_data(used)), y.data_ptr<float>(), out_or_null(stats),
                                    bytes > 0 ? ws.data_ptr() : nullptr, bytes, stream_of(q)),
                  "attention");
        } else {
            Unlocked unlocked;
            repro_attention::cpu_attention(c, q.data_ptr<float>(), k.data_ptr<float>(), v.data_ptr<float>(),
                                           lengths_or_null(keys), words_or_null(words), data_or_null(bias),
                                           y.data_ptr<float>(), out_or_null(stats));
        }
        if (want) {
            ctx->save_for_backward({q_, k_, v_, or_undefined(bias_), keys, words, y, stats});
            if (used.defined()) ctx->saved_data["used"] = used;
            ctx->saved_data["settings"] = std::make_tuple(s.scale, s.causal, s.query_start, s.dropout, s.seed, want_bias);
        }
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();
        const auto settings = ctx->saved_data["settings"].toTuple();
        const auto& e = settings->elements();
        const AttentionSettings s{e[0].toDouble(), e[1].toBool(), e[2].toInt(), e[3].toDouble(), e[4].toInt()};
        const bool want_bias = e[5].toBool();
        const Tensor q = attention_operand(saved[0]), k = attention_operand(saved[1]), v = attention_operand(saved[2]);
        const Tensor bias = saved[3].defined() ? saved[3].resolve_neg().contiguous() : Tensor();
        const Tensor &keys = saved[4], &words = saved[5], &y = saved[6], &stats = saved[7];
        const Tensor dy = grads[0].resolve_neg().contiguous();
        Tensor used;
        if (ctx->saved_data.count("used")) used = ctx->saved_data["used"].toTensor();
        rg_attention_config c = attention_config(q, k, v, s);
        set_mask(c, words);
        Tensor dq = torch::empty(q.sizes(), q.options()), dk = torch::empty(k.sizes(), k.options()),
               dv = torch::empty(k.sizes(), k.options()), dbias;
        if (want_bias) dbias = torch::empty(bias.sizes(), bias.options());
        if (q.is_cuda()) {
            c10::DeviceGuard guard(q.device());
            size_t bytes = 0;
            check(rg_attention_grad_workspace(&c, want_bias, &bytes), "attention gradient plan");
            Tensor ws = workspace_like(bytes, q);
            check(rg_attention_grad_fp32(&c, dy.data_ptr<float>(), q.data_ptr<float>(), k.data_ptr<float>(), v.data_ptr<float>(),
                                         lengths_or_null(keys), words_or_null(words), data_or_null(bias), seed_data(used),
                                         y.data_ptr<float>(), stats.data_ptr<float>(), dq.data_ptr<float>(), dk.data_ptr<float>(),
                                         dv.data_ptr<float>(), out_or_null(dbias), ws.data_ptr(), (size_t)ws.numel(),
                                         stream_of(q)),
                  "attention gradient");
        } else {
            Unlocked unlocked;
            repro_attention::cpu_attention_grad(c, dy.data_ptr<float>(), q.data_ptr<float>(), k.data_ptr<float>(),
                                                v.data_ptr<float>(), lengths_or_null(keys), words_or_null(words),
                                                data_or_null(bias), y.data_ptr<float>(), stats.data_ptr<float>(),
                                                dq.data_ptr<float>(), dk.data_ptr<float>(), dv.data_ptr<float>(),
                                                out_or_null(dbias));
        }
        variable_list result(10);
        result[0] = dq;
        result[1] = dk;
        result[2] = dv;
        result[3] = dbias;
        differentiable_once(result, "attention");
        return result;
    }
};

// q [B, Tq, H, D], k and v [B, Tk, KVH, D] -> [B, Tq, H, D], differentiable.
Tensor attention_apply(const Tensor& q, const Tensor& k, const Tensor& v, double scale, bool causal, int64_t query_start,
                       const OptTensor& key_lengths, const OptTensor& mask, const OptTensor& bias, double dropout, uint64_t seed,
                       const OptTensor& seed_at) {
    const std::pair<const Tensor*, const char*> operands[] = {{&q, "q"}, {&k, "k"}, {&v, "v"}};
    for (const auto& t : operands) {
        require_f32(*t.first, t.second);
        if (t.first->dim() != 4) need(false, std::string("attention: ") + t.second + " must be [batch, positions, heads, size]");
    }
    on_gpu(q, k, "attention");
    on_gpu(q, v, "attention");
    need(k.sizes() == v.sizes() && k.size(0) == q.size(0) && k.size(3) == q.size(3),
         "attention: k and v must have one shape, with q's batch and size");
    need(q.size(3) >= 1 && q.size(3) <= RG_ATTENTION_MAX_D, "attention: a head's size must be 1 to 128");
    static_assert(RG_ATTENTION_MAX_D == 128, "the message above");
    need(q.size(2) >= 1 && k.size(2) >= 1 && q.size(2) % k.size(2) == 0, "attention: k's heads must divide q's");
    need(q.size(1) <= RG_ATTENTION_MAX_LENGTH && k.size(1) <= RG_ATTENTION_MAX_LENGTH &&
             q.size(0) * q.size(2) <= RG_ATTENTION_MAX_HEADS && q.size(2) * q.size(3) <= RG_ATTENTION_MAX_ROW && q.size(0) <= RG_ATTENTION_MAX_HEADS,
         "attention: too many positions or heads");
    need(std::isfinite((float)(scale * 1.4426950408889634)), "attention: the scale must be finite");
    need_probability(dropout, "attention");
    seed_of(seed, seed_at, q, "attention");
    const Tensor given_bias = or_undefined(bias);
    need_capturable({&q, &k, &v, &given_bias}, "attention");
    OptTensor lengths, words;
    if (key_lengths.has_value()) {
        need((key_lengths->scalar_type() == torch::kInt64 || key_lengths->scalar_type() == torch::kInt32) &&
                 key_lengths->device() == q.device() && key_lengths->dim() == 1 && key_lengths->size(0) == q.size(0),
             "attention: key_lengths must be int64 or int32 [batch], on the operands' device");
        lengths = key_lengths->to(torch::kInt64).contiguous();
    }
    if (mask.has_value()) words = packed_mask(*mask, q, k.size(1));
    if (bias.has_value()) {
        require_f32(*bias, "relative_bias");
        need(bias->device() == q.device() && bias->dim() == 2 && bias->size(0) == q.size(2) &&
                 bias->size(1) == std::max<int64_t>(q.size(1) + k.size(1) - 1, 0),
             "attention: relative_bias must be [heads, queries + keys - 1], on the operands' device");
    }
    const bool grad = at::GradMode::is_enabled(), want_bias = grad && bias.has_value() && bias->requires_grad();
    const bool want = want_bias || (grad && (q.requires_grad() || k.requires_grad() || v.requires_grad()));
    return AttentionFunction::apply(q, k, v, bias, lengths, words,
                                    AttentionSettings{scale, causal, query_start, dropout, (int64_t)seed}, seed_at, want,
                                    want_bias);
}

// ---- the bias of relative positions ----

rg_relative_bias_config relative_bias_config(int64_t H, int64_t Tq, int64_t Tk, int64_t start, const c10::List<int64_t>& borders,
                                             bool both, bool dense, std::vector<int>& held) {
    for (const int64_t b : borders) held.push_back((int)b);
    rg_relative_bias_config c{};
    c.Tq = Tq;
    c.Tk = Tk;
    c.query_start = start;
    c.H = (int)H;
    c.count = (int)held.size();
    c.both = both ? 1 : 0;
    c.dense = dense ? 1 : 0;
    c.borders = held.data();
    return c;
}

struct RelativeBiasFunction : torch::autograd::Function<RelativeBiasFunction> {
    static Tensor forward(AutogradContext* ctx, Tensor table_, int64_t Tq, int64_t Tk, int64_t start, c10::List<int64_t> borders,
                          bool both, bool dense, bool want) {
        const Tensor table = table_.resolve_neg().contiguous();
        const int64_t H = table.size(1);
        std::vector<int> held;
        const rg_relative_bias_config c = relative_bias_config(H, Tq, Tk, start, borders, both, dense, held);
        Tensor out = dense ? torch::empty({H, Tq, Tk}, table.options())
                           : torch::empty({H, std::max<int64_t>(Tq + Tk - 1, 0)}, table.options());
        if (table.is_cuda()) {
            c10::DeviceGuard guard(table.device());
            check(rg_relative_bias_fp32(&c, table.data_ptr<float>(), out.data_ptr<float>(), stream_of(table)), "relative bias");
        } else if (out.numel() > 0) {
            Unlocked unlocked;
            repro_attention::cpu_relative_bias(c, table.data_ptr<float>(), out.data_ptr<float>());
        }
        if (want) {
            ctx->saved_data["sizes"] = std::make_tuple(H, Tq, Tk, start, both, dense);
            ctx->saved_data["borders"] = borders;
        }
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const Tensor dout = grads[0].resolve_neg().contiguous();
        const auto sizes = ctx->saved_data["sizes"].toTuple();
        const auto& e = sizes->elements();
        const int64_t H = e[0].toInt(), Tq = e[1].toInt(), Tk = e[2].toInt();
        std::vector<int> held;
        const rg_relative_bias_config c = relative_bias_config(H, Tq, Tk, e[3].toInt(), ctx->saved_data["borders"].toIntList(),
                                                               e[4].toBool(), e[5].toBool(), held);
        Tensor dtable = torch::empty({(int64_t)(held.size() + 1) * (c.both ? 2 : 1), H}, dout.options());
        if (dout.is_cuda()) {
            c10::DeviceGuard guard(dout.device());
            size_t bytes = 0;
            check(rg_relative_bias_grad_workspace(&c, &bytes), "relative bias gradient plan");
            Tensor ws = workspace_like(bytes, dout);
            check(rg_relative_bias_grad_fp32(&c, dout.data_ptr<float>(), dtable.data_ptr<float>(), ws.data_ptr(),
                                             (size_t)ws.numel(), stream_of(dout)),
                  "relative bias gradient");
        } else {
            Unlocked unlocked;
            if (dout.numel() > 0) repro_attention::cpu_relative_bias_grad(c, dout.data_ptr<float>(), dtable.data_ptr<float>());
            else dtable.zero_();
        }
        variable_list result(8);
        result[0] = dtable;
        differentiable_once(result, "relative_position_bias");
        return result;
    }
};

// table [buckets, H], the borders between one side's buckets -> [H, Tq, Tk] (dense) or [H, Tq + Tk - 1].
Tensor relative_bias_apply(const Tensor& table, int64_t Tq, int64_t Tk, int64_t start, const std::vector<int64_t>& borders,
                           bool both, bool dense) {
    require_f32(table, "table");
    need(table.is_cuda() || table.is_cpu(), "relative_position_bias: tensors must be on the CPU or a GPU");
    need(!borders.empty() && borders.size() <= RG_RELATIVE_BIAS_MAX_BORDERS && table.dim() == 2 && table.size(1) >= 1 &&
             table.size(0) == (int64_t)(borders.size() + 1) * (both ? 2 : 1),
         "relative_position_bias: the table must be [buckets, heads]");
    need(table.size(1) <= 4096, "relative_position_bias: at most 4096 heads");
    need(Tq >= 0 && Tk >= 0 && Tq <= RG_ATTENTION_MAX_LENGTH && Tk <= RG_ATTENTION_MAX_LENGTH,
         "relative_position_bias: lengths must be 0 to 4194304");
    static_assert(RG_ATTENTION_MAX_LENGTH == 4194304, "the message above");
    need(start >= -(1ll << 32) && start <= (1ll << 32), "relative_position_bias: query_start is out of range");
    need_capturable({&table}, "relative_position_bias");
    return RelativeBiasFunction::apply(table, Tq, Tk, start, c10::List<int64_t>(borders), both, dense,
                                       at::GradMode::is_enabled() && table.requires_grad());
}

}  // namespace

// 64-bit FNV-1a over the raw bytes of a contiguous CPU tensor, continuing from h: the hash the
// reference's tools print for inputs and outputs (repro_test_util.h:20-24,
// gpt2_ops_suite.cu:80-88), so hashes printed here can be compared with theirs.
uint64_t fnv1a64(const at::Tensor& t, uint64_t h) {
    TORCH_CHECK(!t.is_cuda() && t.is_contiguous(), "fnv1a64: a contiguous CPU tensor");
    const unsigned char* p = static_cast<const unsigned char*>(t.data_ptr());
    const size_t n = (size_t)t.numel() * t.element_size();
    for (size_t i = 0; i < n; ++i) {
        h ^= p[i];
        h *= 0x100000001b3ull;
    }
    return h;
}

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.doc() = "Reproducible GEMM, exact sum and convolution on PyTorch tensors (MI355X or CPU)";
    m.def("fnv1a64", &fnv1a64, py::arg("tensor"), py::arg("h") = 0xcbf29ce484222325ull);
    m.def("gemm", &gemm);
    m.def("gemm_ex", &gemm_ex);
    m.def("exact_sum", &exact_sum);
    m.def("conv2d", &conv2d);
    m.def("conv2d_grad_weight", &conv2d_grad_weight);
    m.def("conv2d_grad_input", &conv2d_grad_input);
    m.def("scan_finite", &scan_finite);
    // The layers' forms: the same operations with fewer launches.
    m.def("linear", &linear);
    m.def("conv2d_bias", &conv2d_bias);
    m.def("exact_sum_watch", &exact_sum_watch);
    m.def("scan_finite_pair", &scan_finite_pair);
    m.def("adamw_step", &adamw_step);
    m.def("adamw8_step", &adamw8_step);
    m.def("adamw8_values", &adamw8_values);
    m.def("norm_apply", &norm_apply);
    m.def("loss_apply", &loss_apply);
    m.def("capturing", [](const Tensor& t) { return capturing(t, "capture"); });
    m.def("need_capturable", [](const std::vector<Tensor>& operands, const std::string& op) {
        std::vector<const Tensor*> each;
        for (const Tensor& t : operands) each.push_back(&t);
        need_capturable(each, op.c_str());
    });
    m.def("dropout_apply", &dropout_apply);
    m.def("attention_apply", &attention_apply);
    m.def("relative_bias_apply", &relative_bias_apply);
    m.def("cpu_threads", &repro_gemm::cpu_thread_count);
    m.def("set_error_class", [](py::object cls) {
        Py_XINCREF(cls.ptr());
        Py_XDECREF(g_error_class);
        g_error_class = cls.ptr();
    });
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const LibraryError& e) {
            if (!g_error_class) {
                PyErr_SetString(PyExc_RuntimeError, (e.message + ": hip error " + std::to_string(e.code)).c_str());
                return;
            }
            PyObject* err = PyObject_CallFunction(g_error_class, "is", e.code, e.what());
            if (err) {
                PyErr_SetObject(g_error_class, err);
                Py_DECREF(err);
            }
        }
    });
    m.attr("has_cuda") = true;
}

// torch_ops_layers.cpp -- torch.ops.pma.* of the gated recurrence, the sampler and the 8-bit linear
// product, over the C ABI of include/pma.h.
//
//   pma::gated_scan(x, f, bias?, gate?, h0?, reset?) -> (y, h)                 differentiable, through
//     pma::gated_scan_forward (which returns its workspace too) and pma::gated_scan_backward
//   pma::gated_scan_step(x, f, h, bias?, gate?) -> (y, new h)
//   pma::gated_scan_step_(x, f, h(a!), bias?, gate?, rows?) -> y               h (or its rows) updated
//   pma::sample(logits, u, temperature?, top_k?, top_p?, min_p?, t, k, p, m) -> (tokens, logprobs)
//   pma::fp8_linear(x, wq, ws, out_dtype) -> y
//
// Arguments are checked here; the Python modules (recurrence, sampling, fp8) document them.
//
// The same functions are the Python extension module _pma_torch (this library, imported): a call
// there skips the dispatcher's argument boxing.  A small call's time is host time: a 64 x 768 step
// takes 6 us so, 9 through torch.ops, 25 through ctypes.  Calls with anything but plain tensors, or
// under a dispatch mode, a tracer or a function transform, return NotImplemented, and the modules go
// through torch.ops.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>
#include <torch/library.h>

#include <atomic>
#include <optional>
#include <string>
#include <tuple>

#include "../../include/pma.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

void check_rc(int rc, const char *fn) {
    if (rc == PMA_OK) return;
    std::string msg = std::string(fn) + " failed: " + pma_status_string(rc);
    if (rc == PMA_ERR_CUDA) msg += std::string(": ") + pma_cuda_error_string(pma_last_cuda_error());
    TORCH_CHECK(false, msg);
}

// The fault word as the host reads it (watch_faults; pinned host memory).  The operators whose kernels wait
// look at it: calls of a compiled program pass by the Python layer's check.
std::atomic<int *> g_watched{nullptr};

void check_faults(const char *fn) {
    int *word = g_watched.load(std::memory_order_acquire);
    if (!word) return;
    const int code = *static_cast<volatile int *>(word);
    if (code == 0) return;
    *static_cast<volatile int *>(word) = 0;
    TORCH_CHECK(false, fn, ": an earlier launch recorded fault code ", code,
                " (a bounded wait expired; its outputs are void)");
}

int dtype_of(const Tensor &t) {
    if (t.scalar_type() == at::kFloat) return PMA_F32;
    TORCH_CHECK_TYPE(t.scalar_type() == at::kBFloat16, "unsupported dtype ", t.scalar_type(), ": float32 or bfloat16");
    return PMA_BF16;
}

void check_cuda(const Tensor &t, const char *name) {
    TORCH_CHECK(t.is_cuda(), "pma: ", name, " must be a CUDA tensor (no CPU fallback)");
}

// Nothing here has a forward-mode derivative: a dual operand is refused, not stripped of its tangent.
void check_no_tangent(const char *fn, std::initializer_list<const Tensor *> ts) {
    for (const Tensor *t : ts)
        TORCH_CHECK(!t || !t->defined() || !t->_fw_grad(/*level=*/0).defined(), fn, " has no forward-mode derivative");
}
const Tensor *ptr_of(const OptTensor &t) { return t ? &*t : nullptr; }

// The operators without a gradient say so instead of dropping it.
void check_no_grad(const char *fn, std::initializer_list<const Tensor *> ts) {
    check_no_tangent(fn, ts);
    if (!at::GradMode::is_enabled()) return;
    for (const Tensor *t : ts)
        TORCH_CHECK(!t || !t->requires_grad(), fn, " is inference-only: run under torch.no_grad() or torch.inference_mode()");
}

void check_like(const Tensor &t, const char *name, at::IntArrayRef shape, at::ScalarType dtype, const at::Device &dev) {
    TORCH_CHECK_VALUE(t.sizes() == shape && t.scalar_type() == dtype && t.device() == dev, name, " must be a ", dtype,
                      " tensor of shape ", shape, " on ", dev, "; got ", t.scalar_type(), " ", t.sizes(), " on ",
                      t.device());
}

pma_stream_t stream_of(const at::Device &dev) {
    return reinterpret_cast<pma_stream_t>(at::cuda::getCurrentCUDAStream(dev.index()).stream());
}

int int_of(int64_t v, const char *name) {
    TORCH_CHECK_VALUE(v <= 0x7fffffff, name, " is too large: ", v);
    return (int)v;
}

// ----------------------------------------------------------------------------------- recurrence
// The channel axis contiguous (a copy only where it is not).
Tensor rows_ok(const Tensor &t) { return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous(); }

struct View {  // pma_seq_tensor of [B, L, C] or [N, C]; null for an absent tensor
    pma_seq_tensor s{};
    bool on = false;
    View() = default;
    explicit View(const Tensor &t) : on(true) {
        s.data = t.data_ptr();
        s.dtype = dtype_of(t);
        s.stride_b = t.stride(0);
        s.stride_l = t.dim() == 3 ? t.stride(1) : 0;
    }
    explicit View(const OptTensor &t) {
        if (t) *this = View(*t);
    }
    const pma_seq_tensor *get() const { return on ? &s : nullptr; }
};
template <typename T> T *ptr(const OptTensor &t) { return t ? static_cast<T *>(t->data_ptr()) : nullptr; }

// Arguments as the kernels take them.
struct ScanArgs {
    Tensor x, f;
    OptTensor bias, gate, h0, reset;
    int B = 0, L = 0, C = 0;
};

void check_common(const Tensor &x, const Tensor &f, const OptTensor &bias, const OptTensor &gate, int64_t dims) {
    check_cuda(x, "x");
    check_cuda(f, "f");
    TORCH_CHECK_VALUE(x.dim() == dims, "x must have ", dims, " axes; got shape ", x.sizes());
    dtype_of(x);
    TORCH_CHECK_VALUE(x.size(-1) > 0, "x must have at least one channel");
    check_like(f, "f", x.sizes(), x.scalar_type(), x.device());
    if (gate) check_like(*gate, "gate", x.sizes(), x.scalar_type(), x.device());
    if (bias) check_like(*bias, "bias", {x.size(-1)}, at::kFloat, x.device());
}

OptTensor contiguous(const OptTensor &t) { return t ? OptTensor(t->contiguous()) : t; }
OptTensor rows_ok(const OptTensor &t) { return t ? OptTensor(rows_ok(*t)) : t; }

ScanArgs scan_args(const Tensor &x, const Tensor &f, const OptTensor &bias, const OptTensor &gate, const OptTensor &h0,
                   const OptTensor &reset) {
    check_common(x, f, bias, gate, 3);
    ScanArgs a;
    a.B = int_of(x.size(0), "batch");
    a.L = int_of(x.size(1), "length");
    a.C = int_of(x.size(2), "channels");
    if (h0) check_like(*h0, "h0", {a.B, a.C}, at::kFloat, x.device());
    if (reset) {
        TORCH_CHECK_TYPE(reset->scalar_type() == at::kBool || reset->scalar_type() == at::kByte,
                         "reset must be a bool or uint8 tensor");
        check_like(*reset, "reset", {a.B, a.L}, reset->scalar_type(), x.device());
    }
    a.x = rows_ok(x);
    a.f = rows_ok(f);
    a.gate = rows_ok(gate);
    a.bias = contiguous(bias);
    a.h0 = contiguous(h0);
    a.reset = contiguous(reset);
    return a;
}

std::tuple<Tensor, Tensor, Tensor> scan_forward(const Tensor &x_in, const Tensor &f_in, const OptTensor &bias,
                                                const OptTensor &gate, const OptTensor &h0, const OptTensor &reset) {
    check_faults("gated_scan");
    const ScanArgs a = scan_args(x_in, f_in, bias, gate, h0, reset);
    const at::Device dev = a.x.device();
    const c10::cuda::CUDAGuard guard(dev);
    Tensor y = at::empty({a.B, a.L, a.C}, a.x.options());
    Tensor h = at::empty({a.B, a.C}, a.x.options().dtype(at::kFloat));
    const size_t n = pma_gated_scan_workspace_bytes(a.B, a.L, a.C);
    Tensor ws = at::empty({(int64_t)n}, a.x.options().dtype(at::kByte));
    const View x(a.x), f(a.f), g(a.gate), yv(y);
    check_rc(pma_gated_scan(a.B, a.L, a.C, x.get(), f.get(), g.get(), ptr<float>(a.bias), ptr<float>(a.h0),
                            ptr<uint8_t>(a.reset), yv.get(), h.data_ptr<float>(), n ? ws.data_ptr() : nullptr, n,
                            stream_of(dev)),
             "pma_gated_scan");
    return {y, h, ws};
}

// Gradients (dx, df, dbias, dgate, dh0); the last three are empty tensors where they are not wanted.
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> scan_backward(const Tensor &x_in, const Tensor &f_in,
                                                                 const OptTensor &bias, const OptTensor &gate,
                                                                 const OptTensor &h0, const OptTensor &reset,
                                                                 const Tensor &ws, const OptTensor &dy_in,
                                                                 const OptTensor &dh_in, bool want_bias, bool want_h0) {
    check_faults("gated_scan_backward");
    const ScanArgs a = scan_args(x_in, f_in, bias, gate, h0, reset);
    const at::Device dev = a.x.device();
    const c10::cuda::CUDAGuard guard(dev);
    const int B = a.B, L = a.L, C = a.C;
    if (dy_in) check_like(*dy_in, "dy", {B, L, C}, a.x.scalar_type(), dev);
    if (dh_in) check_like(*dh_in, "dh", {B, C}, at::kFloat, dev);
    const Tensor dy = dy_in ? rows_ok(*dy_in) : at::zeros({1, 1, C}, a.x.options()).expand({B, L, C});
    const OptTensor dh = contiguous(dh_in);
    const auto f32 = a.x.options().dtype(at::kFloat);
    Tensor dx = at::empty({B, L, C}, a.x.options()), df = at::empty({B, L, C}, a.x.options());
    Tensor dg = gate ? at::empty({B, L, C}, a.x.options()) : at::empty({0}, a.x.options());
    Tensor db = want_bias ? at::empty({C}, f32) : at::empty({0}, f32);
    Tensor d0 = want_h0 ? at::empty({B, C}, f32) : at::empty({0}, f32);
    const size_t n = pma_gated_scan_backward_workspace_bytes(B, L, C);
    Tensor w2 = at::empty({(int64_t)std::max<size_t>(n, 1)}, a.x.options().dtype(at::kByte));
    const View xv(a.x), fv(a.f), gv(a.gate), dyv(dy), dxv(dx), dfv(df), dgv = gate ? View(dg) : View();
    check_rc(pma_gated_scan_backward(B, L, C, xv.get(), fv.get(), gv.get(), ptr<float>(a.bias), ptr<float>(a.h0),
                                     ptr<uint8_t>(a.reset), dyv.get(), ptr<float>(dh), dxv.get(), dfv.get(), dgv.get(),
                                     want_bias ? db.data_ptr<float>() : nullptr, want_h0 ? d0.data_ptr<float>() : nullptr,
                                     ws.numel() ? ws.data_ptr() : nullptr, (size_t)ws.numel(), w2.data_ptr(), n,
                                     stream_of(dev)),
             "pma_gated_scan_backward");
    return {dx, df, db, dg, d0};
}

std::tuple<Tensor, Tensor> gated_scan(const Tensor &x, const Tensor &f, const OptTensor &bias, const OptTensor &gate,
                                      const OptTensor &h0, const OptTensor &reset) {
    auto [y, h, ws] = scan_forward(x, f, bias, gate, h0, reset);
    return {y, h};
}

// The calls below go through the dispatcher, so that tracing sees operators with shape functions.
struct ScanFunction : torch::autograd::Function<ScanFunction> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext *ctx, const Tensor &x, const Tensor &f,
                                                  const OptTensor &bias, const OptTensor &gate, const OptTensor &h0,
                                                  const OptTensor &reset) {
        at::AutoDispatchBelowADInplaceOrView below;
        static const auto op = c10::Dispatcher::singleton()
                                   .findSchemaOrThrow("pma::gated_scan_forward", "")
                                   .typed<std::tuple<Tensor, Tensor, Tensor>(const Tensor &, const Tensor &, const OptTensor &,
                                                                             const OptTensor &, const OptTensor &,
                                                                             const OptTensor &)>();
        auto [y, h, ws] = op.call(x, f, bias, gate, h0, reset);
        auto or_none = [](const OptTensor &t) { return t ? *t : Tensor(); };
        ctx->save_for_backward({x, f, or_none(bias), or_none(gate), or_none(h0), or_none(reset), ws});
        ctx->saved_data["want"] = (bias && bias->requires_grad() ? 1 : 0) + (h0 && h0->requires_grad() ? 2 : 0);
        ctx->set_materialize_grads(false);
        return {y, h};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx,
                                                   torch::autograd::variable_list grads) {
        // create_graph: the gradients depend on the inputs, whatever the incoming ones depend on
        TORCH_CHECK(!at::GradMode::is_enabled(), "gated_scan is not twice differentiable");
        const auto saved = ctx->get_saved_variables();
        auto opt = [&](int i) { return saved[i].defined() ? OptTensor(saved[i]) : OptTensor(); };
        auto given = [&](int i) { return grads[i].defined() ? OptTensor(grads[i]) : OptTensor(); };
        const int64_t want = ctx->saved_data["want"].toInt();
        at::AutoDispatchBelowADInplaceOrView below;
        static const auto op =
            c10::Dispatcher::singleton()
                .findSchemaOrThrow("pma::gated_scan_backward", "")
                .typed<std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>(
                    const Tensor &, const Tensor &, const OptTensor &, const OptTensor &, const OptTensor &,
                    const OptTensor &, const Tensor &, const OptTensor &, const OptTensor &, bool, bool)>();
        auto [dx, df, db, dg, d0] = op.call(saved[0], saved[1], opt(2), opt(3), opt(4), opt(5), saved[6], given(0), given(1),
                                            want & 1, (want & 2) != 0);
        return {dx, df, want & 1 ? db : Tensor(), saved[3].defined() ? dg : Tensor(), want & 2 ? d0 : Tensor(), Tensor()};
    }
};

std::tuple<Tensor, Tensor> gated_scan_autograd(const Tensor &x, const Tensor &f, const OptTensor &bias,
                                               const OptTensor &gate, const OptTensor &h0, const OptTensor &reset) {
    check_no_tangent("gated_scan", {&x, &f, ptr_of(bias), ptr_of(gate), ptr_of(h0)});
    auto needs = [](const OptTensor &t) { return t && t->requires_grad(); };
    if (at::GradMode::is_enabled() &&
        (x.requires_grad() || f.requires_grad() || needs(bias) || needs(gate) || needs(h0))) {
        const auto out = ScanFunction::apply(x, f, bias, gate, h0, reset);
        return {out[0], out[1]};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = c10::Dispatcher::singleton()
                               .findSchemaOrThrow("pma::gated_scan", "")
                               .typed<std::tuple<Tensor, Tensor>(const Tensor &, const Tensor &, const OptTensor &,
                                                                 const OptTensor &, const OptTensor &, const OptTensor &)>();
    return op.call(x, f, bias, gate, h0, reset);
}

Tensor step_into(const Tensor &x_in, const Tensor &f_in, const Tensor &h_in, const Tensor &h_out, const OptTensor &bias_in,
                 const OptTensor &gate_in, const OptTensor &rows_in) {
    const at::Device dev = x_in.device();
    const c10::cuda::CUDAGuard guard(dev);
    const Tensor x = rows_ok(x_in), f = rows_ok(f_in);
    const OptTensor gate = rows_ok(gate_in), bias = contiguous(bias_in), rows = contiguous(rows_in);
    const int N = int_of(x.size(0), "rows"), C = int_of(x.size(1), "channels");
    Tensor y = at::empty({N, C}, x.options());
    const View xv(x), fv(f), gv(gate), yv(y);
    check_rc(pma_gated_scan_step(N, C, xv.get(), fv.get(), gv.get(), ptr<float>(bias), h_in.data_ptr<float>(),
                                 h_out.data_ptr<float>(), ptr<int32_t>(rows), int_of(h_in.size(0), "pool rows"), yv.get(),
                                 stream_of(dev)),
             "pma_gated_scan_step");
    return y;
}

std::tuple<Tensor, Tensor> gated_scan_step(const Tensor &x, const Tensor &f, const Tensor &h, const OptTensor &bias,
                                           const OptTensor &gate) {
    check_common(x, f, bias, gate, 2);
    check_no_grad("gated_scan_step", {&x, &f, &h, ptr_of(bias), ptr_of(gate)});
    check_like(h, "h", x.sizes(), at::kFloat, x.device());
    const Tensor in = h.contiguous();
    Tensor out = at::empty_like(in);
    Tensor y = step_into(x, f, in, out, bias, gate, std::nullopt);
    return {y, out};
}

Tensor gated_scan_step_(const Tensor &x, const Tensor &f, const Tensor &h, const OptTensor &bias, const OptTensor &gate,
                        const OptTensor &rows) {
    check_common(x, f, bias, gate, 2);
    check_no_grad("gated_scan_step", {&x, &f, &h, ptr_of(bias), ptr_of(gate)});
    if (rows) {
        check_like(*rows, "rows", {x.size(0)}, at::kInt, x.device());
        TORCH_CHECK_VALUE(h.dim() == 2, "h must be [pool rows, channels]");
        check_like(h, "h", {h.size(0), x.size(1)}, at::kFloat, x.device());
    } else {
        check_like(h, "h", x.sizes(), at::kFloat, x.device());
    }
    TORCH_CHECK_VALUE(h.is_contiguous(), "h must be contiguous to be updated in place");
    return step_into(x, f, h, h, bias, gate, rows);
}

// -------------------------------------------------------------------------------------- sampler
std::tuple<Tensor, Tensor> sample(const Tensor &logits_in, const Tensor &u_in, const OptTensor &temperature,
                                  const OptTensor &top_k, const OptTensor &top_p, const OptTensor &min_p, double t,
                                  int64_t k, double p, double m) {
    check_cuda(logits_in, "logits");
    check_cuda(u_in, "u");
    TORCH_CHECK_VALUE(logits_in.dim() == 2, "logits must be [B, V]; got ", logits_in.sizes());
    const at::Device dev = logits_in.device();
    const int dtype = dtype_of(logits_in);
    const int64_t B = logits_in.size(0), V = logits_in.size(1);
    TORCH_CHECK_VALUE(V >= 1 && V <= 360448, "logits must have 1 to 360448 columns; got ", V);
    check_like(u_in, "u", {B}, at::kFloat, dev);
    if (temperature) check_like(*temperature, "temperature", {B}, at::kFloat, dev);
    if (top_k) check_like(*top_k, "top_k", {B}, at::kInt, dev);
    if (top_p) check_like(*top_p, "top_p", {B}, at::kFloat, dev);
    if (min_p) check_like(*min_p, "min_p", {B}, at::kFloat, dev);
    const c10::cuda::CUDAGuard guard(dev);
    const Tensor logits = (V > 1 && logits_in.stride(1) != 1) || (B > 1 && logits_in.stride(0) < V) ? logits_in.contiguous()
                                                                                               : logits_in;
    const Tensor u = u_in.contiguous();
    const OptTensor ct = contiguous(temperature), ck = contiguous(top_k), cp = contiguous(top_p), cm = contiguous(min_p);
    Tensor tokens = at::empty({B}, u.options().dtype(at::kLong)), logprobs = at::empty({B}, u.options());
    const int kv = (int)std::min<int64_t>(std::max<int64_t>(k, 0), 0x7fffffff);
    check_rc(pma_sample(int_of(B, "batch"), (int)V, logits.data_ptr(), logits.stride(0), dtype, u.data_ptr<float>(),
                        ptr<float>(ct), (float)t, ptr<int32_t>(ck), kv, ptr<float>(cp), (float)p, ptr<float>(cm), (float)m,
                        tokens.data_ptr<int64_t>(), logprobs.data_ptr<float>(), stream_of(dev)),
             "pma_sample");
    return {tokens, logprobs};
}

// --------------------------------------------------------------------------------- 8-bit linear
Tensor fp8_linear(const Tensor &x_in, const Tensor &wq_in, const Tensor &ws_in, at::ScalarType out_dtype) {
    check_cuda(x_in, "x");
    check_cuda(wq_in, "wq");
    check_cuda(ws_in, "ws");
    check_no_grad("fp8_linear", {&x_in, &ws_in});
    check_faults("fp8_linear");
    TORCH_CHECK_VALUE(x_in.dim() >= 1 && x_in.size(-1) > 0, "x must have at least one column; got ", x_in.sizes());
    const at::Device dev = x_in.device();
    const int dtype = dtype_of(x_in);
    const int64_t K = x_in.size(-1);
    TORCH_CHECK_VALUE(wq_in.dim() == 2 && wq_in.scalar_type() == at::kFloat8_e4m3fn && wq_in.size(1) == K &&
                          wq_in.device() == dev,
                      "wq must be a [rows, ", K, "] float8_e4m3fn tensor on ", dev);
    TORCH_CHECK_TYPE(out_dtype == at::kFloat || out_dtype == at::kBFloat16, "unsupported dtype ", out_dtype,
                     ": float32 or bfloat16");
    const int64_t N = wq_in.size(0), nb = (N + 127) / 128, kb = (K + 127) / 128;
    check_like(ws_in, "ws", {nb, kb}, at::kFloat, dev);
    const c10::cuda::CUDAGuard guard(dev);
    std::vector<int64_t> shape = x_in.sizes().vec();
    shape.back() = N;
    Tensor x = x_in.dim() == 2 ? x_in : x_in.reshape({-1, K});
    const int64_t M = x.size(0);
    if ((K > 1 && x.stride(1) != 1) || (M > 1 && x.stride(0) < K)) x = x.contiguous();
    Tensor y = at::empty(shape, x.options().dtype(out_dtype));
    if (M == 0 || N == 0) return y;
    Tensor wq = wq_in;
    if (wq.stride(1) != 1 || wq.stride(0) % 16 || wq.stride(0) < K || reinterpret_cast<uintptr_t>(wq.data_ptr()) % 16) {
        wq = at::empty({N, (K + 15) / 16 * 16}, wq_in.options()).narrow(1, 0, K);
        wq.copy_(wq_in);
    }
    // the kernel takes a row stride of at least kb: a broadcast or overlapping view becomes an array of its own
    const bool as_is = (kb == 1 || ws_in.stride(1) == 1) && (nb == 1 || ws_in.stride(0) >= kb);
    const Tensor ws = as_is ? ws_in : ws_in.contiguous();
    const int Mi = int_of(M, "rows"), Ni = int_of(N, "outputs"), Ki = int_of(K, "columns");
    const size_t n = pma_fp8_linear_workspace_bytes(Mi, Ki);
    Tensor scratch = at::empty({(int64_t)n}, x.options().dtype(at::kByte));
    check_rc(pma_fp8_linear(Mi, Ni, Ki, x.data_ptr(), x.stride(0), dtype, wq.data_ptr(), wq.stride(0),
                            ws.data_ptr<float>(), nb == 1 ? kb : ws.stride(0), y.data_ptr(), N, dtype_of(y),
                            scratch.data_ptr(), n, stream_of(dev)),
             "pma_fp8_linear");
    return y;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(pma, m) {
    m.def("gated_scan(Tensor x, Tensor f, Tensor? bias=None, Tensor? gate=None, Tensor? h0=None, Tensor? reset=None) -> "
          "(Tensor, Tensor)");
    m.def("gated_scan_forward(Tensor x, Tensor f, Tensor? bias, Tensor? gate, Tensor? h0, Tensor? reset) -> "
          "(Tensor, Tensor, Tensor)");
    m.def("gated_scan_backward(Tensor x, Tensor f, Tensor? bias, Tensor? gate, Tensor? h0, Tensor? reset, Tensor ws, "
          "Tensor? dy, Tensor? dh, bool want_bias, bool want_h0) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
    m.def("gated_scan_step(Tensor x, Tensor f, Tensor h, Tensor? bias=None, Tensor? gate=None) -> (Tensor, Tensor)");
    m.def("gated_scan_step_(Tensor x, Tensor f, Tensor(a!) h, Tensor? bias=None, Tensor? gate=None, Tensor? rows=None) "
          "-> Tensor");
    m.def("sample(Tensor logits, Tensor u, Tensor? temperature=None, Tensor? top_k=None, Tensor? top_p=None, "
          "Tensor? min_p=None, float t=1.0, int k=0, float p=1.0, float m=0.0) -> (Tensor, Tensor)");
    m.def("fp8_linear(Tensor x, Tensor wq, Tensor ws, ScalarType out_dtype) -> Tensor");
}

TORCH_LIBRARY_IMPL(pma, CUDA, m) {
    m.impl("gated_scan", &gated_scan);
    m.impl("gated_scan_forward", &scan_forward);
    m.impl("gated_scan_backward", &scan_backward);
    m.impl("gated_scan_step", &gated_scan_step);
    m.impl("gated_scan_step_", &gated_scan_step_);
    m.impl("sample", &sample);
    m.impl("fp8_linear", &fp8_linear);
}

TORCH_LIBRARY_IMPL(pma, Autograd, m) { m.impl("gated_scan", &gated_scan_autograd); }

// ------------------------------------------------------------------------------ Python extension
namespace {

// Plain tensors (or None where `optional`), no dispatch mode, no tracer and no function transform: otherwise
// the dispatcher's business (a tracer would see the results as constants).
struct Args {
    PyObject *const *a;
    bool plain = true;
    explicit Args(PyObject *const *args) : a(args) {
        constexpr c10::DispatchKeySet above{c10::DispatchKey::Tracer, c10::DispatchKey::FuncTorchDynamicLayerFrontMode};
        plain = !c10::impl::TorchDispatchModeTLS::any_modes_set() &&
                !c10::impl::tls_local_dispatch_key_set().included_.has_any(above);
    }
    const Tensor &tensor(int i) {
        static const Tensor none;
        if (!THPVariable_CheckExact(a[i]) && !Py_IS_TYPE(a[i], reinterpret_cast<PyTypeObject *>(ParameterClass))) {
            plain = false;
            return none;
        }
        return THPVariable_Unpack(a[i]);
    }
    OptTensor opt(int i) { return a[i] == Py_None ? OptTensor() : OptTensor(tensor(i)); }
    double number(int i) {
        const double v = PyFloat_AsDouble(a[i]);
        if (v == -1.0 && PyErr_Occurred()) throw python_error();
        return v;
    }
    int64_t whole(int i) {
        const int64_t v = PyLong_AsLongLong(a[i]);
        if (v == -1 && PyErr_Occurred()) throw python_error();
        return v;
    }
};

PyObject *wrap(const Tensor &t) { return THPVariable_Wrap(t); }
PyObject *wrap(const std::tuple<Tensor, Tensor> &t) {
    THPObjectPtr a(THPVariable_Wrap(std::get<0>(t))), b(THPVariable_Wrap(std::get<1>(t)));
    return PyTuple_Pack(2, a.get(), b.get());
}
PyObject *not_here() { Py_RETURN_NOTIMPLEMENTED; }

bool count_is(Py_ssize_t n, Py_ssize_t want) {
    if (n == want) return true;
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
    return false;
}

// gated_scan(x, f, bias, gate, h0, reset)
PyObject *py_gated_scan(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!count_is(n, 6)) return nullptr;
    Args a(args);
    const Tensor &x = a.tensor(0), &f = a.tensor(1);
    const OptTensor bias = a.opt(2), gate = a.opt(3), h0 = a.opt(4), reset = a.opt(5);
    if (!a.plain) return not_here();
    check_no_tangent("gated_scan", {&x, &f, ptr_of(bias), ptr_of(gate), ptr_of(h0)});
    auto needs = [](const OptTensor &t) { return t && t->requires_grad(); };
    if (at::GradMode::is_enabled() &&
        (x.requires_grad() || f.requires_grad() || needs(bias) || needs(gate) || needs(h0))) {
        const auto out = ScanFunction::apply(x, f, bias, gate, h0, reset);
        return wrap(std::make_tuple(out[0], out[1]));
    }
    at::AutoDispatchBelowADInplaceOrView below;
    return wrap(gated_scan(x, f, bias, gate, h0, reset));
    END_HANDLE_TH_ERRORS
}

// gated_scan_step(x, f, h, bias, gate) and gated_scan_step_(x, f, h, bias, gate, rows)
PyObject *py_step(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!count_is(n, 5)) return nullptr;
    Args a(args);
    const Tensor &x = a.tensor(0), &f = a.tensor(1), &h = a.tensor(2);
    const OptTensor bias = a.opt(3), gate = a.opt(4);
    if (!a.plain) return not_here();
    at::AutoDispatchBelowADInplaceOrView below;
    return wrap(gated_scan_step(x, f, h, bias, gate));
    END_HANDLE_TH_ERRORS
}
PyObject *py_step_(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!count_is(n, 6)) return nullptr;
    Args a(args);
    const Tensor &x = a.tensor(0), &f = a.tensor(1), &h = a.tensor(2);
    const OptTensor bias = a.opt(3), gate = a.opt(4), rows = a.opt(5);
    if (!a.plain) return not_here();
    at::AutoDispatchBelowADInplaceOrView below;
    return wrap(gated_scan_step_(x, f, h, bias, gate, rows));
    END_HANDLE_TH_ERRORS
}

// sample(logits, u, temperature, top_k, top_p, min_p): each setting a number or a tensor
PyObject *py_sample(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!count_is(n, 6)) return nullptr;
    Args a(args);
    const Tensor &logits = a.tensor(0), &u = a.tensor(1);
    OptTensor rows[4];
    double value[4] = {0, 0, 0, 0};
    int64_t top_k = 0;
    for (int i = 0; i < 4; ++i) {
        if (THPVariable_Check(args[2 + i]))
            rows[i] = a.tensor(2 + i);
        else if (i == 1)
            top_k = a.whole(2 + i);
        else
            value[i] = a.number(2 + i);
    }
    if (!a.plain) return not_here();
    at::AutoDispatchBelowADInplaceOrView below;
    return wrap(sample(logits, u, rows[0], rows[1], rows[2], rows[3], value[0], top_k, value[2], value[3]));
    END_HANDLE_TH_ERRORS
}

// fp8_linear(x, wq, ws, float32?)
PyObject *py_fp8_linear(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!count_is(n, 4)) return nullptr;
    Args a(args);
    const Tensor &x = a.tensor(0), &wq = a.tensor(1), &ws = a.tensor(2);
    if (!a.plain) return not_here();
    at::AutoDispatchBelowADInplaceOrView below;
    return wrap(fp8_linear(x, wq, ws, args[3] == Py_True ? at::kFloat : at::kBFloat16));
    END_HANDLE_TH_ERRORS
}

// watch_faults(address of the pinned host int that is registered as the fault word)
PyObject *py_watch_faults(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!count_is(n, 1)) return nullptr;
    void *word = PyLong_AsVoidPtr(args[0]);
    if (!word && PyErr_Occurred()) throw python_error();
    g_watched.store(static_cast<int *>(word), std::memory_order_release);
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

#define PMA_FAST(name, fn) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(fn)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {PMA_FAST("gated_scan", py_gated_scan), PMA_FAST("gated_scan_step", py_step),
                         PMA_FAST("gated_scan_step_", py_step_), PMA_FAST("sample", py_sample),
                         PMA_FAST("fp8_linear", py_fp8_linear), PMA_FAST("watch_faults", py_watch_faults), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_pma_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject *PyInit__pma_torch(void) { return PyModule_Create(&module); }

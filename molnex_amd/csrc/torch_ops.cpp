// torch.ops.molix.layer_norm* and the AdamW ops, registered in C++ over the C ABI of include/molnex.h.
//
// These are called once or more per layer and step, on tensors small enough that the host bounds them, and AdamW's
// arguments are lists of every parameter.  Registered from Python (molnex_amd/_ops.py), a 700 x 128 layer norm forward
// and backward took 179 us, most of it the autograd engine's thread and the caller passing the interpreter's lock to
// and fro, and a step over 60 tensors 119 us, the time to ask each tensor its type, layout and address.  The library
// is a Python module too, whose functions take the lists of tensors straight to the ops: through torch.ops, each of
// 300 tensors is boxed first (a step over 60 tensors of 3.2 M elements took 40 us so, 26 us now), and a layer norm's
// arguments are looked at in Python (96 x 128: 7.6 us, 5.2 us now).
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/autocast_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/library.h>

#include <algorithm>
#include <cmath>
#include <optional>
#include <tuple>
#include <vector>

#include "../../include/molnex.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void check(int rc, const char* what) {
    if (rc != MNX_OK) TORCH_CHECK(false, what, " failed (status ", rc, "): ", mnx_last_error());
}

mnx_stream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

// -1 for a type the kernels do not take.
int dtype_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return MNX_F32;
        case at::kBFloat16: return MNX_BF16;
        case at::kHalf: return MNX_F16;
        default: return -1;
    }
}

bool given(const OptTensor& t) { return t.has_value() && t->defined(); }
const void* data(const OptTensor& t) { return given(t) ? t->const_data_ptr() : nullptr; }
void* out(const Tensor& t) { return t.numel() ? t.mutable_data_ptr() : nullptr; }
OptTensor contiguous(const OptTensor& t) { return given(t) ? OptTensor(t->contiguous()) : std::nullopt; }

// ---------------------------------------------------------------------------
// Layer norm
// ---------------------------------------------------------------------------

struct Shape {
    int64_t rows, width;
    int dtype, wdtype;
};

// Checks the arguments, but for x's device.
Shape norm_shape(const char* name, const Tensor& x, const OptTensor& weight, const OptTensor& bias) {
    Shape s{0, 0, dtype_of(x.scalar_type()), -1};
    TORCH_CHECK_TYPE(s.dtype >= 0, "molix::", name, ": float32, bfloat16 or float16, got ", x.scalar_type());
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= MNX_LAYER_NORM_MAX_WIDTH, "molix::", name,
                      ": the last axis must have 1 to ", MNX_LAYER_NORM_MAX_WIDTH, " values, got ", x.sizes());
    s.width = x.size(-1);
    s.rows = x.numel() / s.width;
    for (const auto* t : {&weight, &bias}) {
        if (!given(*t)) continue;
        TORCH_CHECK_VALUE((*t)->dim() == 1 && (*t)->size(0) == s.width, "molix::", name,
                          ": weight and bias must be (", s.width, ",), got ", (*t)->sizes());
        const int d = dtype_of((*t)->scalar_type());
        TORCH_CHECK_TYPE((d == s.dtype || d == MNX_F32) && (s.wdtype < 0 || s.wdtype == d) &&
                             (*t)->device() == x.device(),
                         "molix::", name, ": weight and bias share one type, ", x.scalar_type(),
                         " or float32, and x's device");
        s.wdtype = d;
    }
    if (s.wdtype < 0) s.wdtype = s.dtype;
    return s;
}

Shape gpu_shape(const char* name, const Tensor& x, const OptTensor& weight, const OptTensor& bias) {
    TORCH_CHECK(x.is_cuda(), "molix::", name, " runs on the GPU only (got a ", x.device(), " tensor)");
    return norm_shape(name, x, weight, bias);
}

// A tensor's rows in place where they are evenly spaced (a column block of a wider matrix), else a contiguous copy.
struct Rows {
    Tensor t;
    int64_t ld;
    Rows(const Tensor& x, int64_t width) : t(x), ld(width) {
        if (x.is_contiguous()) return;
        if (x.dim() == 2 && x.stride(1) == 1 && x.stride(0) >= width) ld = x.stride(0);
        else t = x.contiguous();
    }
    const void* ptr() const { return t.numel() ? t.const_data_ptr() : nullptr; }
};

void check_stats(const char* name, const Tensor& stats, const Tensor& x, int64_t rows) {
    TORCH_CHECK_VALUE(stats.scalar_type() == at::kFloat && stats.dim() == 2 && stats.size(0) == 2 &&
                          stats.size(1) == rows && stats.device() == x.device(),
                      "molix::", name, ": stats float32 (2, ", rows, ")");
}

void check_like(const char* name, const char* what, const Tensor& t, const Tensor& x) {
    TORCH_CHECK_VALUE(t.sizes() == x.sizes() && t.scalar_type() == x.scalar_type() && t.device() == x.device(),
                      "molix::", name, ": ", what, " must be ", x.scalar_type(), " ", x.sizes(), " like x, got ",
                      t.scalar_type(), " ", t.sizes());
}

std::tuple<Tensor, Tensor> layer_norm(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
    const Shape s = gpu_shape("layer_norm", x, weight, bias);
    const c10::DeviceGuard guard(x.device());
    const Rows xs(x, s.width);
    const OptTensor w = contiguous(weight), b = contiguous(bias);
    Tensor y = at::empty(x.sizes(), x.options()), stats = at::empty({2, s.rows}, x.options().dtype(at::kFloat));
    check(mnx_layer_norm_fwd(xs.ptr(), xs.ld, s.rows, s.width, data(w), data(b), eps, s.dtype, s.wdtype, out(y),
                             static_cast<float*>(out(stats)), stream_of(x)),
          "layer_norm");
    return {y, stats};
}

Tensor vector_like(const Tensor& x, const OptTensor& t, bool needed) {
    return at::empty({needed ? x.size(-1) : 0}, given(t) ? t->options() : x.options());
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_backward(const Tensor& grad, const Tensor& x, const OptTensor& weight,
                                                       const OptTensor& bias, const Tensor& stats, double eps,
                                                       bool need_x, bool need_w, bool need_b) {
    (void)eps;  // higher orders read it
    const char* name = "layer_norm_backward";
    const Shape s = gpu_shape(name, x, weight, bias);
    check_like(name, "grad", grad, x);
    check_stats(name, stats, x, s.rows);
    TORCH_CHECK_VALUE((!need_w || given(weight)) && (!need_b || given(bias)), "molix::", name,
                      ": the gradient of a weight or bias that is not there");
    const c10::DeviceGuard guard(x.device());
    const Rows xs(x, s.width), g(grad, s.width);
    const OptTensor w = contiguous(weight);
    const Tensor st = stats.contiguous();
    Tensor gx = need_x ? at::empty(x.sizes(), x.options()) : at::empty({0}, x.options());
    Tensor gw = vector_like(x, weight, need_w), gb = vector_like(x, bias, need_b);
    Tensor ws;
    size_t bytes = 0;
    if (need_w || need_b) {
        bytes = mnx_layer_norm_bwd_workspace_bytes(s.rows, s.width);
        ws = at::empty({int64_t(bytes)}, x.options().dtype(at::kByte));
    }
    check(mnx_layer_norm_bwd(g.ptr(), g.ld, xs.ptr(), xs.ld, s.rows, s.width, data(w), s.dtype, s.wdtype,
                             st.const_data_ptr<float>(), out(gx), out(gw), out(gb), bytes ? out(ws) : nullptr, bytes,
                             stream_of(x)),
          "layer_norm backward");
    return {gx, gw, gb};
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_backward2(const Tensor& grad, const Tensor& x, const OptTensor& weight,
                                                        const Tensor& stats, double eps, const OptTensor& seed_x,
                                                        const OptTensor& seed_w, const OptTensor& seed_b,
                                                        bool need_w) {
    (void)eps;
    const char* name = "layer_norm_backward2";
    Shape s = gpu_shape(name, x, weight, std::nullopt);
    check_like(name, "grad", grad, x);
    check_stats(name, stats, x, s.rows);
    if (given(seed_x)) check_like(name, "seed_x", *seed_x, x);
    if (!given(weight) && (given(seed_w) || given(seed_b)))
        s.wdtype = dtype_of((given(seed_w) ? seed_w : seed_b)->scalar_type());
    for (const auto* t : {&seed_w, &seed_b})
        TORCH_CHECK_VALUE(!given(*t) || ((*t)->dim() == 1 && (*t)->size(0) == s.width && (*t)->device() == x.device() &&
                                         dtype_of((*t)->scalar_type()) == s.wdtype && s.wdtype >= 0),
                          "molix::", name, ": seed_w and seed_b like the weight");
    TORCH_CHECK_VALUE(!need_w || given(weight), "molix::", name, ": the derivative of a weight that is not there");
    const c10::DeviceGuard guard(x.device());
    const Rows xs(x, s.width), g(grad, s.width), u(given(seed_x) ? *seed_x : at::zeros_like(xs.t), s.width);
    const OptTensor w = contiguous(weight), p = contiguous(seed_w), q = contiguous(seed_b);
    const Tensor st = stats.contiguous();
    Tensor dg = at::empty(x.sizes(), x.options()), dx = at::empty(x.sizes(), x.options());
    Tensor dw = vector_like(x, weight, need_w);
    const size_t bytes = mnx_layer_norm_bwd_workspace_bytes(s.rows, s.width);
    Tensor ws = at::empty({int64_t(bytes)}, x.options().dtype(at::kByte));
    check(mnx_layer_norm_bwd2(g.ptr(), g.ld, xs.ptr(), xs.ld, u.ptr(), u.ld, data(p), data(q), s.rows, s.width,
                              data(w), s.dtype, s.wdtype, st.const_data_ptr<float>(), out(dg), out(dx), out(dw),
                              out(ws), bytes, stream_of(x)),
          "layer_norm second order");
    return {dg, dx, dw};
}

// The ops through the dispatcher: differentiable where the caller's mode has gradients on.
template <typename F>
auto op(const char* name) {
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}
auto layer_norm_op() {
    static auto o = op<decltype(layer_norm)>("molix::layer_norm");
    return o;
}
auto layer_norm_backward_op() {
    static auto o = op<decltype(layer_norm_backward)>("molix::layer_norm_backward");
    return o;
}
auto layer_norm_backward2_op() {
    static auto o = op<decltype(layer_norm_backward2)>("molix::layer_norm_backward2");
    return o;
}

bool wants_grad(const OptTensor& t) { return given(t) && t->requires_grad(); }
OptTensor optional(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }
Tensor or_undefined(const OptTensor& t) { return given(t) ? *t : Tensor(); }

// The autograd Functions below know backward mode, outside torch.func's transforms.  Whether t carries a tangent
// (forward mode), and whether this call is inside a transform (the key is in force while one is):
bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
bool has_tangent(const OptTensor& t) { return t.has_value() && has_tangent(*t); }
bool transformed() { return c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerBackMode); }

// The three ops as torch operations in float32, rounded once at the end: differentiable in every mode and to any order.
// Tensors that carry tangents, calls that torch.func's transforms differentiate or batch, and the third order in
// backward mode take them.
std::tuple<Tensor, Tensor> layer_norm_formula(const Tensor& x, const OptTensor& weight, const OptTensor& bias,
                                              double eps) {
    norm_shape("layer_norm", x, weight, bias);
    const auto f32 = [](const OptTensor& t) { return given(t) ? OptTensor(t->to(at::kFloat)) : std::nullopt; };
    const auto [y, mu, r] = at::native_layer_norm(x.to(at::kFloat), {x.size(-1)}, f32(weight), f32(bias), eps);
    return {y.to(x.scalar_type()), at::stack({mu.detach().reshape(-1), r.detach().reshape(-1)})};
}

// A row h of float32 values without mean and of variance one, and its derivative J.
struct Normed {
    Tensor h, r;
    Normed(const Tensor& x, double eps) {
        const Tensor xc = x - x.mean(1, true);
        r = (xc.square().mean(1, true) + eps).rsqrt();
        h = xc * r;
    }
    Tensor J(const Tensor& a) const { return r * (a - a.mean(1, true) - h * (a * h).mean(1, true)); }
};
Tensor rows_f32(const Tensor& t) { return t.reshape({-1, t.size(-1)}).to(at::kFloat); }

std::tuple<Tensor, Tensor, Tensor> layer_norm_backward_formula(const Tensor& grad, const Tensor& x,
                                                               const OptTensor& weight, const OptTensor& bias,
                                                               const Tensor& /*stats*/, double eps, bool need_x,
                                                               bool need_w, bool need_b) {
    norm_shape("layer_norm_backward", x, weight, bias);
    check_like("layer_norm_backward", "grad", grad, x);
    const Normed n(rows_f32(x), eps);
    const Tensor g = rows_f32(grad);
    Tensor gx = at::empty({0}, x.options()), gw = vector_like(x, weight, false), gb = vector_like(x, bias, false);
    if (need_x) gx = n.J(given(weight) ? g * weight->to(at::kFloat) : g).to(x.scalar_type()).reshape(x.sizes());
    if (need_w) gw = (g * n.h).sum(0).to(gw.scalar_type());
    if (need_b) gb = g.sum(0).to(gb.scalar_type());
    return {gx, gw, gb};
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_backward2_formula(const Tensor& grad, const Tensor& x,
                                                                const OptTensor& weight, const Tensor& /*stats*/,
                                                                double eps, const OptTensor& seed_x,
                                                                const OptTensor& seed_w, const OptTensor& seed_b,
                                                                bool need_w) {
    const Tensor g = rows_f32(grad), x2 = rows_f32(x);
    const Normed n(x2, eps);
    const Tensor& h = n.h;
    const Tensor u = given(seed_x) ? rows_f32(*seed_x) : at::zeros_like(x2);
    const Tensor w = given(weight) ? weight->to(at::kFloat) : at::ones({x.size(-1)}, x2.options());
    const Tensor a = g * w, ju = n.J(u);
    Tensor dg = w * ju;
    Tensor dx = -n.r * ((a * h).mean(1, true) * ju + (u * h).mean(1, true) * n.J(a)) - n.r * h * (ju * a).mean(1, true);
    if (given(seed_w)) {
        const Tensor p = seed_w->to(at::kFloat);
        dg = dg + p * h;
        dx = dx + n.J(g * p);
    }
    if (given(seed_b)) dg = dg + seed_b->to(at::kFloat);
    Tensor dw = need_w ? (g * ju).sum(0).to(weight->scalar_type()) : vector_like(x, weight, false);
    return {dg.to(x.scalar_type()).reshape(x.sizes()), dx.to(x.scalar_type()).reshape(x.sizes()), dw};
}

// The statistics are not differentiable: they leave through `out`, not as an output that is marked so, which compiled
// autograd does not take.
class LayerNorm : public torch::autograd::Function<LayerNorm> {
  public:
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight, const OptTensor& bias,
                          double eps, Tensor* out) {
        at::AutoDispatchBelowADInplaceOrView below;
        auto [y, stats] = layer_norm_op().call(x, weight, bias, eps);
        ctx->save_for_backward({x, or_undefined(weight), or_undefined(bias), stats});
        ctx->saved_data["eps"] = eps;
        ctx->set_materialize_grads(false);
        *out = stats;
        return y;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w = saved[1], &b = saved[2];
        // edges are numbered over the tensors that were there
        const bool nx = ctx->needs_input_grad(0), nw = w.defined() && ctx->needs_input_grad(1);
        const bool nb = b.defined() && ctx->needs_input_grad(w.defined() ? 2 : 1);
        if (!grads[0].defined() || !(nx || nw || nb)) return variable_list(5);
        auto [gx, gw, gb] = layer_norm_backward_op().call(grads[0], x, optional(w), optional(b), saved[3],
                                                          ctx->saved_data["eps"].toDouble(), nx, nw, nb);
        return {nx ? gx : Tensor(), nw ? gw : Tensor(), nb ? gb : Tensor(), Tensor(), Tensor()};
    }
};

std::tuple<Tensor, Tensor> layer_norm_autograd(const Tensor& x, const OptTensor& weight, const OptTensor& bias,
                                               double eps) {
    if (has_tangent(x) || has_tangent(weight) || has_tangent(bias)) return layer_norm_formula(x, weight, bias, eps);
    if (at::GradMode::is_enabled() && (x.requires_grad() || wants_grad(weight) || wants_grad(bias))) {
        if (transformed()) return layer_norm_formula(x, weight, bias, eps);
        Tensor stats;
        Tensor y = LayerNorm::apply(x, weight, bias, eps, &stats);
        return {y, stats};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    return layer_norm_op().call(x, weight, bias, eps);
}

class LayerNormBackward : public torch::autograd::Function<LayerNormBackward> {
  public:
    static variable_list forward(AutogradContext* ctx, const Tensor& grad, const Tensor& x, const OptTensor& weight,
                                 const OptTensor& bias, const Tensor& stats, double eps, bool need_x, bool need_w,
                                 bool need_b) {
        at::AutoDispatchBelowADInplaceOrView below;
        auto [gx, gw, gb] = layer_norm_backward_op().call(grad, x, weight, bias, stats, eps, need_x, need_w, need_b);
        ctx->save_for_backward({grad, x, or_undefined(weight), stats});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["needed"] = int64_t(need_x) | int64_t(need_w) << 1 | int64_t(need_b) << 2;
        ctx->set_materialize_grads(false);
        return {gx, gw, gb};
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& seeds) {
        variable_list none(9);
        const auto saved = ctx->get_saved_variables();
        const Tensor& w = saved[2];
        const bool ng = ctx->needs_input_grad(0), nx = ctx->needs_input_grad(1);
        const bool nw = w.defined() && ctx->needs_input_grad(2);
        const int64_t needed = ctx->saved_data["needed"].toInt();
        OptTensor seed[3];
        bool any = false;
        for (int k = 0; k < 3; ++k) {
            if (needed >> k & 1) seed[k] = optional(seeds[k]);
            any |= given(seed[k]);
        }
        if (!any || !(ng || nx || nw)) return none;
        auto [dg, dx, dw] = layer_norm_backward2_op().call(saved[0], saved[1], optional(w), saved[3],
                                                           ctx->saved_data["eps"].toDouble(), seed[0], seed[1],
                                                           seed[2], nw);
        if (ng) none[0] = dg;
        if (nx) none[1] = dx;
        if (nw) none[2] = dw;
        return none;
    }
};

std::tuple<Tensor, Tensor, Tensor> layer_norm_backward_autograd(const Tensor& grad, const Tensor& x,
                                                                const OptTensor& weight, const OptTensor& bias,
                                                                const Tensor& stats, double eps, bool need_x,
                                                                bool need_w, bool need_b) {
    if (has_tangent(grad) || has_tangent(x) || has_tangent(weight))
        return layer_norm_backward_formula(grad, x, weight, bias, stats, eps, need_x, need_w, need_b);
    if (at::GradMode::is_enabled() && (grad.requires_grad() || x.requires_grad() || wants_grad(weight))) {
        if (transformed())
            return layer_norm_backward_formula(grad, x, weight, bias, stats, eps, need_x, need_w, need_b);
        auto r = LayerNormBackward::apply(grad, x, weight, bias, stats, eps, need_x, need_w, need_b);
        return {r[0], r[1], r[2]};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    return layer_norm_backward_op().call(grad, x, weight, bias, stats, eps, need_x, need_w, need_b);
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_backward2_autograd(const Tensor& grad, const Tensor& x,
                                                                 const OptTensor& weight, const Tensor& stats,
                                                                 double eps, const OptTensor& seed_x,
                                                                 const OptTensor& seed_w, const OptTensor& seed_b,
                                                                 bool need_w) {
    bool tracked = false, tangent = false;
    for (const OptTensor& t : {OptTensor(grad), OptTensor(x), weight, seed_x, seed_w, seed_b})
        tracked |= wants_grad(t), tangent |= has_tangent(t);
    if ((at::GradMode::is_enabled() && tracked) || tangent)
        return layer_norm_backward2_formula(grad, x, weight, stats, eps, seed_x, seed_w, seed_b, need_w);
    at::AutoDispatchBelowADInplaceOrView below;
    return layer_norm_backward2_op().call(grad, x, weight, stats, eps, seed_x, seed_w, seed_b, need_w);
}

// ---------------------------------------------------------------------------
// AdamW
// ---------------------------------------------------------------------------

constexpr int64_t kStateBlock = 256;

at::Device gpu_of(const char* name, at::TensorList ts) {
    TORCH_CHECK(ts[0].is_cuda(), "molix::", name, " runs on the GPU only (got a ", ts[0].device(), " tensor)");
    return ts[0].device();
}

void check_values(const char* name, const char* what, const Tensor& t, at::Device device) {
    TORCH_CHECK(t.layout() == at::kStrided, "molix::", name, ": ", what, " must be dense, got ", t.layout());
    TORCH_CHECK(t.device() == device, "molix::", name, ": ", what, " on ", t.device(), ", others on ", device);
    TORCH_CHECK_TYPE(dtype_of(t.scalar_type()) >= 0, "molix::", name, ": ", what,
                     " float32, bfloat16 or float16, got ", t.scalar_type());
}

// Addresses that one call writes: its workgroups run at once, so none may be given twice.  Up to `count` of them; null
// (tensors without elements) any number of times.
class Written {
  public:
    explicit Written(size_t count) {
        size_t size = 16;
        for (; size < 2 * count; size *= 2) --shift_;
        places_.resize(size);
    }
    template <typename Pointers>
    bool add(const Pointers& pointers) {  // whether all are new
        for (const void* p : pointers)
            if (p && !add_one(p)) return false;
        return true;
    }

  private:
    bool add_one(const void* p) {
        for (size_t at = reinterpret_cast<uintptr_t>(p) * 0x9E3779B97F4A7C15u >> shift_;; ++at) {
            const void*& place = places_[at & (places_.size() - 1)];
            if (place == p) return false;
            if (!place) return place = p, true;
        }
    }
    int shift_ = 60;
    std::vector<const void*> places_;
};

Tensor grad_norm(at::TensorList grads) {
    if (grads.empty()) return at::zeros({});
    const at::Device device = gpu_of("grad_norm", grads);
    const c10::DeviceGuard guard(device);
    std::vector<Tensor> kept;
    std::vector<const void*> ptrs;
    std::vector<int64_t> numel;
    std::vector<int32_t> dtype;
    for (const Tensor& g : grads) {
        check_values("grad_norm", "gradients", g, device);
        const bool whole = g.is_non_overlapping_and_dense();
        if (!whole) kept.push_back(g.contiguous());
        ptrs.push_back((whole ? g : kept.back()).const_data_ptr());
        numel.push_back(g.numel());
        dtype.push_back(dtype_of(g.scalar_type()));
    }
    const auto f32 = grads[0].options().dtype(at::kFloat);
    const size_t bytes = mnx_grad_norm_workspace_bytes(numel.data(), int64_t(numel.size()));
    Tensor norm = at::empty({}, f32), ws = at::empty({int64_t(bytes)}, f32.dtype(at::kByte));
    check(mnx_grad_norm(ptrs.data(), numel.data(), dtype.data(), int64_t(ptrs.size()), static_cast<float*>(out(norm)),
                        out(ws), bytes, stream_of(norm)),
          "grad_norm");
    return norm;
}

Tensor grad_norm_autograd(at::TensorList grads) {
    if (at::GradMode::is_enabled())
        for (const Tensor& g : grads)
            TORCH_CHECK(!g.requires_grad(), "molix::grad_norm is not differentiable: detach its tensors, or call it "
                                            "under no_grad");
    at::AutoDispatchBelowADInplaceOrView below;
    static auto o = op<decltype(grad_norm)>("molix::grad_norm");
    return o.call(grads);
}

struct Options {
    double lr, beta1, beta2, eps, weight_decay;
    bool maximize;
    std::optional<double> max_norm;
    bool skip_nonfinite;
    int64_t seed;
};

// Returns the norm that was used; without one, an empty tensor.
Tensor step(const char* name, int bits, at::TensorList params, at::TensorList grads, at::TensorList exp_avgs,
            at::TensorList exp_avg_sqs, at::TensorList bases, at::TensorList steps, const OptTensor& lr,
            const OptTensor& norm_in, const Options& o) {
    const size_t count = params.size();
    TORCH_CHECK_VALUE(grads.size() == count && exp_avgs.size() == count && exp_avg_sqs.size() == count &&
                          steps.size() == count && (bits == 32 || bases.size() == count),
                      "molix::", name, ": lists of ", count, ", ", grads.size(), ", ", exp_avgs.size(), ", ",
                      exp_avg_sqs.size(), " and ", steps.size(), " tensors");
    TORCH_CHECK_VALUE(o.beta1 >= 0 && o.beta1 < 1 && o.beta2 >= 0 && o.beta2 < 1 && o.eps >= 0, "molix::", name,
                      ": betas (", o.beta1, ", ", o.beta2, "), eps ", o.eps);
    TORCH_CHECK_VALUE(!o.max_norm || *o.max_norm >= 0, "molix::", name, ": max_norm ", o.max_norm.value_or(0));
    const bool uses_norm = o.max_norm.has_value() || o.skip_nonfinite;
    if (!count) return given(norm_in) ? *norm_in : uses_norm ? at::zeros({}) : at::empty({0});
    const at::Device device = gpu_of(name, params);
    const c10::DeviceGuard guard(device);
    const at::ScalarType moment = bits == 32 ? at::kFloat : at::kByte;

    std::vector<void*> p_ptr(count), m_ptr(count), v_ptr(count);
    std::vector<const void*> g_ptr(count);
    std::vector<int16_t*> b_ptr(count);
    std::vector<float*> s_ptr(count);
    std::vector<int64_t> numel(count);
    std::vector<int32_t> dtype(count);
    std::vector<Tensor> kept;                          // gradients laid out like their parameters
    std::vector<std::pair<size_t, Tensor>> gaps;  // parameters with gaps and their copies
    for (size_t i = 0; i < count; ++i) {
        const Tensor &p = params[i], &g = grads[i], &m = exp_avgs[i], &v = exp_avg_sqs[i], &s = steps[i];
        check_values(name, "parameters", p, device);
        TORCH_CHECK(g.layout() == at::kStrided, "molix::", name, ": sparse gradients are not supported");
        TORCH_CHECK_VALUE(g.scalar_type() == p.scalar_type() && g.sizes() == p.sizes() && g.device() == device,
                          "molix::", name, ": gradient ", i, " is ", g.scalar_type(), " ", g.sizes(), " on ",
                          g.device(), ", its parameter ", p.scalar_type(), " ", p.sizes(), " on ", device);
        TORCH_CHECK_VALUE(m.scalar_type() == moment && v.scalar_type() == moment && m.sizes() == p.sizes() &&
                              v.sizes() == p.sizes() && m.device() == device && v.device() == device,
                          "molix::", name, ": the moments of tensor ", i, " must be ", moment,
                          " of its shape and device");
        TORCH_CHECK_VALUE(s.scalar_type() == at::kFloat && s.numel() == 1 && s.device() == device, "molix::", name,
                          ": step ", i, " must be one float32 on ", device);
        if (bits == 8) {
            const Tensor& b = bases[i];
            const int64_t blocks = (p.numel() + kStateBlock - 1) / kStateBlock;
            TORCH_CHECK_VALUE(b.scalar_type() == at::kShort && b.dim() == 2 && b.size(0) == blocks && b.size(1) == 2 &&
                                  b.is_contiguous() && b.device() == device,
                              "molix::", name, ": bases ", i, " must be contiguous int16 (", blocks, ", 2) on ",
                              device);
            b_ptr[i] = static_cast<int16_t*>(out(b));
        }
        const Tensor *pp = &p, *gg = &g;
        if (!(p.is_contiguous() && g.is_contiguous() && m.is_contiguous() && v.is_contiguous())) {
            if (!p.is_non_overlapping_and_dense()) {
                TORCH_CHECK_VALUE(at::has_internal_overlap(p) != at::MemOverlap::Yes, "molix::", name, ": parameter ",
                                  i, " has elements that share memory");
                gaps.emplace_back(i, p.detach().contiguous());
                pp = &gaps.back().second;
            }
            TORCH_CHECK_VALUE(m.strides() == pp->strides() && v.strides() == pp->strides(), "molix::", name,
                              ": the moments of tensor ", i,
                              " must have its strides (contiguous where the tensor has gaps)");
            if (g.strides() != pp->strides()) {
                kept.push_back(at::empty_strided(pp->sizes(), pp->strides(), g.options()).copy_(g.detach()));
                gg = &kept.back();
            }
        }
        p_ptr[i] = out(p);
        g_ptr[i] = gg->numel() ? gg->const_data_ptr() : nullptr;
        m_ptr[i] = out(m);
        v_ptr[i] = out(v);
        s_ptr[i] = static_cast<float*>(out(s));
        numel[i] = p.numel();
        dtype[i] = dtype_of(p.scalar_type());
    }
    Written written((bits == 8 ? 5 : 4) * count);
    TORCH_CHECK_VALUE(written.add(p_ptr), "molix::", name, ": a parameter is given twice");
    TORCH_CHECK_VALUE(written.add(m_ptr) && written.add(v_ptr) && written.add(b_ptr), "molix::", name,
                      ": a moment or its bases are given twice");
    TORCH_CHECK_VALUE(written.add(s_ptr), "molix::", name, ": a step count is given twice");
    for (const auto& [i, copy] : gaps) p_ptr[i] = out(copy);

    mnx_adamw_args a{};
    a.count = int64_t(count);
    a.params = p_ptr.data();
    a.grads = g_ptr.data();
    a.exp_avgs = m_ptr.data();
    a.exp_avg_sqs = v_ptr.data();
    a.bases = bits == 8 ? b_ptr.data() : nullptr;
    a.steps = s_ptr.data();
    a.numel = numel.data();
    a.dtype = dtype.data();
    a.state_bits = bits;
    a.maximize = o.maximize;
    a.skip_nonfinite = o.skip_nonfinite;
    a.seed = uint32_t(o.seed);
    a.lr = o.lr;
    a.beta1 = o.beta1;
    a.beta2 = o.beta2;
    a.eps = o.eps;
    a.weight_decay = o.weight_decay;
    a.max_norm = o.max_norm.value_or(-1.0);
    Tensor rate;
    if (given(lr)) {
        TORCH_CHECK_VALUE(lr->numel() == 1 && lr->device() == device, "molix::", name,
                          ": lr must be a number or one value on ", device);
        rate = lr->detach().to(at::kFloat);
        a.lr_device = rate.const_data_ptr<float>();
    }
    const auto f32 = params[0].options().dtype(at::kFloat).requires_grad(false);
    Tensor norm;
    if (given(norm_in)) {
        TORCH_CHECK_VALUE(norm_in->numel() == 1 && norm_in->scalar_type() == at::kFloat && norm_in->device() == device,
                          "molix::", name, ": grad_norm must be one float32 on ", device);
        a.norm_in = norm_in->const_data_ptr<float>();
    } else if (uses_norm) {
        norm = at::empty({}, f32);
        a.norm_out = static_cast<float*>(out(norm));
    }
    a.workspace_bytes = mnx_adamw_workspace_bytes(a.numel, a.count);
    Tensor ws = at::empty({int64_t(a.workspace_bytes)}, f32.dtype(at::kByte));
    a.workspace = out(ws);
    check(mnx_adamw_step(&a, stream_of(ws)), name);
    for (const auto& [i, copy] : gaps) params[i].detach().copy_(copy);
    for (const at::TensorList& l : {params, exp_avgs, exp_avg_sqs, steps, bases})
        for (const Tensor& t : l) t.unsafeGetTensorImpl()->bump_version();
    return norm.defined() ? norm : at::empty({0}, f32);
}

Tensor adamw_step(at::TensorList params, at::TensorList grads, at::TensorList exp_avgs, at::TensorList exp_avg_sqs,
                  at::TensorList steps, double lr, double beta1, double beta2, double eps, double weight_decay,
                  bool maximize, std::optional<double> max_norm, const OptTensor& grad_norm, bool skip_nonfinite,
                  const OptTensor& lr_tensor) {
    return step("adamw_step", 32, params, grads, exp_avgs, exp_avg_sqs, {}, steps, lr_tensor, grad_norm,
                {lr, beta1, beta2, eps, weight_decay, maximize, max_norm, skip_nonfinite, 0});
}

Tensor adamw8_step(at::TensorList params, at::TensorList grads, at::TensorList exp_avgs, at::TensorList exp_avg_sqs,
                   at::TensorList bases, at::TensorList steps, double lr, double beta1, double beta2, double eps,
                   double weight_decay, bool maximize, std::optional<double> max_norm, const OptTensor& grad_norm,
                   bool skip_nonfinite, const OptTensor& lr_tensor, int64_t seed) {
    return step("adamw8_step", 8, params, grads, exp_avgs, exp_avg_sqs, bases, steps, lr_tensor, grad_norm,
                {lr, beta1, beta2, eps, weight_decay, maximize, max_norm, skip_nonfinite, seed});
}

void adamw8_moments(at::TensorList exp_avgs, at::TensorList exp_avg_sqs, at::TensorList bases, at::TensorList out_avgs,
                    at::TensorList out_avg_sqs) {
    const char* name = "adamw8_moments";
    const size_t count = exp_avgs.size();
    TORCH_CHECK_VALUE(exp_avg_sqs.size() == count && bases.size() == count && out_avgs.size() == count &&
                          out_avg_sqs.size() == count,
                      "molix::", name, ": lists of ", count, ", ", exp_avg_sqs.size(), ", ", bases.size(), ", ",
                      out_avgs.size(), " and ", out_avg_sqs.size(), " tensors");
    if (!count) return;
    const at::Device device = gpu_of(name, exp_avgs);
    const c10::DeviceGuard guard(device);
    std::vector<const void*> m_ptr(count), v_ptr(count);
    std::vector<int16_t*> b_ptr(count);
    std::vector<float*> om_ptr(count), ov_ptr(count);
    std::vector<int64_t> numel(count);
    for (size_t i = 0; i < count; ++i) {
        const Tensor &m = exp_avgs[i], &v = exp_avg_sqs[i], &b = bases[i];
        TORCH_CHECK_VALUE(m.scalar_type() == at::kByte && v.scalar_type() == at::kByte && m.sizes() == v.sizes() &&
                              m.strides() == v.strides() && m.is_non_overlapping_and_dense() &&
                              m.device() == device && v.device() == device,
                          "molix::", name, ": the moments of tensor ", i, " must be dense uint8 of one layout");
        const int64_t blocks = (m.numel() + kStateBlock - 1) / kStateBlock;
        TORCH_CHECK_VALUE(b.scalar_type() == at::kShort && b.dim() == 2 && b.size(0) == blocks && b.size(1) == 2 &&
                              b.is_contiguous() && b.device() == device,
                          "molix::", name, ": bases ", i, " must be contiguous int16 (", blocks, ", 2) on ", device);
        for (const Tensor* t : {&out_avgs[i], &out_avg_sqs[i]})
            TORCH_CHECK_VALUE(t->scalar_type() == at::kFloat && t->sizes() == m.sizes() &&
                                  t->strides() == m.strides() && t->device() == device,
                              "molix::", name, ": out of tensor ", i, " must be float32 of its shape and strides");
        m_ptr[i] = m.const_data_ptr();
        v_ptr[i] = v.const_data_ptr();
        b_ptr[i] = static_cast<int16_t*>(out(b));
        om_ptr[i] = static_cast<float*>(out(out_avgs[i]));
        ov_ptr[i] = static_cast<float*>(out(out_avg_sqs[i]));
        numel[i] = m.numel();
    }
    Written written(2 * count);
    TORCH_CHECK_VALUE(written.add(om_ptr) && written.add(ov_ptr), "molix::", name, ": an out is given twice");
    check(mnx_adamw8_moments(m_ptr.data(), v_ptr.data(), b_ptr.data(), numel.data(), int64_t(count), om_ptr.data(),
                             ov_ptr.data(), stream_of(exp_avgs[0])),
          name);
    for (const at::TensorList& l : {out_avgs, out_avg_sqs})
        for (const Tensor& t : l) t.unsafeGetTensorImpl()->bump_version();
}

// ---------------------------------------------------------------------------
// Orthogonalised updates
// ---------------------------------------------------------------------------

// A call's workspace is at most this, or one matrix's: longer lists and larger stacks take several calls.
constexpr size_t kMuonWorkspace = size_t(4) << 30;

// Whether memory that is written overlaps other memory of the call.  Tensors with gaps may interleave: of those only
// the first address counts.
class Overlap {
  public:
    void add(const Tensor& t, bool written) {
        if (!t.numel()) return;
        const auto lo = reinterpret_cast<uintptr_t>(t.const_data_ptr());
        const size_t length = t.is_non_overlapping_and_dense() ? t.numel() * t.element_size() : 1;
        spans_.push_back({lo, lo + length, written});
    }
    bool found() {
        std::sort(spans_.begin(), spans_.end(), [](const Span& a, const Span& b) { return a.lo < b.lo; });
        uintptr_t any = 0, written = 0;
        for (const Span& s : spans_) {
            if (s.lo < (s.written ? any : written)) return true;
            any = std::max(any, s.hi);
            if (s.written) written = std::max(written, s.hi);
        }
        return false;
    }

  private:
    struct Span {
        uintptr_t lo, hi;
        bool written;
    };
    std::vector<Span> spans_;
};

struct Iteration {
    int64_t steps;
    double a, b, c, eps;
};

void check_iteration(const char* name, const Iteration& it) {
    TORCH_CHECK_VALUE(it.steps >= 1 && it.steps <= MNX_MUON_MAX_STEPS, "molix::", name, ": 1 to ", MNX_MUON_MAX_STEPS,
                      " steps, got ", it.steps);
    TORCH_CHECK_VALUE(it.eps >= 0 && std::isfinite(it.eps) && std::isfinite(it.a) && std::isfinite(it.b) &&
                          std::isfinite(it.c),
                      "molix::", name, ": coefficients (", it.a, ", ", it.b, ", ", it.c, "), eps ", it.eps);
}

void check_matrices(const char* name, const char* what, const Tensor& t) {
    TORCH_CHECK_VALUE(t.dim() >= 2 && t.size(-1) <= MNX_MUON_MAX_SIDE && t.size(-2) <= MNX_MUON_MAX_SIDE, "molix::",
                      name, ": ", what, " must be matrices (or stacks of them) with sides of at most ",
                      MNX_MUON_MAX_SIDE, ", got ", t.sizes());
}

// The lists of one call, the tensors contiguous.
struct MuonLists {
    std::vector<void*> p;
    std::vector<const void*> g;
    std::vector<float*> m;
    std::vector<int64_t> batch, rows, cols;
    std::vector<int32_t> dtype;
    void add(const Tensor& to, const Tensor& from, float* momentum) {
        p.push_back(out(to));
        g.push_back(from.numel() ? from.const_data_ptr() : nullptr);
        m.push_back(momentum);
        rows.push_back(from.size(-2));
        cols.push_back(from.size(-1));
        batch.push_back(from.numel() ? from.numel() / (from.size(-2) * from.size(-1)) : 0);
        dtype.push_back(dtype_of(from.scalar_type()));
    }
    // One half of the tensors, or of the matrices of a single one.
    MuonLists half(bool second) const {
        MuonLists l;
        const size_t count = p.size(), lo = second ? count / 2 : 0, hi = second ? count : count / 2;
        if (count == 1) {
            const int64_t skip = second ? batch[0] / 2 : 0, n = skip * rows[0] * cols[0];
            const int64_t bytes = n * (dtype[0] == MNX_F32 ? 4 : 2);
            l = *this;
            l.p[0] = static_cast<char*>(p[0]) + bytes;
            l.g[0] = static_cast<const char*>(g[0]) + bytes;
            if (m[0]) l.m[0] = m[0] + n;
            l.batch[0] = second ? batch[0] - skip : batch[0] / 2;
            return l;
        }
        const auto take = [&](const auto& from, auto& to) { to.assign(from.begin() + lo, from.begin() + hi); };
        take(p, l.p);
        take(g, l.g);
        take(m, l.m);
        take(batch, l.batch);
        take(rows, l.rows);
        take(cols, l.cols);
        take(dtype, l.dtype);
        return l;
    }
};

void muon_call(const char* name, const MuonLists& l, bool momenta, mnx_muon_args a, const Tensor& like) {
    const size_t count = l.p.size();
    if (!count) return;
    a.count = int64_t(count);
    a.params = l.p.data();
    a.grads = l.g.data();
    a.momenta = momenta ? l.m.data() : nullptr;
    a.batch = l.batch.data();
    a.rows = l.rows.data();
    a.cols = l.cols.data();
    a.dtype = l.dtype.data();
    a.workspace_bytes = mnx_muon_workspace_bytes(&a);  // 0: also for more matrices than a call takes
    if ((!a.workspace_bytes || a.workspace_bytes > kMuonWorkspace) && (count > 1 || l.batch[0] > 1)) {
        for (bool second : {false, true}) muon_call(name, l.half(second), momenta, a, like);
        return;
    }
    TORCH_CHECK(a.workspace_bytes, "molix::", name, ": ", mnx_last_error());
    Tensor ws = at::empty({int64_t(a.workspace_bytes)}, like.options().dtype(at::kByte).requires_grad(false));
    a.workspace = out(ws);
    check(mnx_muon_step(&a, stream_of(like)), name);
}

mnx_muon_args muon_args(const Iteration& it) {
    mnx_muon_args a{};
    a.steps = int32_t(it.steps);
    a.coefficients[0] = it.a;
    a.coefficients[1] = it.b;
    a.coefficients[2] = it.c;
    a.eps = it.eps;
    return a;
}

Tensor orthogonalize(const Tensor& x, int64_t steps, double a, double b, double c, double eps) {
    const char* name = "orthogonalize";
    TORCH_CHECK(x.is_cuda(), "molix::", name, " runs on the GPU only (got a ", x.device(), " tensor)");
    check_values(name, "matrices", x, x.device());
    check_matrices(name, "x", x);
    const Iteration it{steps, a, b, c, eps};
    check_iteration(name, it);
    const c10::DeviceGuard guard(x.device());
    const Tensor from = x.contiguous();
    Tensor y = at::empty(x.sizes(), x.options());
    MuonLists l;
    l.add(y, from, nullptr);
    muon_call(name, l, false, muon_args(it), from);
    return y;
}

Tensor orthogonalize_autograd(const Tensor& x, int64_t steps, double a, double b, double c, double eps) {
    TORCH_CHECK(!(at::GradMode::is_enabled() && x.requires_grad()) && !has_tangent(x),
                "molix::orthogonalize is not differentiable: detach its tensor, or call it under no_grad");
    at::AutoDispatchBelowADInplaceOrView below;
    static auto o = op<decltype(orthogonalize)>("molix::orthogonalize");
    return o.call(x, steps, a, b, c, eps);
}

void muon_step(at::TensorList params, at::TensorList grads, at::TensorList momenta, double lr, double momentum,
               bool nesterov, double weight_decay, int64_t steps, double ca, double cb, double cc, double eps,
               bool match_rms, bool maximize, const OptTensor& lr_tensor) {
    const char* name = "muon_step";
    const size_t count = params.size();
    TORCH_CHECK_VALUE(grads.size() == count && momenta.size() == count, "molix::", name, ": lists of ", count, ", ",
                      grads.size(), " and ", momenta.size(), " tensors");
    const Iteration it{steps, ca, cb, cc, eps};
    check_iteration(name, it);
    TORCH_CHECK_VALUE(momentum >= 0 && momentum < 1, "molix::", name, ": momentum ", momentum);
    if (!count) return;
    const at::Device device = gpu_of(name, params);
    const c10::DeviceGuard guard(device);
    MuonLists l;
    Overlap memory;
    std::vector<Tensor> kept;
    std::vector<std::pair<size_t, Tensor>> copies;  // of parameters that are not contiguous
    for (size_t i = 0; i < count; ++i) {
        const Tensor &p = params[i], &g = grads[i], &m = momenta[i];
        check_values(name, "parameters", p, device);
        check_matrices(name, "parameters", p);
        TORCH_CHECK(g.layout() == at::kStrided, "molix::", name, ": sparse gradients are not supported");
        TORCH_CHECK_VALUE(g.scalar_type() == p.scalar_type() && g.sizes() == p.sizes() && g.device() == device,
                          "molix::", name, ": gradient ", i, " is ", g.scalar_type(), " ", g.sizes(), " on ",
                          g.device(), ", its parameter ", p.scalar_type(), " ", p.sizes(), " on ", device);
        TORCH_CHECK_VALUE(m.scalar_type() == at::kFloat && m.sizes() == p.sizes() && m.device() == device &&
                              m.is_contiguous(),
                          "molix::", name, ": momentum ", i, " must be contiguous float32 of its parameter's shape on ",
                          device);
        TORCH_CHECK_VALUE(at::has_internal_overlap(p) != at::MemOverlap::Yes, "molix::", name, ": parameter ", i,
                          " has elements that share memory");
        memory.add(p, true);
        memory.add(m, true);
        memory.add(g, false);
        const Tensor *to = &p, *from = &g;
        if (!p.is_contiguous()) {
            copies.emplace_back(i, p.detach().contiguous());
            kept.push_back(copies.back().second);
            to = &copies.back().second;
        }
        if (!g.is_contiguous()) {
            kept.push_back(g.detach().contiguous());
            from = &kept.back();
        }
        l.add(*to, *from, static_cast<float*>(out(m)));
    }
    TORCH_CHECK_VALUE(!memory.found(), "molix::", name, ": parameters and momenta must not share memory with each "
                                                        "other, nor with a gradient");
    mnx_muon_args a = muon_args(it);
    a.nesterov = nesterov;
    a.maximize = maximize;
    a.adjust = match_rms;
    a.lr = lr;
    a.momentum = momentum;
    a.weight_decay = weight_decay;
    Tensor rate;
    if (given(lr_tensor)) {
        TORCH_CHECK_VALUE(lr_tensor->numel() == 1 && lr_tensor->device() == device, "molix::", name,
                          ": lr must be a number or one value on ", device);
        rate = lr_tensor->detach().to(at::kFloat);
        a.lr_device = rate.const_data_ptr<float>();
    }
    muon_call(name, l, true, a, params[0]);
    for (const auto& [i, copy] : copies) params[i].detach().copy_(copy);
    for (const at::TensorList& ts : {params, momenta})
        for (const Tensor& t : ts) t.unsafeGetTensorImpl()->bump_version();
}

// ---------------------------------------------------------------------------
// Indexed linear map
// ---------------------------------------------------------------------------

struct Grouped {
    int64_t rows;
    int32_t classes;
};

// Checks the rows' plan (class_groups: order, starts) against `rows`.
Grouped check_groups(const char* name, const Tensor& order, const Tensor& starts, const Tensor& x) {
    for (const Tensor* t : {&order, &starts})
        TORCH_CHECK_VALUE(t->scalar_type() == at::kInt && t->dim() == 1 && t->is_contiguous() &&
                              t->device() == x.device(),
                          "molix::", name, ": groups are two contiguous int32 vectors on x's device (class_groups)");
    TORCH_CHECK_VALUE(order.size(0) == x.size(0), "molix::", name, ": groups of ", order.size(0), " rows for ",
                      x.size(0));
    const int64_t classes = starts.size(0) - 2;
    TORCH_CHECK_VALUE(classes >= 1 && classes <= MNX_CLASS_GROUPS_MAX_CLASSES, "molix::", name, ": 1 to ",
                      MNX_CLASS_GROUPS_MAX_CLASSES, " classes, got ", classes);
    return {x.size(0), int32_t(classes)};
}

void check_rows(const char* name, const char* what, const Tensor& x) {
    TORCH_CHECK(x.is_cuda(), "molix::", name, " runs on the GPU only (got a ", x.device(), " tensor)");
    TORCH_CHECK(x.layout() == at::kStrided, "molix::", name, ": ", what, " must be dense, got ", x.layout());
    TORCH_CHECK_TYPE(dtype_of(x.scalar_type()) >= 0, "molix::", name, ": ", what,
                     " float32, bfloat16 or float16, got ", x.scalar_type());
    TORCH_CHECK_VALUE(x.dim() == 2 && x.size(1) >= 1 && x.size(1) <= MNX_INDEXED_MAX_WIDTH, "molix::", name, ": ", what,
                      " must be (rows, width) of at most ", MNX_INDEXED_MAX_WIDTH, " columns, got ", x.sizes());
}

Tensor indexed_linear(const Tensor& x, const Tensor& weight, const Tensor& order, const Tensor& starts,
                      bool transposed) {
    const char* name = "indexed_linear";
    check_rows(name, "x", x);
    const Grouped n = check_groups(name, order, starts, x);
    TORCH_CHECK_VALUE(weight.dim() == 3 && weight.size(0) == n.classes && weight.size(transposed ? 2 : 1) == x.size(1) &&
                          weight.size(transposed ? 1 : 2) >= 1 &&
                          weight.size(transposed ? 1 : 2) <= MNX_INDEXED_MAX_WIDTH,
                      "molix::", name, ": weight must be (", n.classes, ", in, out) for x ", x.sizes(), ", got ",
                      weight.sizes());
    TORCH_CHECK_TYPE(weight.scalar_type() == x.scalar_type() && weight.device() == x.device(), "molix::", name,
                     ": weight is ", weight.scalar_type(), " on ", weight.device(), ", x ", x.scalar_type(), " on ",
                     x.device());
    const c10::DeviceGuard guard(x.device());
    const Rows a(x, x.size(1));
    const Tensor w = weight.contiguous();
    const int64_t in = w.size(1), cols = w.size(2);
    Tensor y = at::empty({n.rows, transposed ? in : cols}, x.options().requires_grad(false));
    check(mnx_indexed_linear(a.ptr(), a.ld, n.rows, order.const_data_ptr<int32_t>(), starts.const_data_ptr<int32_t>(),
                             n.classes, w.const_data_ptr(), in, cols, dtype_of(x.scalar_type()), transposed, out(y),
                             stream_of(x)),
          name);
    return y;
}

// 16-bit rows `ld` apart, the width rounded up to whole pieces of 16 bytes, are read with what pads them.
int64_t pieces_of(const Tensor& t) { return (t.size(1) + 7) / 8 * 8; }
bool padding_exists(const Tensor& t) {
    return size_t(t.storage_offset() + t.size(0) * t.stride(0)) * t.element_size() <= t.storage().nbytes();
}

// Rows of whole pieces (what pads them is of no interest), for the products by the tile.
Tensor in_pieces(const Tensor& t) {
    const int64_t width = t.size(1), ld = pieces_of(t);
    if (t.stride(1) == 1 && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0 &&
        ((t.stride(0) == ld && padding_exists(t)) || (width % 8 == 0 && t.stride(0) % 8 == 0)))
        return t;
    Tensor padded = at::empty({t.size(0), ld}, t.options().requires_grad(false)).narrow(1, 0, width);
    return padded.copy_(t);
}
// Rows as they are, unless those that are read with their padding end before it.
Tensor in_place(const Tensor& t) {
    const bool ends = t.scalar_type() != at::kFloat && t.size(0) && t.size(1) % 8 && t.stride(0) == pieces_of(t) &&
                      !padding_exists(t);
    return ends ? t.contiguous() : t;
}

Tensor indexed_linear_wgrad(const Tensor& x, const Tensor& grad, const Tensor& order, const Tensor& starts) {
    const char* name = "indexed_linear_wgrad";
    check_rows(name, "x", x);
    check_rows(name, "grad", grad);
    const Grouped n = check_groups(name, order, starts, x);
    TORCH_CHECK_VALUE(grad.size(0) == n.rows && grad.scalar_type() == x.scalar_type() && grad.device() == x.device(),
                      "molix::", name, ": grad ", grad.scalar_type(), " ", grad.sizes(), " for x ", x.scalar_type(),
                      " ", x.sizes());
    const c10::DeviceGuard guard(x.device());
    const int64_t in = x.size(1), cols = grad.size(1);
    // 50001 rows of 1001 and 999 bfloat16 values take 566 us as they are; rows of 250 are not worth the copies
    const bool copies = x.scalar_type() != at::kFloat && in >= 384 && cols >= 384 && n.rows > 0;
    const Rows a(copies ? in_pieces(x.detach()) : in_place(x), in), g(copies ? in_pieces(grad.detach()) : in_place(grad), cols);
    Tensor gw = at::empty({n.classes, in, cols}, x.options().requires_grad(false)), ws;
    const size_t bytes = mnx_indexed_linear_wgrad_workspace_bytes(n.rows, n.classes, in, cols, dtype_of(x.scalar_type()));
    if (bytes) ws = at::empty({int64_t(bytes)}, x.options().dtype(at::kByte).requires_grad(false));
    check(mnx_indexed_linear_wgrad(a.ptr(), a.ld, g.ptr(), g.ld, n.rows, order.const_data_ptr<int32_t>(),
                                   starts.const_data_ptr<int32_t>(), n.classes, in, cols, dtype_of(x.scalar_type()),
                                   out(gw), bytes ? out(ws) : nullptr, bytes, stream_of(x)),
          name);
    return gw;
}

auto indexed_linear_op() {
    static auto o = op<decltype(indexed_linear)>("molix::indexed_linear");
    return o;
}
auto indexed_linear_wgrad_op() {
    static auto o = op<decltype(indexed_linear_wgrad)>("molix::indexed_linear_wgrad");
    return o;
}

// Both ops are bilinear, and their gradients are the same ops again: differentiable to any order in backward mode.
class IndexedLinear : public torch::autograd::Function<IndexedLinear> {
  public:
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Tensor& order,
                          const Tensor& starts, bool transposed) {
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->save_for_backward({x, weight, order, starts});
        ctx->saved_data["transposed"] = transposed;
        return indexed_linear_op().call(x, weight, order, starts, transposed);
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        variable_list none(5);
        if (!grads[0].defined()) return none;
        const auto saved = ctx->get_saved_variables();
        const bool t = ctx->saved_data["transposed"].toBool();
        const Tensor &g = grads[0], &x = saved[0], &order = saved[2], &starts = saved[3];
        if (ctx->needs_input_grad(0)) none[0] = indexed_linear_op().call(g, saved[1], order, starts, !t);
        if (ctx->needs_input_grad(1)) none[1] = indexed_linear_wgrad_op().call(t ? g : x, t ? x : g, order, starts);
        return none;
    }
};

class IndexedLinearWgrad : public torch::autograd::Function<IndexedLinearWgrad> {
  public:
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& grad, const Tensor& order,
                          const Tensor& starts) {
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->save_for_backward({x, grad, order, starts});
        return indexed_linear_wgrad_op().call(x, grad, order, starts);
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        variable_list none(4);
        if (!grads[0].defined()) return none;
        const auto saved = ctx->get_saved_variables();
        const Tensor &s = grads[0], &order = saved[2], &starts = saved[3];
        if (ctx->needs_input_grad(0)) none[0] = indexed_linear_op().call(saved[1], s, order, starts, true);
        if (ctx->needs_input_grad(1)) none[1] = indexed_linear_op().call(saved[0], s, order, starts, false);
        return none;
    }
};

void backward_mode_only(const char* name, const Tensor& a, const Tensor& b) {
    TORCH_CHECK(!has_tangent(a) && !has_tangent(b), "molix::", name, " has no forward-mode derivative");
    TORCH_CHECK(!transformed(), "molix::", name, " does not run inside torch.func's transforms");
}

Tensor indexed_linear_autograd(const Tensor& x, const Tensor& weight, const Tensor& order, const Tensor& starts,
                               bool transposed) {
    if (at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad())) {
        backward_mode_only("indexed_linear", x, weight);
        return IndexedLinear::apply(x, weight, order, starts, transposed);
    }
    TORCH_CHECK(!has_tangent(x) && !has_tangent(weight), "molix::indexed_linear has no forward-mode derivative");
    at::AutoDispatchBelowADInplaceOrView below;
    return indexed_linear_op().call(x, weight, order, starts, transposed);
}

Tensor indexed_linear_wgrad_autograd(const Tensor& x, const Tensor& grad, const Tensor& order, const Tensor& starts) {
    if (at::GradMode::is_enabled() && (x.requires_grad() || grad.requires_grad())) {
        backward_mode_only("indexed_linear_wgrad", x, grad);
        return IndexedLinearWgrad::apply(x, grad, order, starts);
    }
    TORCH_CHECK(!has_tangent(x) && !has_tangent(grad), "molix::indexed_linear_wgrad has no forward-mode derivative");
    at::AutoDispatchBelowADInplaceOrView below;
    return indexed_linear_wgrad_op().call(x, grad, order, starts);
}

// (order, starts) of molix::class_groups.
std::tuple<Tensor, Tensor> grouped(const Tensor& index, int64_t classes) {
    const Tensor z = index.to(at::kLong).contiguous();
    const c10::DeviceGuard guard(z.device());
    const auto i32 = z.options().dtype(at::kInt);
    Tensor order = at::empty({z.size(0)}, i32), starts = at::empty({classes + 2}, i32);
    const size_t bytes = mnx_class_groups_workspace_bytes(z.size(0), int32_t(classes));
    Tensor ws = at::empty({int64_t(bytes)}, z.options().dtype(at::kByte));
    check(mnx_class_groups(z.numel() ? z.const_data_ptr<int64_t>() : nullptr, z.size(0), int32_t(classes),
                           static_cast<int32_t*>(out(order)), static_cast<int32_t*>(out(starts)), out(ws), bytes,
                           stream_of(z)),
          "class_groups");
    return {order, starts};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(molix, m) {
    const std::vector<at::Tag> tags{at::Tag::pt2_compliant_tag};
    m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps) -> (Tensor, Tensor)", tags);
    m.def("layer_norm_backward(Tensor grad, Tensor x, Tensor? weight, Tensor? bias, Tensor stats, float eps, "
          "bool need_x, bool need_w, bool need_b) -> (Tensor, Tensor, Tensor)",
          tags);
    m.def("layer_norm_backward2(Tensor grad, Tensor x, Tensor? weight, Tensor stats, float eps, Tensor? seed_x, "
          "Tensor? seed_w, Tensor? seed_b, bool need_w) -> (Tensor, Tensor, Tensor)",
          tags);
    m.def("grad_norm(Tensor[] grads) -> Tensor", tags);
    m.def("adamw_step(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] exp_avgs, Tensor(c!)[] exp_avg_sqs, "
          "Tensor(d!)[] steps, float lr, float beta1, float beta2, float eps, float weight_decay, bool maximize, "
          "float? max_norm, Tensor? grad_norm, bool skip_nonfinite, Tensor? lr_tensor) -> Tensor",
          tags);
    m.def("adamw8_step(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] exp_avgs, Tensor(c!)[] exp_avg_sqs, "
          "Tensor(d!)[] bases, Tensor(e!)[] steps, float lr, float beta1, float beta2, float eps, "
          "float weight_decay, bool maximize, float? max_norm, Tensor? grad_norm, bool skip_nonfinite, "
          "Tensor? lr_tensor, int seed) -> Tensor",
          tags);
    m.def("adamw8_moments(Tensor[] exp_avgs, Tensor[] exp_avg_sqs, Tensor[] bases, Tensor(a!)[] out_avgs, "
          "Tensor(b!)[] out_avg_sqs) -> ()",
          tags);
    m.def("indexed_linear(Tensor x, Tensor weight, Tensor order, Tensor starts, bool transposed) -> Tensor", tags);
    m.def("indexed_linear_wgrad(Tensor x, Tensor grad, Tensor order, Tensor starts) -> Tensor", tags);
    m.def("orthogonalize(Tensor x, int steps, float a, float b, float c, float eps) -> Tensor", tags);
    m.def("muon_step(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] momenta, float lr, float momentum, "
          "bool nesterov, float weight_decay, int steps, float a, float b, float c, float eps, bool match_rms, "
          "bool maximize, Tensor? lr_tensor) -> ()",
          tags);
}

TORCH_LIBRARY_IMPL(molix, CUDA, m) {
    m.impl("layer_norm", layer_norm);
    m.impl("layer_norm_backward", layer_norm_backward);
    m.impl("layer_norm_backward2", layer_norm_backward2);
    m.impl("grad_norm", grad_norm);
    m.impl("adamw_step", adamw_step);
    m.impl("adamw8_step", adamw8_step);
    m.impl("adamw8_moments", adamw8_moments);
    m.impl("indexed_linear", indexed_linear);
    m.impl("indexed_linear_wgrad", indexed_linear_wgrad);
    m.impl("orthogonalize", orthogonalize);
    m.impl("muon_step", muon_step);
}

TORCH_LIBRARY_IMPL(molix, CPU, m) {  // these say that they run on the GPU only
    m.impl("indexed_linear", indexed_linear);
    m.impl("indexed_linear_wgrad", indexed_linear_wgrad);
    m.impl("orthogonalize", orthogonalize);
    m.impl("muon_step", muon_step);
}

TORCH_LIBRARY_IMPL(molix, FuncTorchBatched, m) {  // torch.vmap
    m.impl("layer_norm", layer_norm_formula);
    m.impl("layer_norm_backward", layer_norm_backward_formula);
    m.impl("layer_norm_backward2", layer_norm_backward2_formula);
}

TORCH_LIBRARY_IMPL(molix, Autograd, m) {
    m.impl("layer_norm", layer_norm_autograd);
    m.impl("layer_norm_backward", layer_norm_backward_autograd);
    m.impl("layer_norm_backward2", layer_norm_backward2_autograd);
    m.impl("grad_norm", grad_norm_autograd);
    m.impl("indexed_linear", indexed_linear_autograd);
    m.impl("indexed_linear_wgrad", indexed_linear_wgrad_autograd);
    m.impl("orthogonalize", orthogonalize_autograd);
    // no gradients: they write into leaves, whose versions rise
    for (const char* name : {"adamw_step", "adamw8_step", "adamw8_moments", "muon_step"})
        m.impl(name, torch::CppFunction::makeFallthrough());
}

// ---------------------------------------------------------------------------
// The Python module: the ops called through the dispatcher without boxing.  A function that finds a tensor (or a mode)
// with __torch_function__ among its arguments calls nothing and returns NotImplemented: the caller hands the call over.
// ---------------------------------------------------------------------------

namespace {

// Tensor and Parameter themselves, which have no __torch_function__.
bool plain_tensor(PyObject* o) {
    const auto* type = reinterpret_cast<const PyObject*>(Py_TYPE(o));
    return type == THPVariableClass || type == ParameterClass;
}

// Whether o's class has one in force (or a mode is on, too).
bool has_torch_function(PyObject* o) {
    if (plain_tensor(o)) return false;
    static PyObject* const ask = [] {
        PyObject* module = PyImport_ImportModule("torch._C");
        PyObject* f = module ? PyObject_GetAttrString(module, "_has_torch_function_unary") : nullptr;
        Py_XDECREF(module);
        return f;
    }();
    if (!ask) throw python_error();
    PyObject* r = PyObject_CallOneArg(ask, o);
    if (!r) throw python_error();
    const bool yes = r == Py_True;
    Py_DECREF(r);
    return yes;
}

bool mode_on() { return at::impl::torch_function_mode_enabled(); }

// Whether something looks at the ops of a call with these tensors on their way to the kernels and may repeat or replace
// them: dispatch modes, tracers, fake and functional tensors.  All of the work has to be registered ops then.
bool watched(std::initializer_list<const OptTensor*> tensors) {
    using c10::DispatchKey;
    constexpr c10::DispatchKeySet watchers({DispatchKey::Python, DispatchKey::PythonTLSSnapshot, DispatchKey::PythonDispatcher,
                                            DispatchKey::PreDispatch, DispatchKey::Tracer, DispatchKey::Functionalize});
    const auto tls = c10::impl::tls_local_dispatch_key_set();
    c10::DispatchKeySet keys = tls.included_;
    for (const OptTensor* t : tensors)
        if (given(*t)) keys = keys | (*t)->key_set();
    return (keys - tls.excluded_).has_any(watchers);
}

// The tensors of a list; `overridden` where one of them has __torch_function__.
std::vector<Tensor> tensors(PyObject* o, const char* what, bool& overridden) {
    PyObject* seq = PySequence_Fast(o, "");
    if (!seq) {
        PyErr_Clear();
        TORCH_CHECK_TYPE(false, what, ": a list of tensors, got ", Py_TYPE(o)->tp_name);
    }
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
    PyObject** items = PySequence_Fast_ITEMS(seq);
    std::vector<Tensor> got;
    got.reserve(n);
    Py_ssize_t i = 0;
    for (; i < n; ++i) {
        if (!plain_tensor(items[i])) {
            if (!THPVariable_Check(items[i])) break;
            overridden |= has_torch_function(items[i]);
        }
        got.push_back(THPVariable_Unpack(items[i]));
    }
    const char* other = i < n ? Py_TYPE(items[i])->tp_name : nullptr;
    Py_DECREF(seq);
    TORCH_CHECK_TYPE(!other, what, ": tensors, got ", other ? other : "");
    return got;
}

OptTensor tensor_or_none(PyObject* o, const char* what) {
    if (o == Py_None) return std::nullopt;
    TORCH_CHECK_TYPE(THPVariable_Check(o), what, ": a tensor or None, got ", Py_TYPE(o)->tp_name);
    return THPVariable_Unpack(o);
}
OptTensor tensor_or_none(PyObject* o, const char* what, bool& overridden) {
    OptTensor t = tensor_or_none(o, what);
    if (t.has_value()) overridden |= has_torch_function(o);
    return t;
}

double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
}

int64_t integer(PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
}

bool truth(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw python_error();
    return v;
}

struct Released {  // of the interpreter's lock
    PyThreadState* state = PyEval_SaveThread();
    ~Released() { PyEval_RestoreThread(state); }
};

// (bits, params, grads, exp_avgs, exp_avg_sqs, bases, steps, lr, beta1, beta2, eps, weight_decay, maximize, max_norm,
// grad_norm, skip_nonfinite, lr_tensor, seed); bases and seed for 8 bits
PyObject* py_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 18, "step: 18 arguments, got ", n);
    const bool eight = number(a[0]) == 8;
    if (mode_on()) Py_RETURN_NOTIMPLEMENTED;
    bool overridden = false;
    const auto params = tensors(a[1], "parameters", overridden), grads = tensors(a[2], "gradients", overridden);
    const auto avgs = tensors(a[3], "first moments", overridden), sqs = tensors(a[4], "second moments", overridden);
    const auto bases = eight ? tensors(a[5], "bases", overridden) : std::vector<Tensor>();
    const auto steps = tensors(a[6], "steps", overridden);
    const double lr = number(a[7]), b1 = number(a[8]), b2 = number(a[9]), eps = number(a[10]), wd = number(a[11]);
    const bool maximize = truth(a[12]), skip = truth(a[15]);
    const std::optional<double> max_norm = a[13] == Py_None ? std::nullopt : std::optional<double>(number(a[13]));
    const OptTensor norm_in = tensor_or_none(a[14], "grad_norm", overridden);
    const OptTensor rate = tensor_or_none(a[16], "lr", overridden);
    const int64_t seed = eight ? PyLong_AsLongLong(a[17]) : 0;
    if (PyErr_Occurred()) throw python_error();
    if (overridden) Py_RETURN_NOTIMPLEMENTED;
    Tensor norm;
    {
        Released r;
        static auto step32 = op<decltype(adamw_step)>("molix::adamw_step");
        static auto step8 = op<decltype(adamw8_step)>("molix::adamw8_step");
        norm = eight ? step8.call(params, grads, avgs, sqs, bases, steps, lr, b1, b2, eps, wd, maximize, max_norm,
                                  norm_in, skip, rate, seed)
                     : step32.call(params, grads, avgs, sqs, steps, lr, b1, b2, eps, wd, maximize, max_norm, norm_in,
                                   skip, rate);
    }
    if (norm.dim()) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(norm));
    END_HANDLE_TH_ERRORS
}

// (input, normalized_shape, weight, bias, eps): molix.F.layer_norm where the kernels take the arguments as they are,
// else None (the caller reshapes, converts, or says what is wrong)
PyObject* py_layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 5, "layer_norm: 5 arguments, got ", n);
    if (mode_on()) Py_RETURN_NOTIMPLEMENTED;
    for (int k : {0, 2, 3})
        if (a[k] != Py_None && has_torch_function(a[k])) Py_RETURN_NOTIMPLEMENTED;
    if (!THPVariable_Check(a[0])) Py_RETURN_NONE;
    for (int k : {2, 3})
        if (a[k] != Py_None && !THPVariable_Check(a[k])) Py_RETURN_NONE;
    const Tensor& x = THPVariable_Unpack(a[0]);
    PyObject* width = a[1];
    if (PyTuple_Check(width) && PyTuple_GET_SIZE(width) == 1) width = PyTuple_GET_ITEM(width, 0);
    if (!PyLong_Check(width) || !x.is_cuda() || x.dim() < 1 || at::autocast::is_autocast_enabled(at::kCUDA))
        Py_RETURN_NONE;
    const int64_t w = PyLong_AsLongLong(width);
    if (w == -1 && PyErr_Occurred()) throw python_error();
    const int dt = dtype_of(x.scalar_type());
    if (dt < 0 || w != x.size(-1) || w < 1 || w > MNX_LAYER_NORM_MAX_WIDTH) Py_RETURN_NONE;
    const auto argument = [](PyObject* o) { return o == Py_None ? OptTensor() : OptTensor(THPVariable_Unpack(o)); };
    const OptTensor weight = argument(a[2]), bias = argument(a[3]);
    int wd = -1;
    for (const auto* t : {&weight, &bias}) {
        if (!given(*t)) continue;
        const int d = dtype_of((*t)->scalar_type());
        if ((d != dt && d != MNX_F32) || (wd >= 0 && d != wd) || (*t)->dim() != 1 || (*t)->size(0) != w ||
            (*t)->device() != x.device())
            Py_RETURN_NONE;
        wd = d;
    }
    const double eps = number(a[4]);
    Tensor y;
    {
        Released r;
        y = std::get<0>(layer_norm_op().call(x, weight, bias, eps));
    }
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

PyObject* py_grad_norm(PyObject*, PyObject* list) {
    HANDLE_TH_ERRORS
    if (mode_on()) Py_RETURN_NOTIMPLEMENTED;
    bool overridden = false;
    const auto grads = tensors(list, "gradients", overridden);
    if (overridden) Py_RETURN_NOTIMPLEMENTED;
    Tensor norm;
    {
        Released r;
        static auto o = op<decltype(grad_norm)>("molix::grad_norm");
        norm = o.call(grads);
    }
    return THPVariable_Wrap(std::move(norm));
    END_HANDLE_TH_ERRORS
}

PyObject* py_moments(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 5, "moments: 5 lists, got ", n);
    if (mode_on()) Py_RETURN_NOTIMPLEMENTED;
    bool overridden = false;
    const auto avgs = tensors(a[0], "first moments", overridden), sqs = tensors(a[1], "second moments", overridden);
    const auto bases = tensors(a[2], "bases", overridden);
    const auto om = tensors(a[3], "out", overridden), ov = tensors(a[4], "out", overridden);
    if (overridden) Py_RETURN_NOTIMPLEMENTED;
    {
        Released r;
        static auto o = op<decltype(adamw8_moments)>("molix::adamw8_moments");
        o.call(avgs, sqs, bases, om, ov);
    }
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// (x, weight, index, order, starts): molix.F.indexed_linear of rows; index or the plan (order, starts) may be None.  The
// caller has handed over calls that __torch_function__ takes.  None where the grouping has to be an op of its own.
PyObject* py_indexed_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 5, "indexed_linear: 5 arguments, got ", n);
    const OptTensor x = tensor_or_none(a[0], "x"), w = tensor_or_none(a[1], "weight"), z = tensor_or_none(a[2], "index");
    const OptTensor order = tensor_or_none(a[3], "groups"), starts = tensor_or_none(a[4], "groups");
    TORCH_CHECK_TYPE(given(x) && given(w) && (given(z) || (given(order) && given(starts))),
                     "indexed_linear: x, weight and an index or groups");
    TORCH_CHECK(!transformed(), "molix::indexed_linear does not run inside torch.func's transforms");
    Tensor y;
    {
        Released r;
        if (given(order) && given(starts)) {
            y = indexed_linear_op().call(*x, *w, *order, *starts, false);
        } else if (!watched({&x, &w, &z})) {
            check_rows("indexed_linear", "x", *x);
            TORCH_CHECK_VALUE(z->dim() == 1 && z->size(0) == x->size(0) && z->device() == x->device() &&
                                  at::isIntegralType(z->scalar_type(), false),
                              "indexed_linear: index of integers, one a row, on x's device; got ", z->scalar_type(),
                              " ", z->sizes(), " on ", z->device(), " for x ", x->sizes());
            TORCH_CHECK_VALUE(w->dim() == 3 && w->size(0) >= 1 && w->size(0) <= MNX_CLASS_GROUPS_MAX_CLASSES,
                              "indexed_linear: weight (classes, in, out) of 1 to ", MNX_CLASS_GROUPS_MAX_CLASSES,
                              " classes, got ", w->sizes());
            const auto [o, s] = grouped(*z, w->size(0));
            y = indexed_linear_op().call(*x, *w, o, s, false);
        }
    }
    if (!y.defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// (x, steps, a, b, c, eps)
PyObject* py_orthogonalize(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 6, "orthogonalize: 6 arguments, got ", n);
    if (mode_on() || has_torch_function(a[0])) Py_RETURN_NOTIMPLEMENTED;
    TORCH_CHECK_TYPE(THPVariable_Check(a[0]), "orthogonalize: a tensor, got ", Py_TYPE(a[0])->tp_name);
    const Tensor& x = THPVariable_Unpack(a[0]);
    const int64_t steps = integer(a[1]);
    const double c0 = number(a[2]), c1 = number(a[3]), c2 = number(a[4]), eps = number(a[5]);
    Tensor y;
    {
        Released r;
        static auto o = op<decltype(orthogonalize)>("molix::orthogonalize");
        y = o.call(x, steps, c0, c1, c2, eps);
    }
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// (params, grads, momenta, lr, momentum, nesterov, weight_decay, steps, a, b, c, eps, match_rms, maximize, lr_tensor)
PyObject* py_muon(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 15, "muon: 15 arguments, got ", n);
    if (mode_on()) Py_RETURN_NOTIMPLEMENTED;
    bool overridden = false;
    const auto params = tensors(a[0], "parameters", overridden), grads = tensors(a[1], "gradients", overridden);
    const auto momenta = tensors(a[2], "momenta", overridden);
    const double lr = number(a[3]), mu = number(a[4]), wd = number(a[6]);
    const bool nesterov = truth(a[5]), match = truth(a[12]), maximize = truth(a[13]);
    const int64_t steps = integer(a[7]);
    const double c0 = number(a[8]), c1 = number(a[9]), c2 = number(a[10]), eps = number(a[11]);
    const OptTensor rate = tensor_or_none(a[14], "lr", overridden);
    if (overridden) Py_RETURN_NOTIMPLEMENTED;
    {
        Released r;
        static auto o = op<decltype(muon_step)>("molix::muon_step");
        o.call(params, grads, momenta, lr, mu, nesterov, wd, steps, c0, c1, c2, eps, match, maximize, rate);
    }
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

PyMethodDef kMethods[] = {
    {"step", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_step)), METH_FASTCALL,
     "molix::adamw_step or adamw8_step; the norm, or None"},
    {"layer_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_layer_norm)), METH_FASTCALL,
     "molix::layer_norm of the arguments of molix.F.layer_norm, or None"},
    {"grad_norm", py_grad_norm, METH_O, "molix::grad_norm"},
    {"moments", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_moments)), METH_FASTCALL,
     "molix::adamw8_moments"},
    {"indexed_linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_indexed_linear)), METH_FASTCALL,
     "molix::indexed_linear of rows"},
    {"orthogonalize", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_orthogonalize)), METH_FASTCALL,
     "molix::orthogonalize"},
    {"muon", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_muon)), METH_FASTCALL, "molix::muon_step"},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "libmolnex_torch", nullptr, -1, kMethods, nullptr, nullptr, nullptr,
                       nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_libmolnex_torch() { return PyModule_Create(&kModule); }

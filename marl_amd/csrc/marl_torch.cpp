// torch.ops.marl_amd.{gated_linear, residual_norm, keyed_dropout, sample_logits}: schemas, argument checks, shapes on the
// meta device, gradients, and the calls of the C entry points of libmarl_env.so on the tensors' device and its current
// stream.  In C++ because the smallest of these calls take 5 to 10 us on the GPU: a training call through a Python
// autograd function and ctypes took 180 us of the CPU's time.  The library is bound at run time (marl_torch_bind), so
// whichever build of libmarl_env.so the process uses is the one called.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <optional>
#include <string>
#include <tuple>

#include "marl_env.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;
typedef std::tuple<Tensor, Tensor> Tensor2;
typedef std::tuple<Tensor, Tensor, Tensor> Tensor3;
typedef std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> Tensor5;

#define MARL_ENTRY_POINTS(X)                                                                                             \
    X(marl_strerror) X(marl_last_hip_error) X(marl_gated_forward) X(marl_gated_workspace_bytes) X(marl_gated_backward)   \
    X(marl_residual_norm) X(marl_residual_norm_workspace_bytes) X(marl_residual_norm_backward) X(marl_keyed_dropout)     \
    X(marl_sample_logits)
struct Entry {
#define X(name) decltype(&::name) name;
    MARL_ENTRY_POINTS(X)
#undef X
} lib = {};

void check(int rc, const char* what) {
    if (rc == MARL_OK) return;
    TORCH_CHECK(rc != MARL_EHIP, what, ": ", lib.marl_strerror(rc), " (hipError_t ", lib.marl_last_hip_error(), ")");
    TORCH_CHECK(false, what, ": ", lib.marl_strerror(rc));
}

int type_code(const Tensor& t) { return t.scalar_type() == at::kFloat ? MARL_F32 : t.scalar_type() == at::kBFloat16 ? MARL_BF16 : MARL_F16; }

// one supported element type (the optional ones: the same)
void same_type(const char* op, const Tensor& first, std::initializer_list<const Tensor*> rest) {
    const auto t = first.scalar_type();
    TORCH_CHECK_VALUE(t == at::kFloat || t == at::kBFloat16 || t == at::kHalf, op, ": float32, bfloat16 or float16 tensors, not ", t);
    for (const Tensor* r : rest) TORCH_CHECK_VALUE(!r || !r->defined() || r->scalar_type() == t, op, ": all of these tensors must be ", t);
}
// sizes that the C entry points take as 32 bits: refused here, before they are cut (the entry points have limits of their own)
void fits_32(const char* op, std::initializer_list<int64_t> sizes) {
    for (const int64_t n : sizes) TORCH_CHECK_VALUE(n <= INT32_MAX, op, ": rows of at most 2^31 - 1 elements, and as many weight rows");
}
// what forward kept for a backward pass: contiguous, of this shape
void check_kept(const char* op, const Tensor& t, at::IntArrayRef sizes) {
    TORCH_CHECK_VALUE(t.sizes() == sizes && t.is_contiguous(), op, ": tensors kept by forward must be contiguous ", sizes, ", not ", t.sizes());
}
// one HIP device
void same_device(const char* op, const Tensor& first, std::initializer_list<const Tensor*> rest) {
    for (const Tensor* r : rest) TORCH_CHECK_VALUE(!r || !r->defined() || r->device() == first.device(), op, ": tensors on different devices");
    TORCH_CHECK_VALUE(first.is_cuda(), op, ": tensors must be on the HIP device");
}

const Tensor* ptr(const optional<Tensor>& t) { return t.has_value() ? &*t : nullptr; }

// t [..., d] as rows: without a copy if the leading dimensions are evenly spaced and the elements of a row adjacent, as in
// a slice of columns or of one dimension
struct Rows {
    Tensor t;
    int64_t n = 0, ld = 0;
    explicit Rows(const Tensor& in) : t(in) {
        const int64_t d = in.size(-1);
        n = d ? in.numel() / d : 0;
        ld = d;
        if (in.is_contiguous()) return;
        if (in.dim() == 2 && in.stride(1) == 1 && (n == 1 || in.stride(0) >= d)) { if (n > 1) ld = in.stride(0); }
        else t = in.contiguous();
    }
    const void* p() const { return t.const_data_ptr(); }
};

// makes the tensors' device the current one; its current stream
struct On {
    c10::DeviceGuard guard;
    void* stream;
    explicit On(const Tensor& t) : guard(t.device()), stream(c10::hip::getCurrentHIPStream(t.device().index()).stream()) {
        TORCH_CHECK(lib.marl_strerror, "marl_amd: the trunk operators are not bound to libmarl_env.so (import marl_amd.ops binds them)");
    }
};

Tensor scratch(const Tensor& like, size_t bytes) { return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)); }

std::vector<int64_t> with_last(at::IntArrayRef sizes, int64_t last) {
    std::vector<int64_t> s(sizes.begin(), sizes.end());
    s.back() = last;
    return s;
}

// gradients of an operator that is differentiable once: differentiating them again is an error, not a silent zero
variable_list once(variable_list g, const char* op) {
    if (!c10::GradMode::is_enabled()) return g;
    auto error = std::make_shared<torch::autograd::DelayedError>(std::string(op) + " is differentiable once", (int64_t)g.size());
    return (*error)(std::move(g));
}

// the operator of this name and signature, looked up once for every place that names it
#define MARL_OP(name, ...)                                                                                                   \
    ([]() -> const c10::TypedOperatorHandle<__VA_ARGS__>& {                                                                  \
        static const auto h = c10::Dispatcher::singleton().findSchemaOrThrow("marl_amd::" name, "").typed<__VA_ARGS__>();     \
        return h;                                                                                                            \
    }())

// true also for forward-mode tangents, which the autograd functions refuse; below them they would be dropped
bool wants_grad(std::initializer_list<const Tensor*> ts) {
    for (const Tensor* t : ts)
        if (t && t->defined() && ((c10::GradMode::is_enabled() && t->requires_grad()) || t->_fw_grad(0).defined())) return true;
    return false;
}

// -- gated_linear ------------------------------------------------------------------------------------------------------
int act_code(c10::string_view act) {
    const char* names[] = {"silu", "gelu", "relu", "sigmoid"};
    for (int i = 0; i < 4; ++i) if (act == names[i]) return i;
    TORCH_CHECK_VALUE(false, "gated_linear: act must be silu, gelu, relu or sigmoid, not ", act);
}

std::vector<int64_t> check_gated(const Tensor& x, const Tensor& wg, const Tensor& wu, c10::string_view act) {
    act_code(act);
    TORCH_CHECK_VALUE(wg.dim() == 2 && wu.sizes() == wg.sizes(), "gated_linear: w_gate and w_up must be [h, d] of one shape");
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) == wg.size(1), "gated_linear: x must be [..., d] for weights [h, d]");
    TORCH_CHECK_VALUE(wg.size(0) > 0 && wg.size(1) > 0, "gated_linear: weights without elements");
    fits_32("gated_linear", {wg.size(0), wg.size(1)});
    same_type("gated_linear", x, {&wg, &wu});
    return with_last(x.sizes(), wg.size(0));
}

Tensor3 gated_launch(const Tensor& x, const Tensor& wg, const Tensor& wu, c10::string_view act, bool save) {
    const auto shape = check_gated(x, wg, wu, act);
    same_device("gated_linear", x, {&wg, &wu});
    Tensor y = at::empty(shape, x.options()), f, p;
    if (save) { f = at::empty(shape, x.options().dtype(at::kFloat)); p = at::empty_like(f); }
    if (y.numel()) {
        const Rows rx(x), rg(wg), ru(wu);
        const On on(x);
        const int dt = type_code(x);
        const int32_t h = (int32_t)wg.size(0), d = (int32_t)wg.size(1);
        const size_t bytes = lib.marl_gated_workspace_bytes(dt, rx.n, d, h, rx.p(), rx.ld, rg.p(), rg.ld, ru.p(), ru.ld, 0);
        Tensor ws = bytes ? scratch(x, bytes) : Tensor();
        check(lib.marl_gated_forward(dt, act_code(act), rx.n, d, h, rx.p(), rx.ld, rg.p(), rg.ld, ru.p(), ru.ld, y.mutable_data_ptr(),
                                     save ? f.mutable_data_ptr<float>() : nullptr, save ? p.mutable_data_ptr<float>() : nullptr,
                                     bytes ? ws.mutable_data_ptr() : nullptr, on.stream), "marl_gated_forward");
    }
    return {y, f, p};
}
Tensor gated_linear(const Tensor& x, const Tensor& wg, const Tensor& wu, c10::string_view act) { return std::get<0>(gated_launch(x, wg, wu, act, false)); }
Tensor3 gated_linear_saved(const Tensor& x, const Tensor& wg, const Tensor& wu, c10::string_view act) { return gated_launch(x, wg, wu, act, true); }

void check_gated_backward(const Tensor& gy, const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& f, const Tensor& p) {
    const auto shape = check_gated(x, wg, wu, "silu");
    TORCH_CHECK_VALUE(gy.sizes() == at::IntArrayRef(shape), "gated_linear: gy must be shaped like the result");
    check_kept("gated_linear", f, shape);
    check_kept("gated_linear", p, shape);
    TORCH_CHECK_VALUE(f.scalar_type() == at::kFloat && p.scalar_type() == at::kFloat, "gated_linear: f and p must be float32");
    same_type("gated_linear", x, {&gy});
}

Tensor3 gated_linear_backward(const Tensor& gy, const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& f, const Tensor& p, bool need_x, bool need_w) {
    check_gated_backward(gy, x, wg, wu, f, p);
    same_device("gated_linear", x, {&gy, &wg, &wu, &f, &p});
    const int64_t h = wg.size(0), d = wg.size(1);
    Tensor dx = need_x ? at::empty(x.sizes(), x.options()) : at::empty({0}, x.options());
    Tensor dg = need_w ? at::empty({h, d}, x.options()) : at::empty({0}, x.options()), du = at::empty_like(dg);
    if (!x.numel()) return {dx, dg.zero_(), du.zero_()};
    const Rows rx(x), rg(wg), ru(wu), rgy(gy);
    const On on(x);
    const int dt = type_code(x);
    Tensor ws = scratch(x, lib.marl_gated_workspace_bytes(dt, rx.n, (int32_t)d, (int32_t)h, rx.p(), rx.ld, rg.p(), rg.ld, ru.p(), ru.ld, 1));
    check(lib.marl_gated_backward(dt, rx.n, (int32_t)d, (int32_t)h, rx.p(), rx.ld, rg.p(), rg.ld, ru.p(), ru.ld, f.const_data_ptr<float>(),
                                  p.const_data_ptr<float>(), rgy.p(), rgy.ld, need_x ? dx.mutable_data_ptr() : nullptr,
                                  need_w ? dg.mutable_data_ptr() : nullptr, need_w ? du.mutable_data_ptr() : nullptr, ws.mutable_data_ptr(),
                                  on.stream), "marl_gated_backward");
    return {dx, dg, du};
}

Tensor gated_linear_meta(const Tensor& x, const Tensor& wg, const Tensor& wu, c10::string_view act) { return at::empty(check_gated(x, wg, wu, act), x.options()); }
Tensor3 gated_linear_saved_meta(const Tensor& x, const Tensor& wg, const Tensor& wu, c10::string_view act) {
    const Tensor y = gated_linear_meta(x, wg, wu, act);
    return {y, at::empty_like(y, at::kFloat), at::empty_like(y, at::kFloat)};
}
Tensor3 gated_linear_backward_meta(const Tensor& gy, const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& f, const Tensor& p, bool need_x, bool need_w) {
    check_gated_backward(gy, x, wg, wu, f, p);
    const auto w = [&] { return need_w ? at::empty(wg.sizes(), x.options()) : at::empty({0}, x.options()); };
    return {need_x ? at::empty(x.sizes(), x.options()) : at::empty({0}, x.options()), w(), w()};
}

struct GatedLinear : torch::autograd::Function<GatedLinear> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu, std::string act) {
        at::AutoDispatchBelowADInplaceOrView below;
        auto [y, f, p] = MARL_OP("gated_linear_saved", Tensor3(const Tensor&, const Tensor&, const Tensor&, c10::string_view)).call(x, wg, wu, act);
        ctx->save_for_backward({x, wg, wu, f, p});
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        const auto s = ctx->get_saved_variables();
        const bool nx = ctx->needs_input_grad(0), ng = ctx->needs_input_grad(1), nu = ctx->needs_input_grad(2);
        auto [dx, dg, du] = MARL_OP("gated_linear_backward", Tensor3(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, bool, bool)).call(g[0], s[0], s[1], s[2], s[3], s[4], nx, ng || nu);
        return once({nx ? dx : Tensor(), ng ? dg : Tensor(), nu ? du : Tensor(), Tensor()}, "gated_linear");
    }
};
Tensor gated_linear_autograd(const Tensor& x, const Tensor& wg, const Tensor& wu, c10::string_view act) {
    if (wants_grad({&x, &wg, &wu})) return GatedLinear::apply(x, wg, wu, std::string(act));
    at::AutoDispatchBelowADInplaceOrView below;
    return MARL_OP("gated_linear", Tensor(const Tensor&, const Tensor&, const Tensor&, c10::string_view)).call(x, wg, wu, act);
}

// -- residual_norm -----------------------------------------------------------------------------------------------------
int kind_code(c10::string_view kind) {
    TORCH_CHECK_VALUE(kind == "rms" || kind == "layer", "residual_norm: kind must be rms or layer, not ", kind);
    return kind == "rms" ? MARL_NORM_RMS : MARL_NORM_LAYER;
}

void check_norm(const Tensor& x, const Tensor& block, const Tensor& wpost, const Tensor& wpre, const optional<Tensor>& gate, double eps, c10::string_view kind) {
    kind_code(kind);
    TORCH_CHECK_VALUE(x.dim() >= 1 && block.sizes() == x.sizes(), "residual_norm: x and block must be [..., d] of one shape");
    const int64_t d = x.size(-1);
    TORCH_CHECK_VALUE(d > 0 && d <= MARL_MAX_NORM_WIDTH, "residual_norm: rows of 1 to ", MARL_MAX_NORM_WIDTH, " elements, not ", d);
    TORCH_CHECK_VALUE(wpost.dim() == 1 && wpost.size(0) == d && wpre.sizes() == wpost.sizes(), "residual_norm: w_post and w_pre must be [d]");
    TORCH_CHECK_VALUE(!gate || gate->sizes() == wpost.sizes() || gate->sizes() == x.sizes(), "residual_norm: gate must be [d] or shaped like x");
    TORCH_CHECK_VALUE(eps >= 0.0, "residual_norm: eps must not be negative");
    same_type("residual_norm", x, {&block, &wpost, &wpre, ptr(gate)});
}

// the gate's rows: stride 0 for one gate for all rows
struct GateRows {
    Tensor t;
    int64_t ld = 0;
    GateRows(const optional<Tensor>& gate, const Tensor& x) {
        if (!gate) return;
        if (gate->dim() == 1 && x.dim() > 1) { t = gate->contiguous(); return; }
        const Rows r(*gate);
        t = r.t;
        ld = r.ld;
    }
    const void* p() const { return t.defined() ? t.const_data_ptr() : nullptr; }
};

Tensor3 norm_launch(const Tensor& x, const Tensor& block, const Tensor& wpost, const Tensor& wpre, const optional<Tensor>& gate, double scale, double eps, c10::string_view kind, bool save) {
    check_norm(x, block, wpost, wpre, gate, eps, kind);
    same_device("residual_norm", x, {&block, &wpost, &wpre, ptr(gate)});
    Tensor y = at::empty(x.sizes(), x.options()), n = at::empty(x.sizes(), x.options()), stats;
    if (save) stats = at::empty(with_last(x.sizes(), 4), x.options().dtype(at::kFloat));
    if (x.numel()) {
        const Rows rx(x), rb(block);
        const GateRows g(gate, x);
        const Tensor wo = wpost.contiguous(), wr = wpre.contiguous();
        const On on(x);
        check(lib.marl_residual_norm(type_code(x), kind_code(kind), rx.n, (int32_t)x.size(-1), rx.p(), rx.ld, rb.p(), rb.ld, wo.const_data_ptr(),
                                     wr.const_data_ptr(), g.p(), g.ld, (float)scale, (float)eps, y.mutable_data_ptr(), n.mutable_data_ptr(),
                                     save ? stats.mutable_data_ptr<float>() : nullptr, on.stream), "marl_residual_norm");
    }
    return {y, n, stats};
}
Tensor2 residual_norm(const Tensor& x, const Tensor& block, const Tensor& wpost, const Tensor& wpre, const optional<Tensor>& gate, double scale, double eps, c10::string_view kind) {
    auto [y, n, s] = norm_launch(x, block, wpost, wpre, gate, scale, eps, kind, false);
    return {y, n};
}
Tensor3 residual_norm_saved(const Tensor& x, const Tensor& block, const Tensor& wpost, const Tensor& wpre, const optional<Tensor>& gate, double scale, double eps, c10::string_view kind) {
    return norm_launch(x, block, wpost, wpre, gate, scale, eps, kind, true);
}

// x: contiguous, as the entry point takes it
void check_norm_backward(const optional<Tensor>& gy, const optional<Tensor>& gn, const Tensor& x, const Tensor& block, const Tensor& wpost,
                         const Tensor& wpre, const optional<Tensor>& gate, const Tensor& stats, c10::string_view kind) {
    check_norm(x, block, wpost, wpre, gate, 0.0, kind);
    for (const Tensor* g : {ptr(gy), ptr(gn)})
        TORCH_CHECK_VALUE(!g || !g->defined() || g->sizes() == x.sizes(), "residual_norm: gy and gn must be shaped like the results");
    check_kept("residual_norm", x, x.sizes());
    check_kept("residual_norm", stats, with_last(x.sizes(), 4));
    TORCH_CHECK_VALUE(stats.scalar_type() == at::kFloat, "residual_norm: stats must be float32");
    same_type("residual_norm", x, {ptr(gy), ptr(gn)});
}

Tensor5 residual_norm_backward(const optional<Tensor>& gy, const optional<Tensor>& gn, const Tensor& x, const Tensor& block, const Tensor& wpost,
                               const Tensor& wpre, const optional<Tensor>& gate, const Tensor& stats, double scale, c10::string_view kind) {
    check_norm_backward(gy, gn, x, block, wpost, wpre, gate, stats, kind);
    same_device("residual_norm", x, {ptr(gy), ptr(gn), &block, &wpost, &wpre, ptr(gate), &stats});
    const int64_t d = x.size(-1);
    Tensor dx = at::empty(x.sizes(), x.options()), db = at::empty(x.sizes(), x.options()), dpost = at::empty({d}, x.options()), dpre = at::empty({d}, x.options());
    Tensor dgate = gate ? at::empty(gate->sizes(), x.options()) : at::empty({0}, x.options());
    if (!x.numel()) return {dx, db, dpost.zero_(), dpre.zero_(), dgate.zero_()};
    const Rows rb(block);
    const GateRows g(gate, x);
    const Tensor wo = wpost.contiguous(), wr = wpre.contiguous();
    optional<Rows> ry, rn;
    if (gy && gy->defined()) ry.emplace(*gy);
    if (gn && gn->defined()) rn.emplace(*gn);
    const On on(x);
    Tensor ws = scratch(x, lib.marl_residual_norm_workspace_bytes((int32_t)d));
    check(lib.marl_residual_norm_backward(type_code(x), kind_code(kind), rb.n, (int32_t)d, x.const_data_ptr(), rb.p(), rb.ld, wo.const_data_ptr(),
                                          wr.const_data_ptr(), g.p(), g.ld, stats.const_data_ptr<float>(), ry ? ry->p() : nullptr, ry ? ry->ld : 0,
                                          rn ? rn->p() : nullptr, rn ? rn->ld : 0, (float)scale, dx.mutable_data_ptr(), db.mutable_data_ptr(),
                                          dpost.mutable_data_ptr(), dpre.mutable_data_ptr(), gate ? dgate.mutable_data_ptr() : nullptr,
                                          ws.mutable_data_ptr(), on.stream), "marl_residual_norm_backward");
    return {dx, db, dpost, dpre, dgate};
}

Tensor2 residual_norm_meta(const Tensor& x, const Tensor& block, const Tensor& wpost, const Tensor& wpre, const optional<Tensor>& gate, double, double eps, c10::string_view kind) {
    check_norm(x, block, wpost, wpre, gate, eps, kind);
    return {at::empty(x.sizes(), x.options()), at::empty(x.sizes(), x.options())};
}
Tensor3 residual_norm_saved_meta(const Tensor& x, const Tensor& block, const Tensor& wpost, const Tensor& wpre, const optional<Tensor>& gate, double scale, double eps, c10::string_view kind) {
    auto [y, n] = residual_norm_meta(x, block, wpost, wpre, gate, scale, eps, kind);
    return {y, n, at::empty(with_last(x.sizes(), 4), x.options().dtype(at::kFloat))};
}
Tensor5 residual_norm_backward_meta(const optional<Tensor>& gy, const optional<Tensor>& gn, const Tensor& x, const Tensor& block, const Tensor& wpost, const Tensor& wpre,
                                    const optional<Tensor>& gate, const Tensor& stats, double, c10::string_view kind) {
    check_norm_backward(gy, gn, x, block, wpost, wpre, gate, stats, kind);
    return {at::empty(x.sizes(), x.options()), at::empty(x.sizes(), x.options()), at::empty(wpost.sizes(), x.options()), at::empty(wpost.sizes(), x.options()),
            gate ? at::empty(gate->sizes(), x.options()) : at::empty({0}, x.options())};
}

struct ResidualNorm : torch::autograd::Function<ResidualNorm> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& block, const Tensor& wpost, const Tensor& wpre, const optional<Tensor>& gate, double scale, double eps, std::string kind) {
        at::AutoDispatchBelowADInplaceOrView below;
        auto [y, n, stats] = MARL_OP("residual_norm_saved", Tensor3(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const optional<Tensor>&, double, double, c10::string_view)).call(x, block, wpost, wpre, gate, scale, eps, kind);
        ctx->save_for_backward({x, block, wpost, wpre, gate ? *gate : Tensor(), stats});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["kind"] = kind;
        ctx->set_materialize_grads(false);
        return {y, n};
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        if (!g[0].defined() && !g[1].defined()) return variable_list(8);
        const auto s = ctx->get_saved_variables();
        const auto given = [](const Tensor& t) { return t.defined() ? optional<Tensor>(t) : optional<Tensor>(); };
        auto [dx, db, dpost, dpre, dgate] = MARL_OP("residual_norm_backward", Tensor5(const optional<Tensor>&, const optional<Tensor>&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const optional<Tensor>&, const Tensor&, double, c10::string_view)).call(given(g[0]), given(g[1]), s[0].contiguous(), s[1], s[2], s[3], given(s[4]), s[5], ctx->saved_data["scale"].toDouble(), ctx->saved_data["kind"].toStringRef());
        variable_list out = {dx, db, dpost, dpre, s[4].defined() ? dgate : Tensor(), Tensor(), Tensor(), Tensor()};
        for (size_t i = 0; i < (s[4].defined() ? 5 : 4); ++i) if (!ctx->needs_input_grad(i)) out[i] = Tensor();
        return once(std::move(out), "residual_norm");
    }
};
Tensor2 residual_norm_autograd(const Tensor& x, const Tensor& block, const Tensor& wpost, const Tensor& wpre, const optional<Tensor>& gate, double scale, double eps, c10::string_view kind) {
    if (wants_grad({&x, &block, &wpost, &wpre, ptr(gate)})) {
        auto o = ResidualNorm::apply(x, block, wpost, wpre, gate, scale, eps, std::string(kind));
        return {o[0], o[1]};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    return MARL_OP("residual_norm", Tensor2(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const optional<Tensor>&, double, double, c10::string_view)).call(x, block, wpost, wpre, gate, scale, eps, kind);
}

// -- keyed_dropout -----------------------------------------------------------------------------------------------------
void check_dropout(const Tensor& x, double p, const optional<Tensor>& keys) {
    TORCH_CHECK_VALUE(x.dim() >= 1 && p >= 0.0 && p <= 1.0, "keyed_dropout: x must be [..., d] and p in [0, 1]");
    TORCH_CHECK_VALUE(!keys || (keys->scalar_type() == at::kLong && keys->sizes() == x.sizes().slice(0, x.dim() - 1)),
                      "keyed_dropout: keys must be int64, one per row of x");
    same_type("keyed_dropout", x, {});
    fits_32("keyed_dropout", {x.size(-1)});
}
Tensor keyed_dropout(const Tensor& x, double p, int64_t seed, const optional<Tensor>& keys) {
    check_dropout(x, p, keys);
    same_device("keyed_dropout", x, {ptr(keys)});
    Tensor y = at::empty(x.sizes(), x.options());
    if (x.numel()) {
        const Rows rx(x);
        const Tensor k = keys ? keys->contiguous() : Tensor();
        const On on(x);
        check(lib.marl_keyed_dropout(type_code(x), rx.n, (int32_t)x.size(-1), rx.p(), rx.ld, y.mutable_data_ptr(), keys ? k.const_data_ptr<int64_t>() : nullptr,
                                     p, (uint64_t)seed, on.stream), "marl_keyed_dropout");
    }
    return y;
}
Tensor keyed_dropout_meta(const Tensor& x, double p, int64_t, const optional<Tensor>& keys) {
    check_dropout(x, p, keys);
    return at::empty(x.sizes(), x.options());
}
Tensor call_dropout(const Tensor& x, double p, int64_t seed, const optional<Tensor>& keys) {
    return MARL_OP("keyed_dropout", Tensor(const Tensor&, double, int64_t, const optional<Tensor>&)).call(x, p, seed, keys);
}
struct KeyedDropout : torch::autograd::Function<KeyedDropout> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, double p, int64_t seed, const optional<Tensor>& keys) {
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->save_for_backward({keys ? *keys : Tensor()});
        ctx->saved_data["p"] = p;
        ctx->saved_data["seed"] = seed;
        return call_dropout(x, p, seed, keys);
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {          // linear in x: differentiable again
        const auto keys = ctx->get_saved_variables()[0];
        return {call_dropout(g[0], ctx->saved_data["p"].toDouble(), ctx->saved_data["seed"].toInt(), keys.defined() ? optional<Tensor>(keys) : optional<Tensor>()),
                Tensor(), Tensor(), Tensor()};
    }
};
Tensor keyed_dropout_autograd(const Tensor& x, double p, int64_t seed, const optional<Tensor>& keys) {
    if (wants_grad({&x})) return KeyedDropout::apply(x, p, seed, keys);
    at::AutoDispatchBelowADInplaceOrView below;
    return call_dropout(x, p, seed, keys);
}

// -- sample_logits -----------------------------------------------------------------------------------------------------
void check_sample(const Tensor& logits, const Tensor& u, double temperature, int64_t top_k, double top_p, double min_p, const optional<Tensor>& settings) {
    const int64_t V = logits.dim() ? logits.size(-1) : 0;
    TORCH_CHECK_VALUE(V > 0 && V <= MARL_MAX_CHOICES, "sample_logits: logits must be [..., V] with V from 1 to ", MARL_MAX_CHOICES);
    const auto lead = logits.sizes().slice(0, logits.dim() - 1);
    TORCH_CHECK_VALUE(u.scalar_type() == at::kFloat && u.sizes() == lead, "sample_logits: u must be float32, one number per row");
    if (settings) {
        TORCH_CHECK_VALUE(settings->scalar_type() == at::kFloat && settings->sizes() == at::IntArrayRef(with_last(logits.sizes(), 4)),
                          "sample_logits: settings must be float32 [..., 4]: temperature, top_k, top_p, min_p of every row");
    } else {
        TORCH_CHECK_VALUE(temperature >= 0.0 && top_k >= 0 && top_p > 0.0 && min_p >= 0.0 && min_p <= 1.0,
                          "sample_logits: temperature >= 0, top_k >= 0, top_p > 0 and min_p in [0, 1]");
    }
    same_type("sample_logits", logits, {});
}
Tensor2 sample_logits(const Tensor& logits, const Tensor& u, double temperature, int64_t top_k, double top_p, double min_p, const optional<Tensor>& settings) {
    check_sample(logits, u, temperature, top_k, top_p, min_p, settings);
    same_device("sample_logits", logits, {&u, ptr(settings)});
    Tensor index = at::empty(u.sizes(), u.options().dtype(at::kLong)), log_prob = at::empty(u.sizes(), u.options());
    if (u.numel()) {
        const Rows r(logits);
        const Tensor uc = u.contiguous(), s = settings ? settings->contiguous() : Tensor();
        const On on(logits);
        check(lib.marl_sample_logits(type_code(logits), r.n, (int32_t)logits.size(-1), r.p(), r.ld, uc.const_data_ptr<float>(), (float)temperature,
                                     (int32_t)std::min<int64_t>(top_k, MARL_MAX_CHOICES), (float)top_p, (float)min_p,
                                     settings ? s.const_data_ptr<float>() : nullptr, index.mutable_data_ptr<int64_t>(), log_prob.mutable_data_ptr<float>(),
                                     on.stream), "marl_sample_logits");
    }
    return {index, log_prob};
}
Tensor2 sample_logits_meta(const Tensor& logits, const Tensor& u, double temperature, int64_t top_k, double top_p, double min_p, const optional<Tensor>& settings) {
    check_sample(logits, u, temperature, top_k, top_p, min_p, settings);
    return {at::empty(u.sizes(), u.options().dtype(at::kLong)), at::empty(u.sizes(), u.options())};
}
// not differentiable: its outputs are constants to autograd
Tensor2 sample_logits_autograd(const Tensor& logits, const Tensor& u, double temperature, int64_t top_k, double top_p, double min_p, const optional<Tensor>& settings) {
    at::AutoDispatchBelowADInplaceOrView below;
    return MARL_OP("sample_logits", Tensor2(const Tensor&, const Tensor&, double, int64_t, double, double, const optional<Tensor>&)).call(logits, u, temperature, top_k, top_p, min_p, settings);
}

}  // namespace

// The C entry points from the library at `path` (already loaded by the caller or not).  0, or -1 if it lacks one.
extern "C" __attribute__((visibility("default"))) int marl_torch_bind(const char* path) {
    void* so = dlopen(path, RTLD_NOW | RTLD_LOCAL);
    if (!so) return -1;
    Entry e = {};
#define X(name) if (!(e.name = (decltype(e.name))dlsym(so, #name))) return -1;
    MARL_ENTRY_POINTS(X)
#undef X
    lib = e;
    return 0;
}

TORCH_LIBRARY_FRAGMENT(marl_amd, m) {
    m.def("gated_linear(Tensor x, Tensor w_gate, Tensor w_up, str act=\"silu\") -> Tensor");
    m.def("gated_linear_saved(Tensor x, Tensor w_gate, Tensor w_up, str act) -> (Tensor, Tensor, Tensor)");
    m.def("gated_linear_backward(Tensor gy, Tensor x, Tensor w_gate, Tensor w_up, Tensor f, Tensor p, bool need_x, bool need_w) -> (Tensor, Tensor, Tensor)");
    m.def("residual_norm(Tensor x, Tensor block, Tensor w_post, Tensor w_pre, Tensor? gate=None, float scale=1.0, float eps=1e-5, str kind=\"rms\") -> (Tensor, Tensor)");
    m.def("residual_norm_saved(Tensor x, Tensor block, Tensor w_post, Tensor w_pre, Tensor? gate, float scale, float eps, str kind) -> (Tensor, Tensor, Tensor)");
    m.def("residual_norm_backward(Tensor? gy, Tensor? gn, Tensor x, Tensor block, Tensor w_post, Tensor w_pre, Tensor? gate, Tensor stats, float scale, str kind)"
          " -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
    m.def("keyed_dropout(Tensor x, float p, int seed, Tensor? keys=None) -> Tensor");
    m.def("sample_logits(Tensor logits, Tensor u, float temperature=1.0, int top_k=0, float top_p=1.0, float min_p=0.0, *, Tensor? settings=None) -> (Tensor, Tensor)");
}
#define MARL_IMPL(m, name, fn) m.impl(name, TORCH_FN(fn))
#define MARL_ALL(m, suffix)                                              \
    MARL_IMPL(m, "gated_linear", gated_linear##suffix);                  \
    MARL_IMPL(m, "gated_linear_saved", gated_linear_saved##suffix);      \
    MARL_IMPL(m, "gated_linear_backward", gated_linear_backward##suffix); \
    MARL_IMPL(m, "residual_norm", residual_norm##suffix);                \
    MARL_IMPL(m, "residual_norm_saved", residual_norm_saved##suffix);    \
    MARL_IMPL(m, "residual_norm_backward", residual_norm_backward##suffix); \
    MARL_IMPL(m, "keyed_dropout", keyed_dropout##suffix);                \
    MARL_IMPL(m, "sample_logits", sample_logits##suffix);
TORCH_LIBRARY_IMPL(marl_amd, CUDA, m) { MARL_ALL(m, ) }
TORCH_LIBRARY_IMPL(marl_amd, Meta, m) { MARL_ALL(m, _meta) }
// on CPU tensors: the checks of the arguments, then the refusal of the device
TORCH_LIBRARY_IMPL(marl_amd, CPU, m) {
    MARL_IMPL(m, "gated_linear", gated_linear);
    MARL_IMPL(m, "residual_norm", residual_norm);
    MARL_IMPL(m, "keyed_dropout", keyed_dropout);
    MARL_IMPL(m, "sample_logits", sample_logits);
}
TORCH_LIBRARY_IMPL(marl_amd, AutogradCUDA, m) {
    MARL_IMPL(m, "gated_linear", gated_linear_autograd);
    MARL_IMPL(m, "residual_norm", residual_norm_autograd);
    MARL_IMPL(m, "keyed_dropout", keyed_dropout_autograd);
    MARL_IMPL(m, "sample_logits", sample_logits_autograd);
}

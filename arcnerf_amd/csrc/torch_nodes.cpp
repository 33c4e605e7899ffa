// The residual feed-forward layers as autograd nodes: layer_norm, linear_act_residual and gated_ffn on torch tensors, over the C entry points of
// include/arcnerf_hip.h.  Python calls these through arcnerf_amd.ops.autograd, which documents them.
//
// Why native: at the sizes of one training chunk's small nets a Python autograd.Function spends more time than its kernels (layer norm of
// 20011 x 319 f16, forward + backward: 48 us of kernels, 143 us a pass from Python nodes), most of it in the backward, which the engine runs
// on a thread of its own that has to take the interpreter lock.
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <cstdlib>
#include <cstring>
#include <limits>
#include <string>

#include "../../include/arcnerf_hip.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::tensor_list;

void call(int rc, const char *what) { TORCH_CHECK(rc == ARCN_OK, "arcnerf_hip ", what, " failed (rc=", rc, "): ", arcn_last_error()); }

int type_code(const Tensor &t, const char *name) {
    switch (t.scalar_type()) {
    case at::kFloat: return ARCN_DTYPE_F32;
    case at::kBFloat16: return ARCN_DTYPE_BF16;
    case at::kHalf: return ARCN_DTYPE_F16;
    default: TORCH_CHECK(false, "arcnerf_amd: ", name, " is ", t.scalar_type(), "; float32, bfloat16 and float16 are taken");
    }
    return -1;
}

// an output every element of which is written (ARCN_POISON_OUTPUTS=1, a test aid: NaN first)
Tensor fresh(at::IntArrayRef shape, const Tensor &like, at::ScalarType type) {
    static const bool poison = [] {
        const char *e = std::getenv("ARCN_POISON_OUTPUTS");
        return e && std::strcmp(e, "1") == 0;
    }();
    Tensor t = at::empty(shape, like.options().dtype(type));
    if (poison) t.fill_(std::numeric_limits<double>::quiet_NaN());
    return t;
}
Tensor fresh(at::IntArrayRef shape, const Tensor &like) { return fresh(shape, like, like.scalar_type()); }
Tensor scratch_floats(int64_t n, const Tensor &like) { return at::empty({n}, like.options().dtype(at::kFloat)); }

// t with its numbers in memory as they are (the imaginary part of a conjugate is a view that says "negated")
Tensor plain(const Tensor &t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }
Tensor packed(const Tensor &t) { return t.defined() ? plain(t).contiguous() : t; }

// (..., width) as rows: a column slice of a wider buffer as it is, anything else contiguous
struct Rows {
    Tensor t;
    int64_t n = 0, ld = 0;
    const void *p() const { return t.const_data_ptr(); }
};
Rows rows_of(const char *name, const Tensor &t, int64_t width, const Tensor &like) {
    TORCH_CHECK(t.is_cuda(), "arcnerf_amd ops run on the GPU only (got a ", t.device(), " ", name, "); there is no CPU fallback");
    TORCH_CHECK(t.dim() >= 1 && t.size(-1) == width && width >= 1 && width <= (1 << 24), "arcnerf_amd: ", name, " must be (..., ", width, "), got ", t.sizes());
    TORCH_CHECK(t.scalar_type() == like.scalar_type() && t.device() == like.device(), "arcnerf_amd: ", name, " is ", t.scalar_type(), " on ", t.device(),
                ", not ", like.scalar_type(), " on ", like.device());
    Rows r;
    r.t = plain(t);
    if (r.t.dim() == 2 && (r.t.stride(1) == 1 || width == 1) && (r.t.stride(0) >= width || r.t.size(0) <= 1)) {
        r.n = r.t.size(0);
        r.ld = r.n > 1 ? r.t.stride(0) : width;
        return r;
    }
    r.t = r.t.contiguous();
    r.n = r.t.numel() / width;
    r.ld = width;
    return r;
}

// a contiguous parameter of the rows' device and type (or f32 where `or_f32`)
Tensor param(const char *name, const Tensor &t, at::IntArrayRef shape, const Tensor &like, bool or_f32 = false) {
    if (!t.defined()) return t;
    TORCH_CHECK(t.sizes() == shape && t.device() == like.device() && (t.scalar_type() == like.scalar_type() || (or_f32 && t.scalar_type() == at::kFloat)),
                "arcnerf_amd: ", name, " must be ", shape, " ", like.scalar_type(), or_f32 ? " or float32" : "", " on ", like.device(), ", got ", t.sizes(), " ",
                t.scalar_type(), " on ", t.device());
    return packed(t);
}
const void *ptr(const Tensor &t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void *out_ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

void check_like(const char *name, const Tensor &t, at::IntArrayRef shape) {
    TORCH_CHECK(!t.defined() || t.sizes() == shape, "arcnerf_amd: the ", name, " must be ", shape, ", got ", t.sizes());
}

std::vector<int64_t> with_last(const Tensor &x, int64_t n) {
    std::vector<int64_t> s = x.sizes().vec();
    TORCH_CHECK(!s.empty() && n <= (1 << 24), "arcnerf_amd: x must be (..., width) and a width at most 2^24, got ", x.sizes(), " and ", n);
    s.back() = n;
    return s;
}

// launches of a call: on its tensors' device, whatever the current one is, on that device's current stream
struct Launch {
    c10::DeviceGuard guard;
    void *stream;
    explicit Launch(const Tensor &t) : guard(t.device()), stream(c10::hip::getCurrentHIPStream(t.device().index()).stream()) {}
};

// First order only: where a graph of the gradients is asked for they hang on a node that raises.  Its edges lead to everything that the
// gradients depend on (`from`: what the node saved and the gradient that came in), so that a differentiation which asks for any of these
// runs it, also one with other paths to them (a loss that has terms in both the result and its gradient, a list of inputs).
tensor_list first_order(tensor_list grads, bool graph, const char *what, const tensor_list &from) {
    if (!graph) return grads;
    auto err = std::make_shared<torch::autograd::Error>(std::string("arcnerf_amd: ") + what + " can be differentiated once only", torch::autograd::collect_next_edges(from));
    for (Tensor &g : grads)
        if (g.defined()) {
            g = g.detach();
            torch::autograd::set_history(g, err);
        }
    return grads;
}

bool needs_graph(std::initializer_list<const Tensor *> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor *t : ts)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// The kernels are launched on raw pointers: a tangent would be dropped without a word, and a trace would record the allocation of a result and
// nothing that fills it.
void refuse_untracked(std::initializer_list<const Tensor *> ts, const char *what) {
    TORCH_CHECK(!torch::jit::tracer::isTracing() && !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value() &&
                    !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch),
                "arcnerf_amd: ", what, " cannot be traced (torch.jit.trace, make_fx)");
    for (const Tensor *t : ts)
        TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), "arcnerf_amd: ", what, " has no forward-mode derivative");
}

// which inputs of a node want a gradient: its edges are those of the tensors that were given, in order
std::vector<int64_t> edges(std::initializer_list<const Tensor *> ts) {
    std::vector<int64_t> e;
    int64_t n = 0;
    for (const Tensor *t : ts) e.push_back(t->defined() ? n++ : -1);
    return e;
}
struct Needs {
    AutogradContext *ctx;
    std::vector<int64_t> e;
    explicit Needs(AutogradContext *c) : ctx(c), e(c->saved_data["edges"].toIntVector()) {}
    bool operator()(size_t k) const { return e[k] >= 0 && ctx->needs_input_grad((size_t)e[k]); }
};
OptTensor opt(const Tensor &t) { return t.defined() ? OptTensor(t) : OptTensor(); }

// ---- layer norm -----------------------------------------------------------------------------------------------------------------------
Tensor norm_forward(const Tensor &x, const Tensor &w, const Tensor &b, double eps, Tensor *stats) {
    const int64_t C = x.dim() ? x.size(-1) : 0;
    const Rows r = rows_of("x", x, C, x);
    const int dt = type_code(x, "x");
    const Tensor wc = param("weight", w, {C}, x, true), bc = param("bias", b, {C}, x, true);
    TORCH_CHECK(!w.defined() || !b.defined() || w.scalar_type() == b.scalar_type(), "arcnerf_amd: weight and bias must be of one type");
    Tensor y = fresh(x.sizes(), x);
    if (stats) *stats = fresh({r.n, 2}, x, at::kFloat);
    Launch go(x);
    call(arcn_layer_norm_fwd(r.p(), r.ld, ptr(wc), ptr(bc), dt, w.defined() ? type_code(w, "weight") : b.defined() ? type_code(b, "bias") : dt, (float)eps,
                             y.data_ptr(), stats ? stats->data_ptr<float>() : nullptr, r.n, (int)C, go.stream),
         "layer_norm_fwd");
    return y;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const OptTensor &w_, const OptTensor &b_, double eps) {
        const Tensor w = w_.value_or(Tensor()), b = b_.value_or(Tensor());
        ctx->saved_data["edges"] = edges({&x, &w, &b});
        Tensor stats;
        Tensor y = norm_forward(x, w, b, eps, &stats);
        ctx->save_for_backward({x, w, stats});
        ctx->saved_data["param_type"] = (int64_t)(w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : x.scalar_type());
        return y;
    }
    static tensor_list backward(AutogradContext *ctx, tensor_list g) {
        const bool graph = at::GradMode::is_enabled();
        at::NoGradGuard no_grad;
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w = saved[1], &stats = saved[2];
        const int64_t C = x.size(-1);
        const auto wt = (at::ScalarType)ctx->saved_data["param_type"].toInt();
        const Needs need(ctx);
        const bool want_dw = need(1), want_db = need(2);
        tensor_list out(4);
        if (need(0)) out[0] = fresh(x.sizes(), x);
        if (want_dw) out[1] = fresh({C}, x, wt);
        if (want_db) out[2] = fresh({C}, x, wt);
        const Rows r = rows_of("x", x, C, x), dy = rows_of("dy", g[0], C, x);
        if (r.n == 0) {
            for (int k : {1, 2})
                if (out[k].defined()) out[k].zero_();
            return first_order(std::move(out), graph, "layer_norm", {x, w, g[0]});
        }
        const int dt = type_code(x, "x");
        const Tensor wc = packed(w);
        const int64_t nf = want_dw || want_db ? arcn_layer_norm_bwd_scratch_floats(r.n, (int)C, dt) : 0;
        const Tensor scratch = nf ? scratch_floats(nf, x) : Tensor();
        Launch go(x);
        call(arcn_layer_norm_bwd(r.p(), r.ld, dy.p(), dy.ld, ptr(wc), stats.const_data_ptr<float>(), dt, wt == x.scalar_type() ? dt : ARCN_DTYPE_F32,
                                 out_ptr(out[0]), out_ptr(out[1]), out_ptr(out[2]), (float *)out_ptr(scratch), nf, r.n, (int)C, go.stream),
             "layer_norm_bwd");
        return first_order(std::move(out), graph, "layer_norm", {x, w, g[0]});
    }
};

Tensor layer_norm(const Tensor &x, const OptTensor &w_, const OptTensor &b_, double eps) {
    const Tensor w = w_.value_or(Tensor()), b = b_.value_or(Tensor());
    refuse_untracked({&x, &w, &b}, "layer_norm");
    return needs_graph({&x, &w, &b}) ? LayerNorm::apply(x, opt(w), opt(b), eps) : norm_forward(x, w, b, eps, nullptr);
}

// ---- dense layer ------------------------------------------------------------------------------------------------------------------------
Tensor dense_forward(const Tensor &x, const Tensor &w, const Tensor &b, const Tensor &res, int64_t act, double beta) {
    TORCH_CHECK(w.dim() == 2, "arcnerf_amd: weight must be (N, K), got ", w.sizes());
    const int64_t N = w.size(0), K = w.size(1);
    const Rows r = rows_of("x", x, K, x);
    const int dt = type_code(x, "x");
    const Tensor wc = param("weight", w, {N, K}, x), bc = param("bias", b, {N}, x);
    Tensor y = fresh(with_last(x, N), x);
    check_like("residual", res, y.sizes());
    const Rows rr = res.defined() ? rows_of("residual", res, N, x) : Rows();
    Launch go(x);
    call(arcn_dense_fwd(r.p(), r.ld, ptr(wc), ptr(bc), ptr(rr.t), rr.ld, y.data_ptr(), dt, (int)act, (float)beta, r.n, (int)K, (int)N, go.stream), "dense_fwd");
    return y;
}

// The column sums of dz, made where it is still in f32: of the 16-bit types, where a bias's gradient is wanted
struct BiasSums {
    Tensor t;
    int64_t n = 0;
    BiasSums() = default;
    BiasSums(bool want, int64_t rows, int64_t N, const Tensor &like) {
        if (want && like.scalar_type() != at::kFloat) t = scratch_floats(arcn_bias_sums_floats(rows, (int)N), like);
    }
    float *p() const { return (float *)out_ptr(t); }
    int64_t floats() const { return t.defined() ? t.numel() : 0; }
};

// dw (N, K) = dz^T x, db = column sums of dz (or undefined), as `sums` has them or its own
std::pair<Tensor, Tensor> dense_dw(const Rows &dz, int64_t N, const Rows &x, int64_t K, bool want_db, const BiasSums &sums, int dt, void *stream) {
    Tensor dw = fresh({N, K}, x.t), db = want_db ? fresh({N}, x.t) : Tensor();
    const int64_t nf = arcn_dense_dw_scratch_floats(x.n, (int)N, (int)K, dt);
    const Tensor scratch = scratch_floats(nf, x.t);
    call(arcn_dense_dw_sums(dz.p(), dz.ld, x.p(), x.ld, sums.p(), sums.n, dw.data_ptr(), out_ptr(db), dt, scratch.data_ptr<float>(), nf, x.n, (int)N, (int)K, stream), "dense_dw");
    return {dw, db};
}

struct LinearActResidual : torch::autograd::Function<LinearActResidual> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w, const OptTensor &b_, const OptTensor &res_, int64_t act, double beta) {
        const Tensor b = b_.value_or(Tensor()), res = res_.value_or(Tensor());
        ctx->saved_data["edges"] = edges({&x, &w, &b, &res});
        ctx->save_for_backward({x, w, b});
        ctx->saved_data["act"] = act;
        ctx->saved_data["beta"] = beta;
        return dense_forward(x, w, b, res, act, beta);
    }
    static tensor_list backward(AutogradContext *ctx, tensor_list g) {
        const bool graph = at::GradMode::is_enabled();
        at::NoGradGuard no_grad;
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], b = saved[2];
        const Tensor w = packed(saved[1]);
        const int64_t N = w.size(0), K = w.size(1), act = ctx->saved_data["act"].toInt();
        const Needs need(ctx);
        const bool want_dx = need(0), want_dw = need(1), want_db = need(2);
        tensor_list out(6);
        if (need(3)) out[3] = g[0];
        if (want_dx || want_dw || want_db) {
            const Rows r = rows_of("x", x, K, x);
            Rows dz = rows_of("dy", g[0], N, x);
            const int dt = type_code(x, "x");
            BiasSums sums;
            Launch go(x);
            if (act != ARCN_ACT_NONE) {
                const Rows dy = dz;
                const Tensor bc = packed(b);
                dz.t = fresh({r.n, N}, x);
                dz.ld = N;
                if (want_dx) out[0] = fresh(x.sizes(), x);
                sums = BiasSums(want_db, r.n, N, x);
                call(arcn_dense_dz_sums(r.p(), r.ld, ptr(w), ptr(bc), dy.p(), dy.ld, dz.t.data_ptr(), out_ptr(out[0]), sums.p(), sums.floats(), &sums.n, dt, (int)act,
                                        (float)ctx->saved_data["beta"].toDouble(), r.n, (int)K, (int)N, go.stream),
                     "dense_dz");
            } else if (want_dx) {
                out[0] = fresh(x.sizes(), x);
                call(arcn_dense_dx(dz.p(), dz.ld, ptr(w), nullptr, out[0].data_ptr(), dt, r.n, (int)N, (int)K, go.stream), "dense_dx");
            }
            if (want_dw || want_db) {
                auto [dw, db] = dense_dw(dz, N, r, K, want_db, sums, dt, go.stream);
                if (want_dw) out[1] = dw;
                out[2] = db;
            }
        }
        return first_order(std::move(out), graph, "linear_act_residual", {x, saved[1], b, g[0]});
    }
};

Tensor linear_act_residual(const Tensor &x, const Tensor &w, const OptTensor &b_, const OptTensor &res_, int64_t act, double beta) {
    const Tensor b = b_.value_or(Tensor()), res = res_.value_or(Tensor());
    refuse_untracked({&x, &w, &b, &res}, "linear_act_residual");
    return needs_graph({&x, &w, &b, &res}) ? LinearActResidual::apply(x, w, opt(b), opt(res), act, beta) : dense_forward(x, w, b, res, act, beta);
}

// ---- gated block ------------------------------------------------------------------------------------------------------------------------
Tensor gated_forward(const Tensor &x, const Tensor &wg, const Tensor &wu, const Tensor &bg, const Tensor &bu, int64_t act, double beta) {
    TORCH_CHECK(wg.dim() == 2, "arcnerf_amd: w_gate must be (H, K), got ", wg.sizes());
    const int64_t H = wg.size(0), K = wg.size(1);
    const Rows r = rows_of("x", x, K, x);
    const int dt = type_code(x, "x");
    const Tensor g = param("w_gate", wg, {H, K}, x), u = param("w_up", wu, {H, K}, x), gb = param("b_gate", bg, {H}, x), ub = param("b_up", bu, {H}, x);
    Tensor h = fresh(with_last(x, H), x);
    Launch go(x);
    call(arcn_gated_fwd(r.p(), r.ld, ptr(g), ptr(u), ptr(gb), ptr(ub), h.data_ptr(), dt, (int)act, (float)beta, r.n, (int)K, (int)H, go.stream), "gated_fwd");
    return h;
}

struct GatedFfn : torch::autograd::Function<GatedFfn> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &wg, const Tensor &wu, const Tensor &wd, const OptTensor &bg_, const OptTensor &bu_,
                          const OptTensor &bd_, const OptTensor &res_, int64_t act, double beta) {
        const Tensor bg = bg_.value_or(Tensor()), bu = bu_.value_or(Tensor()), bd = bd_.value_or(Tensor()), res = res_.value_or(Tensor());
        ctx->saved_data["edges"] = edges({&x, &wg, &wu, &wd, &bg, &bu, &bd, &res});
        const Tensor h = gated_forward(x, wg, wu, bg, bu, act, beta);
        Tensor y = dense_forward(h, wd, bd, res, ARCN_ACT_NONE, 1.0);
        ctx->save_for_backward({x, wg, wu, wd, bg, bu, h});
        ctx->saved_data["act"] = act;
        ctx->saved_data["beta"] = beta;
        return y;
    }
    static tensor_list backward(AutogradContext *ctx, tensor_list g) {
        const bool graph = at::GradMode::is_enabled();
        at::NoGradGuard no_grad;
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &h = saved[6];
        const Tensor wg = packed(saved[1]), wu = packed(saved[2]), wd = packed(saved[3]);
        const int64_t H = wg.size(0), K = wg.size(1), N = wd.size(0);
        const Needs need(ctx);
        const int dt = type_code(x, "x");
        tensor_list out(10);
        if (need(7)) out[7] = g[0];
        const Rows r = rows_of("x", x, K, x), dy = rows_of("dy", g[0], N, x);
        Launch go(x);
        if (need(3) || need(6)) {
            auto [dw, db] = dense_dw(dy, N, rows_of("h", h, H, x), H, need(6), BiasSums(), dt, go.stream);
            if (need(3)) out[3] = dw;
            out[6] = db;
        }
        const bool inner_w = need(1) || need(2), inner_b = need(4) || need(5);
        if (need(0) || inner_w || inner_b) {
            const Tensor bg = packed(saved[4]), bu = packed(saved[5]);
            Rows dgu;
            dgu.t = fresh({r.n, 2 * H}, x);
            dgu.n = r.n;
            dgu.ld = 2 * H;
            BiasSums sums(inner_b, r.n, 2 * H, x);
            call(arcn_gated_bwd_sums(r.p(), r.ld, ptr(wg), ptr(wu), ptr(bg), ptr(bu), dy.p(), dy.ld, ptr(wd), dgu.t.data_ptr(), sums.p(), sums.floats(), &sums.n, dt,
                                     (int)ctx->saved_data["act"].toInt(), (float)ctx->saved_data["beta"].toDouble(), r.n, (int)K, (int)H, (int)N, go.stream),
                 "gated_bwd");
            if (need(0)) {
                out[0] = fresh(x.sizes(), x);
                call(arcn_dense_dx(dgu.p(), dgu.ld, ptr(wg), ptr(wu), out[0].data_ptr(), dt, r.n, (int)(2 * H), (int)K, go.stream), "dense_dx");
            }
            if (inner_w || inner_b) {
                auto [dw, db] = dense_dw(dgu, 2 * H, r, K, inner_b, sums, dt, go.stream);
                if (need(1)) out[1] = dw.narrow(0, 0, H);
                if (need(2)) out[2] = dw.narrow(0, H, H);
                if (need(4)) out[4] = db.narrow(0, 0, H);
                if (need(5)) out[5] = db.narrow(0, H, H);
            }
        }
        return first_order(std::move(out), graph, "gated_ffn", {x, saved[1], saved[2], saved[3], saved[4], saved[5], g[0]});
    }
};

Tensor gated_ffn(const Tensor &x, const Tensor &wg, const Tensor &wu, const Tensor &wd, const OptTensor &bg_, const OptTensor &bu_, const OptTensor &bd_,
                 const OptTensor &res_, int64_t act, double beta) {
    const Tensor bg = bg_.value_or(Tensor()), bu = bu_.value_or(Tensor()), bd = bd_.value_or(Tensor()), res = res_.value_or(Tensor());
    refuse_untracked({&x, &wg, &wu, &wd, &bg, &bu, &bd, &res}, "gated_ffn");
    TORCH_CHECK(wd.dim() == 2 && wg.dim() == 2 && wd.size(1) == wg.size(0), "arcnerf_amd: w_down must be (N, H) for w_gate (H, K), got ", wd.sizes(), " and ", wg.sizes());
    if (needs_graph({&x, &wg, &wu, &wd, &bg, &bu, &bd, &res})) return GatedFfn::apply(x, wg, wu, wd, opt(bg), opt(bu), opt(bd), opt(res), act, beta);
    return dense_forward(gated_forward(x, wg, wu, bg, bu, act, beta), wd, bd, res, ARCN_ACT_NONE, 1.0);
}

}  // namespace

PYBIND11_MODULE(arcnerf_torch, m) {
    m.doc() = "autograd nodes of the residual feed-forward layers (arcnerf_amd.ops.autograd)";
    m.def("layer_norm", &layer_norm);
    m.def("linear_act_residual", &linear_act_residual);
    m.def("gated_ffn", &gated_ffn);
}

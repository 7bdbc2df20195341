// Autograd nodes of the row operators (fiery_amd/row_ops.py) over the C entry points of include/fiery_hip.h.
//
// The kernels of a training step on a few thousand rows take 10-50 us; autograd nodes written in Python cost twice that in the
// interpreter (a step of layer norm on 12 rows: 100 us, 44 of which torch itself takes for one multiplication and its gradient).
// These are the same nodes in C++.  Host code only: the library is reached through the addresses that Python took from it, so the
// product's and the simulator's builds serve alike, and a node launches on the stream that its forward pass was given, which is
// the one autograd makes current for the backward pass.
#include <ATen/TracerMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

#include <initializer_list>
#include <optional>
#include <stdexcept>
#include <utility>
#include <vector>

#include "fiery_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// the library's entry points, in the order in which native.Lib lists their addresses (ROW_ENTRIES)
struct Entries {
    decltype(&fiery_last_error) last_error;
    decltype(&fiery_layer_norm_fwd) norm_fwd;
    decltype(&fiery_layer_norm_bwd_workspace_floats) norm_bwd_workspace;
    decltype(&fiery_layer_norm_bwd) norm_bwd;
    decltype(&fiery_dropout) dropout;
    decltype(&fiery_dropout_add_layer_norm_fwd) join_fwd;
    decltype(&fiery_dropout_add_layer_norm_bwd) join_bwd;
    decltype(&fiery_dropout_add_layer_norm_fwd_unrounded) join_fwd_unrounded;
    decltype(&fiery_dropout_add_layer_norm_bwd_unrounded) join_bwd_unrounded;
};

// where a call goes
struct To {
    const Entries* lib;
    fiery_stream_t stream;
};
To to_of(int64_t entries, int64_t stream) { return {reinterpret_cast<const Entries*>(entries), reinterpret_cast<fiery_stream_t>(stream)}; }

void check(const To& to, int rc) {
    if (rc != FIERY_OK) throw std::runtime_error(std::string("libfiery_hip: error ") + std::to_string(rc) + ": " + to.lib->last_error());
}

// (the launch happens with the tensor's device current)
struct OnDevice {
    c10::OptionalDeviceGuard guard;
    explicit OnDevice(const Tensor& t) {
        if (t.is_cuda()) guard.reset_device(t.device());
    }
};

int type_of(at::ScalarType t) { return t == at::kFloat ? FIERY_TYPE_F32 : t == at::kBFloat16 ? FIERY_TYPE_BF16 : FIERY_TYPE_F16; }
int type_of(const Tensor& t) { return type_of(t.scalar_type()); }
// (null is an absent operand to the entry points: a tensor that has values and no memory, fake or zero, must not become one)
void* ptr(const Tensor& t) {
    if (!t.defined()) return nullptr;
    void* p = t.data_ptr();
    if (!p && t.numel()) throw std::runtime_error("row operators: a tensor without memory");
    return p;
}
float* floats(const Tensor& t, int64_t at = 0) { return t.defined() ? static_cast<float*>(ptr(t)) + at : nullptr; }
int64_t* numbers(const Tensor& t) { return static_cast<int64_t*>(ptr(t)); }
Tensor dense_like(const Tensor& t, at::ScalarType type) { return at::empty(t.sizes(), t.options().dtype(type).requires_grad(false)); }

struct Sizes {
    int64_t rows, c;
};
Sizes sizes_of(const Tensor& x) {
    const int64_t c = x.size(-1);
    return {x.numel() / c, c};
}

// the tensor itself unless its memory holds its values negated (views such as the imaginary part of a conjugate)
Tensor values_of(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }

// The tensor itself and the elements between its rows where they lie at one stride with their values side by side, else a copy.
std::pair<Tensor, int64_t> rows_of(const Tensor& given) {
    const Tensor t = values_of(given);
    const int64_t last = t.dim() - 1, c = t.size(last);
    if (t.is_contiguous()) return {t, c};
    if (t.stride(last) == 1 || c == 1) {
        int64_t ld = -1, expect = 0;
        bool even = true;
        for (int64_t i = last - 1; i >= 0 && even; --i) {
            if (t.size(i) == 1) continue;
            if (ld < 0)
                ld = t.stride(i);
            else
                even = t.stride(i) == expect;
            expect = t.stride(i) * t.size(i);
        }
        if (even) return {t, ld < 0 ? c : ld};
    }
    return {t.contiguous(), c};
}

struct Mask {
    int64_t threshold, share, one_column;
};

// A trace sees the allocation of a result and not the launch that fills it: the traced function would return what the memory held.
void untraced() {
    using c10::impl::TorchDispatchModeTLS;
    if (at::tracer::impl::is_dispatch_enabled() || c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch) ||
        TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value())
        throw std::runtime_error("row operators: tracing (torch.jit.trace, make_fx, torch.export) is not provided");
}

// Gradients of gradients: where a graph of the backward pass is made, its results hang on an error node below everything that they
// depend on, so that differentiating them is refused however it is reached.
template <typename Grads>
variable_list once(const variable_list& incoming, const variable_list& saved, Grads grads) {
    untraced();
    variable_list out;
    {
        const at::NoGradGuard no_graph;
        out = grads();
    }
    if (!at::GradMode::is_enabled()) return out;
    const size_t n = out.size();
    variable_list in;
    std::vector<size_t> place;
    for (size_t i = 0; i < n; ++i)
        if (out[i].defined()) {
            in.push_back(out[i].detach());
            place.push_back(i);
        }
    bool through = false;
    for (const auto* list : {&incoming, &saved})
        for (const Tensor& t : *list)
            if (t.defined() && t.requires_grad()) {
                in.push_back(t);
                through = true;
            }
    if (!through) return out;
    torch::autograd::DelayedError error("row operators: gradients of gradients are not provided", static_cast<int64_t>(in.size()));
    variable_list refused = error(std::move(in));
    for (size_t k = 0; k < place.size(); ++k) out[place[k]] = refused[k];
    return out;
}

// ---- layer norm ------------------------------------------------------------------------------------------------------------
Tensor norm_forward(const Tensor& xr, int64_t ld, const Tensor& weight, const Tensor& bias, double eps, const To& to, const Tensor& stats) {
    const Sizes s = sizes_of(xr);
    Tensor y = dense_like(xr, xr.scalar_type());
    if (s.rows) {
        const Tensor& params = weight.defined() ? weight : bias;
        check(to, to.lib->norm_fwd(ptr(xr), ld, type_of(xr), s.rows, static_cast<int>(s.c), ptr(weight), ptr(bias), params.defined() ? type_of(params) : 0,
                                   static_cast<float>(eps), ptr(y), s.c, floats(stats), floats(stats, s.rows), to.stream));
    }
    return y;
}

// The parameters' gradients where they are wanted, and the workspace of their sums: allocated per call, so that calls on other
// streams and captured graphs share none.
struct ParamGrads {
    Tensor dw, db, workspace;
    int64_t floats = 0;
    int type = 0;
    // edge: weight's place among the node's edges, bias's where there is no weight
    ParamGrads(const To& to, const Tensor& like, AutogradContext* ctx, size_t edge, const Tensor& weight, int64_t bias_type, const Sizes& s) {
        const bool want_w = weight.defined() && ctx->needs_input_grad(edge);
        const bool want_b = bias_type >= 0 && ctx->needs_input_grad(edge + (weight.defined() ? 1 : 0));
        const auto param = like.options().dtype(weight.defined() ? weight.scalar_type() : want_b ? static_cast<at::ScalarType>(bias_type) : at::kFloat).requires_grad(false);
        if (want_w) dw = at::empty({s.c}, param);
        if (want_b) db = at::empty({s.c}, param);
        if (!want_w && !want_b) return;
        type = type_of(want_w ? dw : db);
        if (s.rows) floats = to.lib->norm_bwd_workspace(s.rows, static_cast<int>(s.c));
        if (floats) workspace = at::empty({floats}, like.options().dtype(at::kFloat).requires_grad(false));
    }
    void zero() {
        if (dw.defined()) dw.zero_();
        if (db.defined()) db.zero_();
    }
};

const char* const kMeta = "m";

// (an absent tensor is a nullopt to autograd and takes no place among a node's edges; inside, it is an undefined tensor)
using Maybe = std::optional<Tensor>;
Tensor or_none(const Maybe& t) { return t.has_value() ? *t : Tensor(); }
Maybe resolved(const Maybe& t) { return t.has_value() ? Maybe(values_of(*t)) : t; }
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); }
constexpr int64_t kNone = -1;
int64_t type_or_none(const Tensor& t) { return t.defined() ? static_cast<int64_t>(t.scalar_type()) : kNone; }

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& weight_, const Maybe& bias_, double eps, int64_t entries, int64_t stream) {
        const Tensor weight = or_none(weight_), bias = or_none(bias_);
        const auto [xr, ld] = rows_of(x);
        const Tensor stats = at::empty({2 * sizes_of(x).rows}, x.options().dtype(at::kFloat).requires_grad(false));       // mean, then rstd
        ctx->save_for_backward({xr, weight, stats});
        ctx->saved_data[kMeta] = std::vector<int64_t>{ld, type_or_none(bias), entries, stream};
        return norm_forward(xr, ld, weight, bias, eps, to_of(entries, stream), stats);
    }
    static variable_list backward(AutogradContext* ctx, variable_list incoming) {
        const variable_list saved = ctx->get_saved_variables();
        return once(incoming, saved, [&]() -> variable_list {
            const Tensor &xr = saved[0], &weight = saved[1], &stats = saved[2];
            const auto meta = ctx->saved_data[kMeta].toIntVector();
            const To to = to_of(meta[2], meta[3]);
            const OnDevice on(xr);
            const Sizes s = sizes_of(xr);
            Tensor dx;
            if (ctx->needs_input_grad(0)) dx = dense_like(xr, xr.scalar_type());
            ParamGrads p(to, xr, ctx, 1, weight, meta[1], s);
            if (s.rows) {
                const auto [dy, dy_ld] = rows_of(incoming[0]);
                check(to, to.lib->norm_bwd(ptr(dy), dy_ld, ptr(xr), meta[0], type_of(xr), s.rows, static_cast<int>(s.c), ptr(weight),
                                           weight.defined() ? type_of(weight) : p.type, floats(stats), floats(stats, s.rows), ptr(dx), s.c, ptr(p.dw), ptr(p.db),
                                           floats(p.workspace), p.floats, to.stream));
            } else {
                p.zero();
            }
            return {dx, p.dw, p.db, Tensor(), Tensor(), Tensor()};
        });
    }
};

// ---- dropout -----------------------------------------------------------------------------------------------------------------
Tensor drop(const Tensor& x, const Tensor& residual, at::ScalarType type, const Mask& m, const int64_t* rng, int64_t call, int64_t* used, const To& to) {
    const Sizes s = sizes_of(x);
    Tensor y = dense_like(x, type);
    if (s.rows) {
        const auto [xr, ld] = rows_of(x);
        const auto [rr, r_ld] = residual.defined() ? rows_of(residual) : std::pair<Tensor, int64_t>();
        check(to, to.lib->dropout(ptr(xr), ld, type_of(xr), ptr(rr), r_ld, s.rows, static_cast<int>(s.c), static_cast<int>(m.threshold),
                                  m.threshold ? rng : nullptr, call, m.share, static_cast<int>(m.one_column), used, ptr(y), s.c, type_of(type),
                                  to.stream));
    }
    return y;
}

Tensor used_numbers(const Tensor& x, const Mask& m) {
    return m.threshold ? at::empty({2}, x.options().dtype(at::kLong).requires_grad(false)) : Tensor();
}

struct Dropout : torch::autograd::Function<Dropout> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& residual_, const Maybe& rng, int64_t threshold, int64_t share,
                          int64_t one_column, int64_t call, int64_t entries, int64_t stream) {
        const Tensor residual = or_none(residual_);
        const Mask m{threshold, share, one_column};
        const Tensor used = used_numbers(x, m);
        ctx->save_for_backward({used});
        ctx->saved_data[kMeta] = std::vector<int64_t>{static_cast<int64_t>(x.scalar_type()), threshold, share, one_column, entries, stream, residual.defined()};
        return drop(x, residual, residual.defined() ? residual.scalar_type() : x.scalar_type(), m, numbers(or_none(rng)), call, numbers(used), to_of(entries, stream));
    }
    static variable_list backward(AutogradContext* ctx, variable_list incoming) {
        const variable_list saved = ctx->get_saved_variables();
        return once(incoming, saved, [&]() -> variable_list {
            const Tensor& used = saved[0];
            const auto meta = ctx->saved_data[kMeta].toIntVector();
            const OnDevice on(incoming[0]);
            Tensor dx, dr;
            if (ctx->needs_input_grad(0))
                dx = drop(incoming[0], Tensor(), static_cast<at::ScalarType>(meta[0]), {meta[1], meta[2], meta[3]}, numbers(used), 0, nullptr, to_of(meta[4], meta[5]));
            if (meta[6] && ctx->needs_input_grad(1)) dr = incoming[0];
            return {dx, dr, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
        });
    }
};

// ---- residual + dropout + layer norm --------------------------------------------------------------------------------------------
// stats: mean and rstd of the rows, then the two numbers that the masks were drawn with; undefined where no backward pass follows
int64_t* used_behind(const Tensor& stats, int64_t rows) { return reinterpret_cast<int64_t*>(floats(stats, 2 * rows)); }

variable_list join_forward(const Tensor& x, const Tensor& residual, const Tensor& weight, const Tensor& bias, const Tensor& rng, const Mask& m, int64_t call,
                           double eps, bool of_sum, const To& to, const Tensor& stats) {
    const Sizes s = sizes_of(x);
    Tensor y = dense_like(x, x.scalar_type()), h = dense_like(x, residual.scalar_type());
    if (s.rows) {
        const auto [xr, ld] = rows_of(x);
        const auto [rr, r_ld] = rows_of(residual);
        const Tensor& params = weight.defined() ? weight : bias;
        const auto call_fwd = of_sum ? to.lib->join_fwd_unrounded : to.lib->join_fwd;
        check(to, call_fwd(ptr(xr), ld, type_of(xr), ptr(rr), r_ld, type_of(rr), s.rows, static_cast<int>(s.c), ptr(weight), ptr(bias),
                           params.defined() ? type_of(params) : 0, static_cast<float>(eps), static_cast<int>(m.threshold),
                           m.threshold ? numbers(rng) : nullptr, call, m.share, static_cast<int>(m.one_column), used_behind(stats, s.rows), ptr(y), s.c, ptr(h), s.c,
                           floats(stats), floats(stats, s.rows), to.stream));
    }
    return {y, h};
}

struct DropoutAddLayerNorm : torch::autograd::Function<DropoutAddLayerNorm> {
    // inputs: the backward pass reads x and the residual, not h (an h of 32 bits is not rounded: then it reads that)
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& residual, const Maybe& weight_, const Maybe& bias_, const Maybe& rng,
                                 int64_t threshold, int64_t share, int64_t one_column, int64_t call, double eps, bool inputs, int64_t entries, int64_t stream) {
        const Tensor weight = or_none(weight_), bias = or_none(bias_);
        const Mask m{threshold, share, one_column};
        const Tensor stats = at::empty({2 * sizes_of(x).rows + 4}, x.options().dtype(at::kFloat).requires_grad(false));
        const bool of_sum = inputs && residual.scalar_type() != at::kFloat;
        const auto [xr, x_ld] = of_sum ? rows_of(x) : std::pair<Tensor, int64_t>(x, 0);
        const auto [rr, r_ld] = of_sum ? rows_of(residual) : std::pair<Tensor, int64_t>(residual, 0);
        variable_list out = join_forward(xr, rr, weight, bias, or_none(rng), m, call, eps, of_sum, to_of(entries, stream), stats);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({of_sum ? rr : out[1], weight, stats, of_sum ? xr : Tensor()});
        ctx->saved_data[kMeta] = std::vector<int64_t>{static_cast<int64_t>(x.scalar_type()), type_or_none(bias), threshold, share, one_column, entries, stream,
                                                      of_sum ? r_ld : sizes_of(x).c, x_ld};
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list incoming) {
        const variable_list saved = ctx->get_saved_variables();
        return once(incoming, saved, [&]() -> variable_list {
            const Tensor &h = saved[0], &weight = saved[1], &stats = saved[2], &x = saved[3];              // (x: then h is the residual)
            const auto meta = ctx->saved_data[kMeta].toIntVector();
            const auto x_type = static_cast<at::ScalarType>(meta[0]);
            const Mask m{meta[2], meta[3], meta[4]};
            const To to = to_of(meta[5], meta[6]);
            const OnDevice on(h);
            Sizes s = sizes_of(h);
            int64_t* const used = used_behind(stats, s.rows);
            const Tensor &dy = incoming[0], &dh = incoming[1];
            const bool want_x = ctx->needs_input_grad(0), want_r = ctx->needs_input_grad(1);
            Tensor dx, dr;
            if (!dy.defined()) {                                        // only h went on: there is no norm to differentiate
                const int64_t rows = std::exchange(s.rows, 0);
                if (want_x && dh.defined()) {
                    dx = dense_like(h, x_type);
                    const auto [hg, dh_ld] = rows_of(dh);
                    if (rows) check(to, to.lib->join_bwd(nullptr, 0, ptr(hg), dh_ld, nullptr, 0, type_of(x_type), type_of(h), rows, static_cast<int>(s.c), nullptr, 0,
                                                         nullptr, nullptr, static_cast<int>(m.threshold), used, m.share, static_cast<int>(m.one_column), ptr(dx),
                                                         s.c, nullptr, 0, nullptr, nullptr, nullptr, 0, to.stream));
                }
                if (want_r) dr = dh;
            } else {
                if (want_x) dx = dense_like(h, x_type);
                if (want_r) dr = dense_like(h, h.scalar_type());
            }
            ParamGrads p(to, h, ctx, 2, weight, meta[1], s);
            if (s.rows) {
                const auto [gr, dy_ld] = rows_of(dy);
                const auto [hg, dh_ld] = dh.defined() ? rows_of(dh) : std::pair<Tensor, int64_t>();
                const int param_type = weight.defined() ? type_of(weight) : p.type;
                if (x.defined())
                    check(to, to.lib->join_bwd_unrounded(ptr(gr), dy_ld, ptr(hg), dh_ld, ptr(x), meta[8], ptr(h), meta[7], type_of(h), s.rows, static_cast<int>(s.c),
                                                         ptr(weight), param_type, floats(stats), floats(stats, s.rows), static_cast<int>(m.threshold), used,
                                                         m.share, static_cast<int>(m.one_column), ptr(dx), s.c, ptr(dr), s.c, ptr(p.dw), ptr(p.db),
                                                         floats(p.workspace), p.floats, to.stream));
                else
                    check(to, to.lib->join_bwd(ptr(gr), dy_ld, ptr(hg), dh_ld, ptr(h), meta[7], type_of(x_type), type_of(h), s.rows, static_cast<int>(s.c), ptr(weight),
                                               param_type, floats(stats), floats(stats, s.rows), static_cast<int>(m.threshold), used, m.share,
                                               static_cast<int>(m.one_column), ptr(dx), s.c, ptr(dr), s.c, ptr(p.dw), ptr(p.db), floats(p.workspace), p.floats,
                                               to.stream));
            } else {
                p.zero();
            }
            return {dx, dr, p.dw, p.db, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
        });
    }
};

// What the operators do not provide is an error.  (A dual tensor without a gradient would go past the nodes and lose its tangent.)
void provided(std::initializer_list<const Tensor*> operands) {
    untraced();
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const Tensor* t : operands)
        if (t->defined() && t->_fw_grad(0).defined()) throw std::runtime_error("row operators: forward-mode derivatives are not provided");
}

// ---- what Python calls, with arguments that it has checked ------------------------------------------------------------------------
Tensor dense(const Maybe& t) { return t.has_value() ? values_of(*t).contiguous() : Tensor(); }
bool wants(const Tensor& t) { return t.defined() && t.requires_grad(); }

Tensor layer_norm(const Tensor& x, const Maybe& weight, const Maybe& bias, double eps, int64_t entries, int64_t stream) {
    const OnDevice on(x);
    const Tensor w = dense(weight), b = dense(bias);
    provided({&x, &w, &b});
    if (at::GradMode::is_enabled() && (wants(x) || wants(w) || wants(b))) return LayerNorm::apply(x, maybe(w), maybe(b), eps, entries, stream);
    const auto [xr, ld] = rows_of(x);
    return norm_forward(xr, ld, w, b, eps, to_of(entries, stream), Tensor());
}

Tensor dropout(const Tensor& x, const Maybe& residual, const Maybe& rng_, const std::tuple<int64_t, int64_t, int64_t>& mask, int64_t call, int64_t entries,
               int64_t stream) {
    const OnDevice on(x);
    const Tensor r = or_none(residual);
    const Maybe rng = resolved(rng_);
    provided({&x, &r});
    const auto [threshold, share, one_column] = mask;
    if (at::GradMode::is_enabled() && (wants(x) || wants(r))) return Dropout::apply(x, residual, rng, threshold, share, one_column, call, entries, stream);
    return drop(x, r, r.defined() ? r.scalar_type() : x.scalar_type(), {threshold, share, one_column}, numbers(or_none(rng)), call, nullptr, to_of(entries, stream));
}

std::pair<Tensor, Tensor> dropout_add_layer_norm(const Tensor& x, const Tensor& residual, const Maybe& weight, const Maybe& bias, const Maybe& rng_,
                                                 const std::tuple<int64_t, int64_t, int64_t>& mask, int64_t call, double eps, bool inputs, int64_t entries,
                                                 int64_t stream) {
    const OnDevice on(x);
    const Tensor w = dense(weight), b = dense(bias);
    const Maybe rng = resolved(rng_);
    provided({&x, &residual, &w, &b});
    const auto [threshold, share, one_column] = mask;
    variable_list out;
    if (at::GradMode::is_enabled() && (wants(x) || wants(residual) || wants(w) || wants(b)))
        out = DropoutAddLayerNorm::apply(x, residual, maybe(w), maybe(b), rng, threshold, share, one_column, call, eps, inputs, entries, stream);
    else
        out = join_forward(x, residual, w, b, or_none(rng), {threshold, share, one_column}, call, eps, false, to_of(entries, stream), Tensor());
    return {out[0], out[1]};
}

}  // namespace

PYBIND11_MODULE(_row_autograd, m) {
    m.attr("abi_version") = FIERY_ABI_VERSION;
    m.def("rows_of", &rows_of);
    m.def("layer_norm", &layer_norm);
    m.def("dropout", &dropout);
    m.def("dropout_add_layer_norm", &dropout_add_layer_norm);
}

// Tensor front end of the public operators (lsdm_amd/ops.py): argument checks, allocation and the autograd nodes over the C entry points of
// include/lsdm_hip.h.  It is C++ because the smallest calls cost what their host code costs: the same nodes written in Python took 70 - 115 us for
// a forward and backward pass whose kernels take 20.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>

#include "../../include/lsdm_hip.h"

#include <unordered_set>

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct LsdmFailure : std::runtime_error { using std::runtime_error::runtime_error; };      // becomes lsdm_amd._lib.LsdmError

constexpr int64_t kMaxSize = (int64_t)1 << 30, kMaxOut = (int64_t)1 << 25;
constexpr int64_t kNormMaxWidth = 16384;

template <class... A>
std::string text(const A&... a) {
    std::ostringstream s;
    (void)std::initializer_list<int>{(s << a, 0)...};
    return s.str();
}
template <class... A>
[[noreturn]] void value_error(const A&... a) { throw pybind11::value_error(text(a...)); }

void ok(int64_t rc, const char* what) {
    if (rc < 0) throw LsdmFailure(text(what, " failed (", rc, "): ", lsdm_last_error(nullptr)));
}

int dtype_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return LSDM_F32;
        case at::kBFloat16: return LSDM_BF16;
        case at::kHalf: return LSDM_F16;
        default: return -1;
    }
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// A tracer (torch.jit.trace, make_fx, fake tensors) records tensors' operations; what the kernels write through pointers is none, and the recorded graph would
// return memory that nothing wrote.
void check_traced(const char* who) {
    using c10::impl::TorchDispatchModeKey;
    bool traced = torch::jit::tracer::isTracing();
    if (c10::impl::TorchDispatchModeTLS::any_modes_set())
        for (const auto k : {TorchDispatchModeKey::FAKE, TorchDispatchModeKey::PROXY, TorchDispatchModeKey::FUNCTIONAL})
            traced = traced || c10::impl::TorchDispatchModeTLS::get_mode(k).has_value();
    if (traced) throw LsdmFailure(text(who, " cannot be traced: its kernels run outside of torch's operations (capture the call into a HIP graph instead)"));
}
// a dual tensor's tangent would be dropped, which reads as a derivative of zero
void check_tangents(const char* who, std::initializer_list<const Tensor*> inputs) {
    for (const Tensor* t : inputs)
        if (t->defined() && t->_fw_grad(0).defined()) throw LsdmFailure(text(who, " has no forward-mode derivative; an input carries a tangent"));
}
void check_operand(const char* who, const Tensor& x) {
    if (!x.is_cuda()) throw LsdmFailure(text(who, " runs in liblsdm_hip.so on HIP device tensors; got ", x.device()));
    if (x.layout() != at::kStrided || dtype_of(x.scalar_type()) < 0) value_error(who, ": a dense tensor of dtype float32, bfloat16 or float16 is needed, got ", x.scalar_type());
}
void check_device(const char* who, const char* name, const Tensor& t, const Tensor& x) {
    if (!t.defined()) return;
    if (t.device() != x.device()) throw LsdmFailure(text(who, ": ", name, " is on ", t.device(), ", x on ", x.device()));
    if (t.layout() != at::kStrided) value_error(who, ": ", name, " must be a dense tensor");
}

// rows of `width` elements with unit stride and one row stride; copies only what no row stride can describe
struct Rows { Tensor t; int64_t ld; };
Rows rows_of(const Tensor& t, int64_t width) {
    Tensor r = (t.dim() == 2 ? t : t.reshape({t.numel() / width, width})).resolve_neg();       // (a lazily negated view: z.conj().imag)
    if (r.stride(1) == 1 && r.stride(0) >= width) return {r, r.stride(0)};
    return {r.contiguous(), width};
}
bool unaligned(const Rows& r, int64_t width) {
    const int64_t es = r.t.element_size();
    return ((reinterpret_cast<int64_t>(r.t.data_ptr()) | r.ld * es | width * es) & 15) != 0;
}
Tensor scratch(int64_t bytes, const Tensor& like) { return bytes > 0 ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor(); }
Tensor maybe_contiguous(const Tensor& t) { return t.defined() ? t.resolve_neg().contiguous() : t; }

// A graph node that sits on the default stream -- a leaf's gradient node that an eager graph keeps alive, or a part of such a graph -- cannot take part in a
// capture on another stream: autograd would have to join the default stream to it, and the failure surfaces where the process cannot recover.  Everything
// that the call's backward pass can reach is looked at (a leaf may stand behind casts and views), and the call refused before anything is recorded.
void check_capture(const char* who, const Tensor& x, std::initializer_list<const Tensor*> inputs) {
    const auto current = c10::hip::getCurrentHIPStream(x.device().index());
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(current.stream(), &status) != hipSuccess) {       // (the default stream while another one is captured)
        (void)hipGetLastError();
        return;
    }
    if (status == hipStreamCaptureStatusNone) return;
    const auto def = c10::hip::getDefaultHIPStream(x.device().index());
    std::vector<std::shared_ptr<torch::autograd::Node>> open;
    std::unordered_set<torch::autograd::Node*> seen;
    auto visit = [&](const std::shared_ptr<torch::autograd::Node>& n) {
        if (n && seen.insert(n.get()).second) open.push_back(n);
    };
    for (const Tensor* t : inputs)
        if (t->defined() && t->requires_grad()) visit(t->is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(*t) : t->grad_fn());
    while (!open.empty()) {
        const auto node = std::move(open.back());
        open.pop_back();
        const auto s = node->stream();
        // (by number: the node's stream carries the device type that torch shows, this one the runtime's)
        if (s && s->device_index() == x.device().index() && s->id() != current.id() && s->id() == def.id())
            throw LsdmFailure(text(who, ": a leaf of this captured call, or a part of the graph behind it, is held by a live autograd graph that was built on the default "
                                        "stream; release that graph (or build it on a side stream) before the capture"));
        for (const auto& e : node->next_edges()) visit(e.function);
    }
}

variable_list differentiable_once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    for (Tensor& g : grads)
        if (g.defined()) {
            variable_list one{g.detach().set_requires_grad(true)};
            g = torch::autograd::DelayedError("the gradients of lsdm_amd.ops are differentiable once", 1).apply(std::move(one))[0];
        }
    return grads;
}

// ------------------------------------------------------------------------------------------------ 8-bit checkpoints
std::pair<Tensor, Tensor> pack_rows(const Rows& x, int64_t width) {
    const int64_t n = x.t.size(0);
    Tensor codes = at::empty({n, width}, x.t.options().dtype(at::kChar)), exps = at::empty({n, (width + 31) / 32}, x.t.options().dtype(at::kByte));
    if (codes.numel())
        ok(lsdm_pack8(x.t.device().index(), dtype_of(x.t.scalar_type()), n, width, x.t.data_ptr(), x.ld, codes.data_ptr(), exps.data_ptr(), stream_of(x.t)), "lsdm_pack8");
    return {codes, exps};
}

std::pair<Tensor, Tensor> pack8(const Tensor& x_) {
    check_traced("checkpoint8");
    check_operand("checkpoint8", x_);
    const Tensor x = x_.detach();
    if (x.dim() < 1) value_error("checkpoint8: a tensor of at least one axis is needed");
    const int64_t width = x.size(-1);
    if (width > kMaxSize) value_error("checkpoint8: the last axis may hold at most 2^30 values");
    if (x.numel() == 0)
        return {at::empty({0, width}, x.options().dtype(at::kChar)), at::empty({0, (width + 31) / 32}, x.options().dtype(at::kByte))};
    return pack_rows(rows_of(x, width), width);
}

Tensor unpack8(const Tensor& codes, const Tensor& exps, const std::vector<int64_t>& shape, at::ScalarType dtype) {
    check_traced("Checkpoint8.restore");
    if (dtype_of(dtype) < 0) value_error("Checkpoint8.restore: dtype must be float32, bfloat16 or float16, got ", dtype);
    if (!codes.is_cuda() || exps.device() != codes.device()) throw LsdmFailure("Checkpoint8.restore: codes and exps must be on one HIP device");
    const bool dense = codes.dim() == 2 && codes.scalar_type() == at::kChar && codes.is_contiguous() && exps.dim() == 2 && exps.scalar_type() == at::kByte &&
                       exps.is_contiguous() && exps.size(0) == codes.size(0) && exps.size(1) == (codes.size(1) + 31) / 32;
    if (!dense) value_error("Checkpoint8.restore: codes must be dense int8 (rows, width), exps dense uint8 (rows, ceil(width / 32))");
    Tensor out = at::empty(shape, codes.options().dtype(dtype));
    if (out.numel() != codes.numel()) value_error("Checkpoint8.restore: the shape does not hold the codes");
    if (out.numel())
        ok(lsdm_unpack8(out.device().index(), dtype_of(dtype), codes.size(0), codes.size(1), codes.data_ptr(), exps.data_ptr(), out.data_ptr(), stream_of(out)), "lsdm_unpack8");
    return out;
}

// ------------------------------------------------------------------------------------------------ linear
struct LinearForward { Tensor y, deriv; };
LinearForward linear_forward(const Tensor& x_, const Tensor& w_, const Tensor& bias_, const Tensor& residual, int act, bool want_deriv, bool deriv8) {
    const int64_t N = w_.size(0), K = w_.size(1);
    const Rows x = rows_of(x_, K), w = rows_of(w_, K);
    const Tensor bias = maybe_contiguous(bias_);
    const int64_t M = x.t.size(0);
    std::vector<int64_t> shape(x_.sizes().begin(), x_.sizes().end());
    shape.back() = N;
    LinearForward f;
    f.y = at::empty(shape, x.t.options());
    if (want_deriv) f.deriv = at::empty({M, N}, deriv8 ? x.t.options().dtype(at::kByte) : x.t.options());      // (its bits: lsdm_hip.h)
    if (M == 0 || N == 0) return f;
    const int dt = dtype_of(x.t.scalar_type());
    const int flags = (bias.defined() && bias.scalar_type() == at::kFloat ? LSDM_OP_PARAM_F32 : 0) | (deriv8 ? LSDM_OP_DERIV8 : 0);
    Rows r{Tensor(), 0};
    if (residual.defined()) r = rows_of(residual, N);
    const int64_t bytes = lsdm_linear_workspace(dt, flags | (unaligned(x, K) ? LSDM_OP_X_UNALIGNED : 0) | (unaligned(w, K) ? LSDM_OP_W_UNALIGNED : 0), M, N, K);
    ok(bytes, "lsdm_linear_workspace");
    const Tensor ws = scratch(bytes, x.t);
    ok(lsdm_linear(x.t.device().index(), dt, act, flags, M, N, K, x.t.data_ptr(), x.ld, w.t.data_ptr(), w.ld, ptr(bias), ptr(r.t), r.ld, f.y.data_ptr(), ptr(f.deriv),
                   ptr(ws), bytes, stream_of(x.t)), "lsdm_linear");
    return f;
}

struct LinearNode : torch::autograd::Function<LinearNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const std::optional<Tensor>& bias_, const std::optional<Tensor>& residual_, int64_t act,
                          bool checkpoint, bool need_x, bool need_w, bool need_b) {
        const Tensor bias = bias_.value_or(Tensor()), residual = residual_.value_or(Tensor());
        const bool inner = need_x || need_w || need_b, deriv8 = checkpoint && x.scalar_type() != at::kFloat;
        LinearForward f = linear_forward(x, w, bias, residual, (int)act, inner && act != LSDM_ACT_NONE, deriv8);
        Tensor codes, exps;
        if (need_w && checkpoint) std::tie(codes, exps) = pack_rows(rows_of(x, w.size(1)), w.size(1));
        ctx->save_for_backward({need_w && !checkpoint ? x : Tensor(), codes, exps, need_x ? w : Tensor(), f.deriv});
        ctx->saved_data["x"] = x.sizes().vec();
        ctx->saved_data["w"] = w.sizes().vec();
        ctx->saved_data["b"] = (int64_t)(bias.defined() ? bias.scalar_type() : x.scalar_type());
        ctx->saved_data["deriv8"] = deriv8;
        ctx->saved_data["has_bias"] = bias.defined();
        ctx->saved_data["has_residual"] = residual.defined();
        return f.y;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        check_traced("the backward pass of linear");
        const Tensor& dy_ = grads[0];
        variable_list out(9);
        if (!dy_.defined()) return out;
        // (edges are numbered over the tensors that were given)
        const bool has_bias = ctx->saved_data["has_bias"].toBool(), has_residual = ctx->saved_data["has_residual"].toBool();
        const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1), need_b = has_bias && ctx->needs_input_grad(2),
                   need_r = has_residual && ctx->needs_input_grad(has_bias ? 3 : 2);
        if (need_x || need_w || need_b) {
            const variable_list saved = ctx->get_saved_variables();
            const Tensor &x = saved[0], &codes = saved[1], &exps = saved[2], &w = saved[3], &deriv = saved[4];
            const std::vector<int64_t> xshape = ctx->saved_data["x"].toIntVector(), wshape = ctx->saved_data["w"].toIntVector();
            const at::ScalarType btype = (at::ScalarType)ctx->saved_data["b"].toInt();
            const bool deriv8 = ctx->saved_data["deriv8"].toBool();
            const int64_t N = wshape[0], K = wshape[1];
            int64_t M = 1;
            for (size_t i = 0; i + 1 < xshape.size(); ++i) M *= xshape[i];
            const bool some = M > 0 && N > 0;
            auto fresh = [&](const std::vector<int64_t>& shape, at::ScalarType t) {
                return some ? at::empty(shape, dy_.options().dtype(t)) : at::zeros(shape, dy_.options().dtype(t));
            };
            Tensor dx, dw, db;
            if (need_x) dx = fresh(xshape, dy_.scalar_type());
            if (need_w) dw = fresh(wshape, dy_.scalar_type());
            if (need_b) db = fresh({N}, btype);
            if (some) {
                const Rows dy = rows_of(dy_, N);
                Rows xr{Tensor(), 0}, wr{Tensor(), 0};
                const int flags = (btype == at::kFloat ? LSDM_OP_PARAM_F32 : 0) | (deriv8 ? LSDM_OP_DERIV8 : 0);
                int plan = flags | LSDM_OP_BACKWARD | (need_x ? LSDM_OP_DX : 0) | (need_w ? LSDM_OP_DW : 0) | (need_b ? LSDM_OP_DB : 0) |
                           (deriv.defined() ? LSDM_OP_DERIV : 0) | (codes.defined() ? LSDM_OP_CODES : 0) | (unaligned(dy, N) ? LSDM_OP_DY_UNALIGNED : 0);
                if (need_w && x.defined()) {
                    xr = rows_of(x, K);
                    if (unaligned(xr, K)) plan |= LSDM_OP_X_UNALIGNED;
                }
                if (need_x) {
                    wr = rows_of(w, K);
                    if (unaligned(wr, K)) plan |= LSDM_OP_W_UNALIGNED;
                }
                const int dt = dtype_of(dy.t.scalar_type());
                const int64_t bytes = lsdm_linear_workspace(dt, plan, M, N, K);
                ok(bytes, "lsdm_linear_workspace");
                const Tensor ws = scratch(bytes, dy.t);
                ok(lsdm_linear_backward(dy.t.device().index(), dt, flags, M, N, K, dy.t.data_ptr(), dy.ld, ptr(deriv), ptr(xr.t), xr.ld, ptr(codes), ptr(exps), ptr(wr.t),
                                        wr.ld, ptr(dx), ptr(dw), ptr(db), ptr(ws), bytes, stream_of(dy.t)), "lsdm_linear_backward");
            }
            out[0] = dx; out[1] = dw; out[2] = db;
        }
        if (need_r) out[3] = dy_;
        return differentiable_once(std::move(out));
    }
};

Tensor linear(const Tensor& x, const Tensor& w, const std::optional<Tensor>& bias_, int64_t act, const std::optional<Tensor>& residual_, bool checkpoint) {
    const Tensor bias = bias_.value_or(Tensor()), residual = residual_.value_or(Tensor());
    check_traced("linear");
    check_tangents("linear", {&x, &w, &bias, &residual});
    check_operand("linear", x);
    check_device("linear", "weight", w, x);
    check_device("linear", "bias", bias, x);
    check_device("linear", "residual", residual, x);
    if (w.dim() != 2 || x.dim() < 1 || x.size(-1) != w.size(1)) value_error("linear: expected x (..., K) and weight (N, K), got ", x.sizes(), " and ", w.sizes());
    const int64_t N = w.size(0), K = w.size(1);
    if (K < 1) value_error("linear: weight has no columns");
    if (x.numel() / K > kMaxSize || N > kMaxOut || K > kMaxSize) value_error("linear: x holds at most 2^30 rows and columns, weight 2^25 rows");
    if (w.scalar_type() != x.scalar_type() || (residual.defined() && residual.scalar_type() != x.scalar_type()))
        value_error("linear: weight and residual must have x's dtype ", x.scalar_type());
    if (bias.defined() && (bias.dim() != 1 || bias.size(0) != N || (bias.scalar_type() != x.scalar_type() && bias.scalar_type() != at::kFloat)))
        value_error("linear: bias must be [", N, "] of dtype ", x.scalar_type(), " or float32, got ", bias.sizes(), " ", bias.scalar_type());
    if (residual.defined()) {
        bool same = residual.dim() == x.dim() && residual.size(-1) == N;
        for (int64_t i = 0; same && i + 1 < x.dim(); ++i) same = residual.size(i) == x.size(i);
        if (!same) value_error("linear: residual must have the result's shape (x's leading axes, ", N, "), got ", residual.sizes());
    }
    if (at::GradMode::is_enabled()) {
        const bool gx = x.requires_grad(), gw = w.requires_grad(), gb = bias.defined() && bias.requires_grad(), gr = residual.defined() && residual.requires_grad();
        if (gx || gw || gb || gr) {
            check_capture("linear", x, {&x, &w, &bias, &residual});
            return LinearNode::apply(x, w, bias_, residual_, act, checkpoint, gx, gw, gb);
        }
    }
    return linear_forward(x, w, bias, residual, (int)act, false, false).y;
}

// ------------------------------------------------------------------------------------------------ layer norm
struct NormForward { Tensor y, mean, rstd, codes, exps; };
NormForward norm_forward(const Tensor& x_, const Tensor& w_, const Tensor& b_, double eps, bool keep, bool checkpoint) {
    const int64_t D = x_.size(-1);
    const Rows x = rows_of(x_, D);
    const Tensor w = maybe_contiguous(w_), b = maybe_contiguous(b_);
    const int64_t n = x.t.size(0);
    NormForward f;
    f.y = at::empty(x_.sizes(), x.t.options());
    if (keep) {
        f.rstd = at::empty({n}, x.t.options().dtype(at::kFloat));
        if (checkpoint) {
            f.codes = at::empty({n, D}, x.t.options().dtype(at::kChar));
            f.exps = at::empty({n, (D + 31) / 32}, x.t.options().dtype(at::kByte));
        } else {
            f.mean = at::empty({n}, x.t.options().dtype(at::kFloat));
        }
    }
    const bool f32 = (w.defined() && w.scalar_type() == at::kFloat) || (b.defined() && b.scalar_type() == at::kFloat);
    if (n)
        ok(lsdm_layer_norm(x.t.device().index(), dtype_of(x.t.scalar_type()), f32 ? LSDM_OP_PARAM_F32 : 0, n, D, x.t.data_ptr(), x.ld, ptr(w), ptr(b), (float)eps, f.y.data_ptr(),
                           (float*)ptr(f.mean), (float*)ptr(f.rstd), ptr(f.codes), ptr(f.exps), stream_of(x.t)), "lsdm_layer_norm");
    return f;
}

struct NormNode : torch::autograd::Function<NormNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& w_, const std::optional<Tensor>& b_, double eps, bool checkpoint) {
        const Tensor w = w_.value_or(Tensor()), b = b_.value_or(Tensor());
        NormForward f = norm_forward(x, w, b, eps, true, checkpoint);
        ctx->save_for_backward({checkpoint ? Tensor() : x, f.mean, f.rstd, f.codes, f.exps, w});
        ctx->saved_data["has_w"] = w.defined();
        ctx->saved_data["has_b"] = b.defined();
        ctx->saved_data["p"] = (int64_t)(w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : x.scalar_type());
        return f.y;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        check_traced("the backward pass of layer_norm");
        const Tensor& dy_ = grads[0];
        variable_list out(5);
        if (!dy_.defined()) return out;
        const bool has_w = ctx->saved_data["has_w"].toBool(), has_b = ctx->saved_data["has_b"].toBool();
        const bool need_x = ctx->needs_input_grad(0), need_w = has_w && ctx->needs_input_grad(1), need_b = has_b && ctx->needs_input_grad(has_w ? 2 : 1);
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &mean = saved[1], &rstd = saved[2], &codes = saved[3], &exps = saved[4];
        const Tensor w = maybe_contiguous(saved[5]);
        const at::ScalarType ptype = (at::ScalarType)ctx->saved_data["p"].toInt();
        const int64_t D = dy_.size(-1), n = rstd.size(0);
        auto fresh = [&](at::IntArrayRef shape, at::ScalarType t) { return n ? at::empty(shape, dy_.options().dtype(t)) : at::zeros(shape, dy_.options().dtype(t)); };
        if (need_x) out[0] = fresh(dy_.sizes(), dy_.scalar_type());
        if (need_w) out[1] = fresh({D}, ptype);
        if (need_b) out[2] = fresh({D}, ptype);
        if (n) {
            const Rows dy = rows_of(dy_, D);
            Rows xr{Tensor(), 0};
            if (x.defined()) xr = rows_of(x, D);
            int64_t bytes = 0;
            if (need_w || need_b) { bytes = lsdm_layer_norm_workspace(n, D); ok(bytes, "lsdm_layer_norm_workspace"); }
            const Tensor ws = scratch(bytes, dy.t);
            ok(lsdm_layer_norm_backward(dy.t.device().index(), dtype_of(dy.t.scalar_type()), ptype == at::kFloat ? LSDM_OP_PARAM_F32 : 0, n, D, dy.t.data_ptr(), dy.ld, ptr(xr.t),
                                        xr.ld, ptr(codes), ptr(exps), ptr(w), (const float*)ptr(mean), (const float*)ptr(rstd), ptr(out[0]), ptr(out[1]), ptr(out[2]), ptr(ws),
                                        bytes, stream_of(dy.t)), "lsdm_layer_norm_backward");
        }
        return differentiable_once(std::move(out));
    }
};

Tensor layer_norm(const Tensor& x, const std::optional<Tensor>& w_, const std::optional<Tensor>& b_, double eps, bool checkpoint) {
    const Tensor w = w_.value_or(Tensor()), b = b_.value_or(Tensor());
    check_traced("layer_norm");
    check_tangents("layer_norm", {&x, &w, &b});
    check_operand("layer_norm", x);
    check_device("layer_norm", "weight", w, x);
    check_device("layer_norm", "bias", b, x);
    if (x.dim() < 1 || x.size(-1) < 1 || x.size(-1) > kNormMaxWidth) value_error("layer_norm: the last axis must hold 1 to ", kNormMaxWidth, " values, got shape ", x.sizes());
    const int64_t D = x.size(-1);
    for (const Tensor* p : {&w, &b})
        if (p->defined() && (p->dim() != 1 || p->size(0) != D || (p->scalar_type() != x.scalar_type() && p->scalar_type() != at::kFloat)))
            value_error("layer_norm: weight and bias must be [", D, "] of dtype ", x.scalar_type(), " or float32, got ", p->sizes(), " ", p->scalar_type());
    if (w.defined() && b.defined() && w.scalar_type() != b.scalar_type()) value_error("layer_norm: weight and bias must have the same dtype");
    if (!(eps >= 0.0)) value_error("layer_norm: eps must be >= 0, got ", eps);
    if (checkpoint && x.scalar_type() == at::kFloat)
        value_error("layer_norm: checkpoint8 takes bfloat16 or float16 (float32 gradients would show the codes' rounding decisions)");
    if (at::GradMode::is_enabled() && (x.requires_grad() || (w.defined() && w.requires_grad()) || (b.defined() && b.requires_grad()))) {
        check_capture("layer_norm", x, {&x, &w, &b});
        return NormNode::apply(x, w_, b_, eps, checkpoint);
    }
    return norm_forward(x, w, b, eps, false, false).y;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    pybind11::register_local_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const LsdmFailure& e) {
            PyErr_SetString(pybind11::module_::import("lsdm_amd._lib").attr("LsdmError").ptr(), e.what());
        }
    });
    m.def("linear", &linear);
    m.def("layer_norm", &layer_norm);
    m.def("pack8", &pack8);
    m.def("unpack8", [](const Tensor& codes, const Tensor& exps, const std::vector<int64_t>& shape, const pybind11::object& dtype) {
        return unpack8(codes, exps, shape, torch::python::detail::py_object_to_dtype(dtype));
    });
}

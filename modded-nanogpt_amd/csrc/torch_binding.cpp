// Host side of linear_act, qk_norm_rope and distill_topk for torch: checks that the tensors can be used as they are, allocates results and
// workspaces, calls the C ABI on the tensors' GPU and its current stream, and records the gradient functions.  Python adds the argument
// messages, the copies of tensors that cannot be used as they are, and the registered operators.  (Written in C++ because a call costs
// 4 to 5 us of host time this way and 12 to 17 from Python, more than the kernels take for one token; gradients run without the interpreter.)
//
// Functions that may be given anything return None for tensors they cannot use as they are; the *_raw ones raise.
#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>
#include <torch/csrc/utils/pybind.h>
#include "../../include/ngpt_fp8.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* out_ptr(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
Tensor given(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

void check(int code, const char* what) {
    if (code != 0) TORCH_CHECK(false, what, " failed with code ", code, ": ", ngpt_last_error());
}

// A tensor that carries a forward-mode derivative is refused wherever it comes in: such derivatives do not go by the grad mode.
const Tensor& no_tangent(const Tensor& t) {
    TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), "nanogpt operators have no forward-mode derivative");
    return t;
}
// Memory on that GPU (the wrappers of torch.func have none).
bool on_gpu(const Tensor& t, const Tensor& like) {
    return !t.defined() || (t.is_cuda() && t.has_storage() && t.device() == like.device() && no_tangent(t).defined());
}
bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

Tensor workspace(int64_t bytes, const Tensor& like) { return bytes > 0 ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor(); }

// [..., K] as rows: their number and stride, if each is contiguous and they are evenly spaced and do not overlap.  A dimension of size one has no
// stride that counts, but the values of a single row have: a column of a matrix is one row, `size` apart.
struct Rows {
    int64_t n = 0, len = 0, ld = 0;
    bool ok = false;
    explicit Rows(const Tensor& t, int64_t most = INT64_MAX) {      // `most`: the longest distance between rows that can be read in place
        const int64_t d = t.dim();
        if (d < 1) return;
        len = t.size(d - 1);
        n = len ? t.numel() / len : 0;
        ld = len;
        ok = t.is_contiguous();
        if (ok || (len > 1 && t.stride(d - 1) != 1)) return;
        ok = n <= 1;
        if (ok) return;
        int64_t i = d - 2;
        while (t.size(i) == 1) --i;                   // (n > 1: there is one)
        ld = t.stride(i);
        ok = ld >= len && ld <= most;
        for (int64_t next = ld; i >= 0; --i) {        // where a dimension has to continue: one distance for all rows
            ok = ok && (t.size(i) == 1 || t.stride(i) == next);
            next *= t.size(i);
        }
    }
};

constexpr int64_t kInt = 0x7fffffff;

// ------------------------------------------------------------------------------------------------ linear_act

bool linear_usable(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& residual) {
    if (!on_gpu(x, x) || !on_gpu(w, x) || !on_gpu(bias, x) || !on_gpu(residual, x)) return false;
    if (w.dim() != 2 || x.dim() < 1 || x.size(-1) != w.size(1)) return false;
    for (const Tensor* t : {&x, &w, &bias, &residual})
        if (t->defined() && t->scalar_type() != at::kBFloat16) return false;
    const Rows xr(x, NGPT_LINEAR_MAX_STRIDE), wr(w, NGPT_LINEAR_MAX_STRIDE);
    if (!xr.ok || !wr.ok || xr.n == 0 || wr.n == 0 || xr.len == 0 || xr.n > kInt || wr.n > kInt || xr.len > kInt) return false;
    if (bias.defined() && (bias.dim() != 1 || bias.size(0) != wr.n || !bias.is_contiguous() || ((uintptr_t)bias.const_data_ptr() & 15))) return false;
    if (residual.defined()) {
        if (residual.dim() != x.dim() || residual.size(-1) != wr.n || !Rows(residual, NGPT_LINEAR_MAX_STRIDE).ok) return false;
        for (int64_t i = 0; i + 1 < x.dim(); ++i)
            if (residual.size(i) != x.size(i)) return false;
    }
    return true;
}

std::tuple<Tensor, Tensor> linear_forward(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& residual, int64_t act, bool keep_pre) {
    const c10::DeviceGuard guard(x.device());
    const Rows xr(x), wr(w);
    auto shape = x.sizes().vec();
    shape.back() = wr.n;
    Tensor out = at::empty(shape, x.options()), pre = keep_pre ? at::empty(shape, x.options()) : Tensor();
    check(ngpt_linear_act_fwd(ptr(x), xr.ld, ptr(w), wr.ld, ptr(bias), ptr(residual), residual.defined() ? Rows(residual).ld : 0, (int)xr.n, (int)wr.n,
                              (int)xr.len, (int)act, out_ptr(out), out_ptr(pre), stream_of(x)), "ngpt_linear_act_fwd");
    return {out, pre};
}

std::tuple<Tensor, Tensor, Tensor> linear_backward(const Tensor& grad, const Tensor& x, const Tensor& w, const Tensor& pre, int64_t act, bool need_dx,
                                                   bool need_dw, bool need_db) {
    const c10::DeviceGuard guard(x.device());
    const Rows xr(x), wr(w);
    const Tensor dout = no_tangent(grad).contiguous().resolve_neg();
    Tensor dx = need_dx ? at::empty(x.sizes(), x.options()) : Tensor(), dw = need_dw ? at::empty(w.sizes(), w.options()) : Tensor();
    Tensor db = need_db ? at::empty({wr.n}, w.options()) : Tensor();
    if (need_dx || need_dw || need_db) {
        const Tensor ws = workspace(ngpt_linear_act_bwd_workspace_bytes_for(ptr(dout), ptr(x), xr.ld, (int)xr.n, (int)wr.n, (int)xr.len, (int)act, need_dx,
                                                                            need_dw, need_db), x);
        check(ngpt_linear_act_bwd(ptr(dout), ptr(pre), ptr(x), xr.ld, ptr(w), wr.ld, (int)xr.n, (int)wr.n, (int)xr.len, (int)act, out_ptr(dx), out_ptr(dw),
                                  out_ptr(db), out_ptr(ws), ws.defined() ? ws.numel() : 0, stream_of(x)), "ngpt_linear_act_bwd");
    }
    return {dx, dw, db};
}

// A gradient of a gradient is not provided.  Where a graph of the backward pass is asked for, the gradients hang on what they were computed from
// (`saved`, `grads`) by a node that raises when it is differentiated, instead of counting as constants.
variable_list once(variable_list result, const variable_list& saved, const variable_list& grads, const char* what) {
    if (!at::GradMode::is_enabled()) return result;
    variable_list from{Tensor()};
    for (const variable_list* list : {&saved, &grads})
        for (const Tensor& t : *list)
            if (wants_grad(t)) from.push_back(t);
    if (from.size() == 1) return result;
    for (Tensor& g : result)
        if (g.defined()) {
            from[0] = g;
            auto refuse = std::make_shared<torch::autograd::DelayedError>(std::string(what) + ": the gradient cannot be differentiated again", (int64_t)from.size());
            g = (*refuse)(variable_list(from))[0];
        }
    return result;
}

struct LinearAct : torch::autograd::Function<LinearAct> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& bias, const OptTensor& residual, int64_t act) {
        const bool keep = act != NGPT_ACT_NONE && (wants_grad(x) || wants_grad(w) || wants_grad(given(bias)));
        auto [out, pre] = linear_forward(x, w, given(bias), given(residual), act, keep);
        ctx->save_for_backward({x, w, pre});
        ctx->saved_data["p"] = (act << 2) | (bias.has_value() ? 1 : 0) | (residual.has_value() ? 2 : 0);
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const int64_t p = ctx->saved_data["p"].toInt();
        const bool has_bias = p & 1, has_res = p & 2;
        variable_list result(5);
        if (!grads[0].defined()) return result;
        const auto saved = ctx->get_saved_variables();
        TORCH_CHECK(linear_usable(saved[0], saved[1], Tensor(), Tensor()) && on_gpu(saved[2], saved[0]) && (!saved[2].defined() || saved[2].is_contiguous()),
                    "linear_act: what was saved for the backward came back in another form");
        auto [dx, dw, db] = linear_backward(grads[0], saved[0], saved[1], saved[2], p >> 2, ctx->needs_input_grad(0), ctx->needs_input_grad(1),
                                            has_bias && ctx->needs_input_grad(2));
        result[0] = dx;
        result[1] = dw;
        result[2] = db;
        result = once(std::move(result), saved, grads, "linear_act");
        if (has_res) result[3] = grads[0];
        return result;
    }
};

OptTensor linear_act(const Tensor& x, const Tensor& w, const OptTensor& bias, const OptTensor& residual, int64_t act) {
    if (!linear_usable(x, w, given(bias), given(residual))) return std::nullopt;
    if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w) || wants_grad(given(bias)) || wants_grad(given(residual))))
        return LinearAct::apply(x, w, bias, residual, act);
    return std::get<0>(linear_forward(x, w, given(bias), given(residual), act, false));
}

std::tuple<Tensor, OptTensor> linear_raw(const Tensor& x, const Tensor& w, const OptTensor& bias, const OptTensor& residual, int64_t act, bool keep_pre) {
    TORCH_CHECK(linear_usable(x, w, given(bias), given(residual)), "linear_act: unusable tensors");
    auto [out, pre] = linear_forward(x, w, given(bias), given(residual), act, keep_pre);
    return {out, pre.defined() ? OptTensor(pre) : std::nullopt};
}

std::tuple<OptTensor, OptTensor, OptTensor> linear_backward_raw(const Tensor& dout, const Tensor& x, const Tensor& w, const OptTensor& pre, int64_t act,
                                                                bool need_dx, bool need_dw, bool need_db) {
    TORCH_CHECK(linear_usable(x, w, Tensor(), Tensor()) && on_gpu(dout, x) && on_gpu(given(pre), x) && dout.scalar_type() == at::kBFloat16 &&
                dout.dim() == x.dim() && dout.size(-1) == w.size(0) && dout.numel() / w.size(0) == x.numel() / w.size(1) &&
                (act == NGPT_ACT_NONE || (pre.has_value() && pre->sizes() == dout.sizes() && pre->is_contiguous())), "linear_act_backward: unusable tensors");
    auto [dx, dw, db] = linear_backward(dout, x, w, given(pre), act, need_dx, need_dw, need_db);
    auto opt = [](const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; };
    return {opt(dx), opt(dw), opt(db)};
}

// ------------------------------------------------------------------------------------------------ qk_norm_rope

struct RopeCall {
    int dtype = 0, tab = 0, B = 1, T = 0, Hq = 0, Hk = 0, D = 0, R = 0, P = 0, pos64 = 0;
    int64_t qs[3], ks[3], ps[2] = {0, 0};
};

int dtype_of(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? NGPT_DT_BF16 : (t.scalar_type() == at::kFloat ? NGPT_DT_F32 : -1); }

void head_strides(const Tensor& t, int64_t (&s)[3]) {
    s[0] = t.dim() == 4 ? t.stride(0) : 0;
    s[1] = t.stride(-3);
    s[2] = t.stride(-2);
}

bool rope_call(RopeCall& c, const Tensor& q, const Tensor& k, const Tensor& cos, const Tensor& sin, const Tensor& pos, const Tensor& qw, const Tensor& kw) {
    if (!on_gpu(q, q)) return false;
    for (const Tensor* t : {&k, &cos, &sin, &pos, &qw, &kw})
        if (!on_gpu(*t, q)) return false;
    const int64_t d = q.dim();
    if ((d != 3 && d != 4) || k.dim() != d || q.size(-1) != k.size(-1)) return false;
    for (int64_t i = 0; i < d - 2; ++i)
        if (q.size(i) != k.size(i)) return false;
    if (q.numel() == 0 || k.numel() == 0 || q.numel() / q.size(-1) > kInt || k.numel() / k.size(-1) > kInt || q.size(-1) > kInt) return false;
    c.dtype = dtype_of(q);
    c.tab = dtype_of(cos);
    if (c.dtype < 0 || k.scalar_type() != q.scalar_type() || c.tab < 0 || sin.scalar_type() != cos.scalar_type()) return false;
    if (cos.dim() != 2 || cos.sizes() != sin.sizes() || !cos.is_contiguous() || !sin.is_contiguous() || cos.size(0) > kInt || cos.size(1) > kInt / 2) return false;
    if (q.stride(-1) != 1 || k.stride(-1) != 1) return false;
    for (const Tensor* t : {&qw, &kw})
        if (t->defined() && (t->dim() != 1 || t->size(0) != q.size(-1) || t->scalar_type() != q.scalar_type() || !t->is_contiguous())) return false;
    c.B = d == 4 ? (int)q.size(0) : 1;
    c.T = (int)q.size(-3);
    c.Hq = (int)q.size(-2);
    c.Hk = (int)k.size(-2);
    c.D = (int)q.size(-1);
    c.R = (int)(2 * cos.size(1));
    c.P = (int)cos.size(0);
    if (pos.defined()) {
        if (pos.scalar_type() != at::kLong && pos.scalar_type() != at::kInt) return false;
        c.pos64 = pos.scalar_type() == at::kLong;
        if (pos.dim() == 1 && pos.size(0) == c.T) c.ps[0] = 0;
        else if (d == 4 && pos.dim() == 2 && pos.size(0) == c.B && pos.size(1) == c.T) c.ps[0] = pos.stride(0);
        else return false;
        c.ps[1] = pos.stride(-1);
    }
    head_strides(q, c.qs);
    head_strides(k, c.ks);
    return true;
}

std::tuple<Tensor, Tensor> rope_forward(const RopeCall& c, const Tensor& q, const Tensor& k, const Tensor& cos, const Tensor& sin, const Tensor& pos,
                                        const Tensor& qw, const Tensor& kw, double eps, bool interleaved) {
    const c10::DeviceGuard guard(q.device());
    Tensor qo = at::empty(q.sizes(), q.options()), ko = at::empty(k.sizes(), k.options());
    check(ngpt_qk_norm_rope(ptr(q), c.qs, ptr(k), c.ks, c.dtype, c.B, c.T, c.Hq, c.Hk, c.D, c.R, ptr(cos), ptr(sin), c.tab, c.P, ptr(pos), c.pos64, c.ps,
                            ptr(qw), ptr(kw), (float)eps, interleaved, out_ptr(qo), out_ptr(ko), stream_of(q)), "ngpt_qk_norm_rope");
    return {qo, ko};
}

Tensor unit_stride(const Tensor& t) { return no_tangent(t).stride(-1) == 1 ? t.resolve_neg() : t.contiguous().resolve_neg(); }

std::tuple<Tensor, Tensor, Tensor, Tensor> rope_backward(const RopeCall& c, const Tensor& gq, const Tensor& gk, const Tensor& q, const Tensor& k, const Tensor& cos,
                                                         const Tensor& sin, const Tensor& pos, const Tensor& qw, const Tensor& kw, double eps,
                                                         bool interleaved, bool need_dqw, bool need_dkw) {
    const c10::DeviceGuard guard(q.device());
    // an output that nothing depends on has no gradient
    const Tensor dqo = gq.defined() ? unit_stride(gq) : at::zeros(q.sizes(), q.options()), dko = gk.defined() ? unit_stride(gk) : at::zeros(k.sizes(), k.options());
    int64_t dqs[3], dks[3];
    head_strides(dqo, dqs);
    head_strides(dko, dks);
    Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options());
    Tensor dqw = need_dqw ? at::empty(qw.sizes(), qw.options()) : Tensor(), dkw = need_dkw ? at::empty(kw.sizes(), kw.options()) : Tensor();
    const Tensor ws = need_dqw || need_dkw ? workspace(ngpt_qk_norm_rope_bwd_workspace_bytes(c.D), q) : Tensor();
    check(ngpt_qk_norm_rope_bwd(ptr(dqo), dqs, ptr(dko), dks, ptr(q), c.qs, ptr(k), c.ks, c.dtype, c.B, c.T, c.Hq, c.Hk, c.D, c.R, ptr(cos), ptr(sin), c.tab, c.P,
                                ptr(pos), c.pos64, c.ps, ptr(qw), ptr(kw), (float)eps, interleaved, out_ptr(dq), out_ptr(dk), out_ptr(dqw), out_ptr(dkw),
                                out_ptr(ws), ws.defined() ? ws.numel() : 0, stream_of(q)), "ngpt_qk_norm_rope_bwd");
    return {dq, dk, dqw, dkw};
}

struct QKNormRope : torch::autograd::Function<QKNormRope> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& cos, const Tensor& sin, const OptTensor& pos,
                                 const OptTensor& qw, const OptTensor& kw, double eps, bool interleaved) {
        RopeCall c;
        TORCH_CHECK(rope_call(c, q, k, cos, sin, given(pos), given(qw), given(kw)), "qk_norm_rope: unusable tensors");
        auto [qo, ko] = rope_forward(c, q, k, cos, sin, given(pos), given(qw), given(kw), eps, interleaved);
        ctx->save_for_backward({q, k, cos, sin, given(pos), given(qw), given(kw)});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["i"] = interleaved;
        ctx->set_materialize_grads(false);
        return {qo, ko};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list result(9);
        if (!grads[0].defined() && !grads[1].defined()) return result;
        const auto s = ctx->get_saved_variables();
        RopeCall c;
        TORCH_CHECK(rope_call(c, s[0], s[1], s[2], s[3], s[4], s[5], s[6]), "qk_norm_rope: what was saved for the backward came back in another form");
        // inputs that are tensors are numbered without the absent ones
        size_t edge = 4 + (s[4].defined() ? 1 : 0);
        const bool need_dqw = s[5].defined() && ctx->needs_input_grad(edge);
        edge += s[5].defined() ? 1 : 0;
        const bool need_dkw = s[6].defined() && ctx->needs_input_grad(edge);
        auto [dq, dk, dqw, dkw] = rope_backward(c, grads[0], grads[1], s[0], s[1], s[2], s[3], s[4], s[5], s[6], ctx->saved_data["eps"].toDouble(),
                                                ctx->saved_data["i"].toBool(), need_dqw, need_dkw);
        result[0] = dq;
        result[1] = dk;
        result[5] = dqw;
        result[6] = dkw;
        return once(std::move(result), s, grads, "qk_norm_rope");
    }
};

using Pair = std::optional<std::tuple<Tensor, Tensor>>;

Pair qk_norm_rope(const Tensor& q, const Tensor& k, const Tensor& cos, const Tensor& sin, const OptTensor& pos, const OptTensor& qw, const OptTensor& kw,
                  double eps, bool interleaved) {
    RopeCall c;
    if (!rope_call(c, q, k, cos, sin, given(pos), given(qw), given(kw))) return std::nullopt;
    if (at::GradMode::is_enabled() && (wants_grad(q) || wants_grad(k) || wants_grad(given(qw)) || wants_grad(given(kw)))) {
        auto r = QKNormRope::apply(q, k, cos, sin, pos, qw, kw, eps, interleaved);
        return std::make_tuple(r[0], r[1]);
    }
    return rope_forward(c, q, k, cos, sin, given(pos), given(qw), given(kw), eps, interleaved);
}

std::tuple<Tensor, Tensor, OptTensor, OptTensor> rope_backward_raw(const Tensor& gq, const Tensor& gk, const Tensor& q, const Tensor& k, const Tensor& cos,
                                                                   const Tensor& sin, const OptTensor& pos, const OptTensor& qw, const OptTensor& kw,
                                                                   double eps, bool interleaved, bool need_dqw, bool need_dkw) {
    RopeCall c;
    TORCH_CHECK(rope_call(c, q, k, cos, sin, given(pos), given(qw), given(kw)) && on_gpu(gq, q) && on_gpu(gk, q) && gq.sizes() == q.sizes() &&
                gk.sizes() == k.sizes() && gq.scalar_type() == q.scalar_type() && gk.scalar_type() == q.scalar_type() && (!need_dqw || qw.has_value()) &&
                (!need_dkw || kw.has_value()), "qk_norm_rope_backward: unusable tensors");
    auto [dq, dk, dqw, dkw] = rope_backward(c, gq, gk, q, k, cos, sin, given(pos), given(qw), given(kw), eps, interleaved, need_dqw, need_dkw);
    auto opt = [](const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; };
    return {dq, dk, opt(dqw), opt(dkw)};
}

// ------------------------------------------------------------------------------------------------ distill_topk

struct DistillParams {
    double tau, A, B, C;
};

bool distill_usable(const Tensor& logits, const Tensor& ids, const Tensor& teacher, const Tensor& lse, const Tensor& weight) {
    if (!on_gpu(logits, logits)) return false;
    for (const Tensor* t : {&ids, &teacher, &lse, &weight})
        if (!on_gpu(*t, logits) || (t->defined() && !t->is_contiguous())) return false;
    if (logits.dim() != 2 || dtype_of(logits) < 0 || !Rows(logits).ok || logits.numel() == 0 || logits.size(0) > kInt || logits.size(1) > kInt) return false;
    const int64_t T = logits.size(0);
    if (ids.dim() != 2 || ids.size(0) != T || ids.size(1) == 0 || ids.size(1) > kInt || (ids.scalar_type() != at::kLong && ids.scalar_type() != at::kInt)) return false;
    if (teacher.sizes() != ids.sizes() || teacher.scalar_type() != at::kFloat) return false;
    for (const Tensor* t : {&lse, &weight})
        if (t->defined() && (t->dim() != 1 || t->size(0) != T || t->scalar_type() != at::kFloat)) return false;
    return true;
}

#define DISTILL_ARGS                                                                                                                              \
    ptr(logits), dtype_of(logits), Rows(logits).ld, ptr(ids), ids.scalar_type() == at::kLong, (const float*)ptr(teacher), (const float*)ptr(lse), \
        (const float*)ptr(weight), (int)logits.size(0), (int)logits.size(1), (int)ids.size(1), (float)p.tau, (float)p.A, (float)p.B, (float)p.C

std::tuple<Tensor, Tensor> distill_forward(const Tensor& logits, const Tensor& ids, const Tensor& teacher, const Tensor& lse, const Tensor& weight,
                                           const DistillParams& p, bool keep_stats) {
    const c10::DeviceGuard guard(logits.device());
    const auto f32 = logits.options().dtype(at::kFloat);
    Tensor losses = at::empty({logits.size(0)}, f32), stats = keep_stats ? at::empty({logits.size(0), 4}, f32) : Tensor();
    check(ngpt_distill_fwd(DISTILL_ARGS, (float*)out_ptr(losses), (float*)out_ptr(stats), stream_of(logits)), "ngpt_distill_fwd");
    return {losses, stats};
}

Tensor distill_backward(const Tensor& grad_, const Tensor& logits, const Tensor& ids, const Tensor& teacher, const Tensor& lse, const Tensor& weight,
                        const Tensor& stats, const DistillParams& p) {
    const c10::DeviceGuard guard(logits.device());
    const Tensor dlosses = no_tangent(grad_).resolve_neg();
    Tensor grad = at::empty(logits.sizes(), logits.options());
    check(ngpt_distill_bwd(DISTILL_ARGS, (const float*)ptr(stats), (const float*)ptr(dlosses), dlosses.stride(0), out_ptr(grad), logits.size(1),
                           stream_of(logits)), "ngpt_distill_bwd");
    return grad;
}

struct DistillTopK : torch::autograd::Function<DistillTopK> {
    static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& ids, const Tensor& teacher, const OptTensor& lse, const OptTensor& weight,
                          double tau, double A, double B, double C) {
        auto [losses, stats] = distill_forward(logits, ids, teacher, given(lse), given(weight), {tau, A, B, C}, true);
        ctx->save_for_backward({logits, ids, teacher, given(lse), given(weight), stats});
        ctx->saved_data["p"] = std::vector<double>{tau, A, B, C};
        return losses;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list result(9);
        if (!grads[0].defined()) return result;
        const auto s = ctx->get_saved_variables();
        const auto v = ctx->saved_data["p"].toDoubleVector();
        TORCH_CHECK(distill_usable(s[0], s[1], s[2], s[3], s[4]) && on_gpu(s[5], s[0]) && s[5].is_contiguous(),
                    "distill_topk: what was saved for the backward came back in another form");
        result[0] = distill_backward(grads[0], s[0], s[1], s[2], s[3], s[4], s[5], {v[0], v[1], v[2], v[3]});
        return once(std::move(result), s, grads, "distill_topk");
    }
};

OptTensor distill_topk(const Tensor& logits, const Tensor& ids, const Tensor& teacher, const OptTensor& lse, const OptTensor& weight, double tau, double A,
                       double B, double C) {
    if (!distill_usable(logits, ids, teacher, given(lse), given(weight))) return std::nullopt;
    if (at::GradMode::is_enabled() && wants_grad(logits)) return DistillTopK::apply(logits, ids, teacher, lse, weight, tau, A, B, C);
    return std::get<0>(distill_forward(logits, ids, teacher, given(lse), given(weight), {tau, A, B, C}, false));
}

std::tuple<Tensor, Tensor> distill_raw(const Tensor& logits, const Tensor& ids, const Tensor& teacher, const OptTensor& lse, const OptTensor& weight, double tau,
                                       double A, double B, double C) {
    TORCH_CHECK(distill_usable(logits, ids, teacher, given(lse), given(weight)), "distill_topk: unusable tensors");
    return distill_forward(logits, ids, teacher, given(lse), given(weight), {tau, A, B, C}, true);
}

Tensor distill_backward_raw(const Tensor& dlosses, const Tensor& logits, const Tensor& ids, const Tensor& teacher, const OptTensor& lse, const OptTensor& weight,
                            const Tensor& stats, double tau, double A, double B, double C) {
    TORCH_CHECK(distill_usable(logits, ids, teacher, given(lse), given(weight)) && on_gpu(dlosses, logits) && on_gpu(stats, logits) && dlosses.dim() == 1 &&
                dlosses.size(0) == logits.size(0) && dlosses.scalar_type() == at::kFloat && stats.scalar_type() == at::kFloat && stats.is_contiguous() &&
                stats.numel() == 4 * logits.size(0), "distill_topk_backward: unusable tensors");
    return distill_backward(dlosses, logits, ids, teacher, given(lse), given(weight), stats, {tau, A, B, C});
}

Pair distill_fused(const Tensor& logits, const Tensor& ids, const Tensor& teacher, const OptTensor& lse_, const OptTensor& weight_, double tau, double A, double B,
                   double C, double grad_scale) {
    const Tensor lse = given(lse_), weight = given(weight_);
    const DistillParams p{tau, A, B, C};
    if (!distill_usable(logits, ids, teacher, lse, weight)) return std::nullopt;
    const c10::DeviceGuard guard(logits.device());
    if (logits.size(1) > ngpt_distill_fused_max_cols(dtype_of(logits))) {      // a row longer than a workgroup's registers: two passes
        auto [losses, stats] = distill_forward(logits, ids, teacher, lse, weight, p, true);
        const Tensor scale = at::full({1}, grad_scale, logits.options().dtype(at::kFloat)).expand({logits.size(0)});
        return std::make_tuple(losses, distill_backward(scale, logits, ids, teacher, lse, weight, stats, p));
    }
    Tensor losses = at::empty({logits.size(0)}, logits.options().dtype(at::kFloat)), grad = at::empty(logits.sizes(), logits.options());
    check(ngpt_distill_fwd_bwd(DISTILL_ARGS, (float)grad_scale, (float*)out_ptr(losses), out_ptr(grad), logits.size(1), stream_of(logits)),
          "ngpt_distill_fwd_bwd");
    return std::make_tuple(losses, grad);
}

// ------------------------------------------------------------------------------------------------ for Python

// The public functions' first call, without pybind's conversions (they take 1 us): positional arguments only.  None is returned for anything but
// ordinary tensors in usable form, and under a dispatch mode (a tracer, a counter of operations), which has to see the registered operator.
struct Given {
    PyObject* const* args;
    bool ok = !c10::impl::TorchDispatchModeTLS::any_modes_set() && !at::tracer::impl::is_dispatch_enabled();

    OptTensor maybe(int i) {
        PyObject* o = args[i];
        if (o == Py_None) return std::nullopt;
        if (!THPVariable_CheckTypeExact(Py_TYPE(o))) {      // Tensor or Parameter: a subclass may mean something else
            ok = false;
            return std::nullopt;
        }
        const Tensor& t = THPVariable_Unpack(o);
        ok = ok && !t.is_neg();                             // memory that holds the negated values: the dispatcher makes them real
        return t;
    }
    Tensor tensor(int i) {
        OptTensor t = maybe(i);
        ok = ok && t.has_value();
        return t.has_value() ? std::move(*t) : Tensor();
    }
    double number(int i) {
        const double v = PyFloat_AsDouble(args[i]);
        if (v == -1.0 && PyErr_Occurred()) throw python_error();
        return v;
    }
    int64_t integer(int i) {
        const int64_t v = PyLong_AsLongLong(args[i]);
        if (v == -1 && PyErr_Occurred()) throw python_error();
        return v;
    }
};

PyObject* to_python(OptTensor t) {
    if (!t.has_value()) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(*t));
}
PyObject* to_python(Pair t) {
    if (!t.has_value()) Py_RETURN_NONE;
    THPObjectPtr a(THPVariable_Wrap(std::move(std::get<0>(*t)))), b(THPVariable_Wrap(std::move(std::get<1>(*t))));
    return a && b ? PyTuple_Pack(2, a.get(), b.get()) : nullptr;
}

PyObject* py_linear_act(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 5, "linear_act: 5 arguments");
    Given g{args};
    const Tensor x = g.tensor(0), w = g.tensor(1);
    const OptTensor bias = g.maybe(2), residual = g.maybe(3);
    if (!g.ok) Py_RETURN_NONE;
    return to_python(linear_act(x, w, bias, residual, g.integer(4)));
    END_HANDLE_TH_ERRORS
}

PyObject* py_qk_norm_rope(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 9, "qk_norm_rope: 9 arguments");
    Given g{args};
    const Tensor q = g.tensor(0), k = g.tensor(1), cos = g.tensor(2), sin = g.tensor(3);
    const OptTensor pos = g.maybe(4), qw = g.maybe(5), kw = g.maybe(6);
    if (!g.ok) Py_RETURN_NONE;
    return to_python(qk_norm_rope(q, k, cos, sin, pos, qw, kw, g.number(7), g.integer(8) != 0));
    END_HANDLE_TH_ERRORS
}

PyObject* py_distill_topk(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 9, "distill_topk: 9 arguments");
    Given g{args};
    const Tensor logits = g.tensor(0), ids = g.tensor(1), teacher = g.tensor(2);
    const OptTensor lse = g.maybe(3), weight = g.maybe(4);
    if (!g.ok) Py_RETURN_NONE;
    return to_python(distill_topk(logits, ids, teacher, lse, weight, g.number(5), g.number(6), g.number(7), g.number(8)));
    END_HANDLE_TH_ERRORS
}

PyObject* py_distill_fused(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 10, "distill_fused: 10 arguments");
    Given g{args};
    const Tensor logits = g.tensor(0), ids = g.tensor(1), teacher = g.tensor(2);
    const OptTensor lse = g.maybe(3), weight = g.maybe(4);
    if (!g.ok) Py_RETURN_NONE;
    return to_python(distill_fused(logits, ids, teacher, lse, weight, g.number(5), g.number(6), g.number(7), g.number(8), g.number(9)));
    END_HANDLE_TH_ERRORS
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) { return {name, (PyCFunction)(void (*)(void))F, METH_FASTCALL, nullptr}; }

PyMethodDef methods[] = {method<py_linear_act>("linear_act"), method<py_qk_norm_rope>("qk_norm_rope"), method<py_distill_topk>("distill_topk"),
                         method<py_distill_fused>("distill_fused"), {nullptr, nullptr, 0, nullptr}};

}  // namespace

PYBIND11_MODULE(_ngpt_torch, m) {
    if (PyModule_AddFunctions(m.ptr(), methods) != 0) throw pybind11::error_already_set();
    // the one rule for Python's copies too; looks at sizes and strides only
    m.def("rows_in_place", [](const Tensor& t, int64_t most) { return Rows(t, most).ok; }, pybind11::arg("t"), pybind11::arg("most") = INT64_MAX);
    m.attr("LINEAR_MAX_STRIDE") = NGPT_LINEAR_MAX_STRIDE;
    m.def("linear_raw", &linear_raw);
    m.def("linear_backward_raw", &linear_backward_raw);
    m.def("rope_backward_raw", &rope_backward_raw);
    m.def("distill_raw", &distill_raw);
    m.def("distill_backward_raw", &distill_backward_raw);
}

"""Operators around the attention and MLP of a block, and the loss against a teacher:

    linear_act             out = residual + act(x @ w.T + bias), differentiable in all four
    qk_norm_rope           per-head rms norm of queries and keys and the position rotation in one pass, differentiable
    distill_topk           distillation loss against a teacher's top logits, differentiable in the student's logits
    distill_topk_fwd_bwd   the same loss and its gradient at once, reading the logits once

The functions go straight to the kernels of libngpt_fp8.so through the compiled torch binding; under `torch.compile` or with fake tensors they
go through the registered operators nanogpt::linear_act, qk_norm_rope, distill_topk (and their *_backward), which do the same.  All tensors
of a call live on one GPU; work is enqueued on that GPU's current stream.  There is no CPU implementation.
"""
from __future__ import annotations

import torch
from torch import Tensor
from torch.compiler import is_dynamo_compiling

from . import _lib

ACTIVATIONS = {"none": 0, "relu2": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
RMS_EPS = 1.1920928955078125e-07          # machine epsilon of fp32, what the other norms of this package add
_FLOATS = (torch.bfloat16, torch.float32)
_binding = None


def _b():
    """The compiled binding, loaded on first use."""
    global _binding
    if _binding is None:
        _binding = _lib.load_torch()
    return _binding


def _same_gpu(first: Tensor, *others: Tensor | None) -> None:
    for t in (first, *others):
        if t is not None and not t.is_cuda:
            raise RuntimeError("nanogpt operators run on the GPU only (got a CPU tensor); there is no CPU fallback")
        assert t is None or t.device == first.device, f"tensors on {first.device} and {t.device}"


def _plain(*tensors: Tensor | None) -> bool:
    """Ordinary tensors that hold their own values, outside of a trace and of dispatch modes: the kernels can be launched here."""
    if torch.compiler.is_compiling() or torch._C._len_torch_dispatch_stack() or torch._C._get_tracing_state() is not None:
        return False
    for t in tensors:
        if t is not None and (type(t) is not Tensor and type(t) is not torch.nn.Parameter or t.is_neg()):
            return False
    return True


def _rows(t: Tensor | None, *most: int) -> Tensor | None:
    """[..., K] whose rows are contiguous, evenly spaced (at most `most` values apart) and do not overlap: itself, or a copy."""
    return t if t is None or t.ndim == 0 or _b().rows_in_place(t, *most) else t.contiguous()


def _direct(*tensors: Tensor | None) -> bool:
    """Memory that a kernel can be given: not the meta device, whose tensors take the registered operators."""
    for t in tensors:
        if t is not None and torch._C._functorch.is_functorch_wrapped_tensor(t):
            raise RuntimeError("nanogpt operators do not go through torch.func's transforms; use torch.autograd")
    return not any(t is not None and t.is_meta for t in tensors)


def _launched(out, what: str):
    if out is None:
        raise RuntimeError(f"{what}: the kernels cannot take these tensors (a dimension of 2^31 or more, no heads, or a tensor without memory of its own)")
    return out


def _contiguous(t: Tensor | None) -> Tensor | None:
    return None if t is None else t.contiguous()


# ------------------------------------------------------------------------------------------------
# linear_act

def _linear_shapes(x: Tensor, w: Tensor, bias: Tensor | None, residual: Tensor | None, activation: str) -> int:
    assert activation in ACTIVATIONS, f"activation {activation!r}: one of {', '.join(ACTIVATIONS)}"
    assert w.ndim == 2 and x.ndim >= 1 and x.shape[-1] == w.shape[1], f"x {tuple(x.shape)} and w {tuple(w.shape)}: x is [..., K], w [N, K]"
    assert bias is None or bias.shape == (w.shape[0],), f"bias {tuple(bias.shape)}: one value per row of w"
    assert residual is None or residual.shape == (*x.shape[:-1], w.shape[0]), f"residual {tuple(residual.shape)}: the shape of the result"
    for t in (x, w, bias, residual):
        assert t is None or t.dtype == torch.bfloat16, f"linear_act takes bfloat16, got {t.dtype}"
    return ACTIVATIONS[activation]


def _linear_usable(x, w, bias, residual):
    """The same values in a form the kernels read in place (these copies are differentiable)."""
    if bias is not None and (not bias.is_contiguous() or bias.data_ptr() % 16):
        bias = bias.clone(memory_format=torch.contiguous_format)
    most = _b().LINEAR_MAX_STRIDE
    return _rows(x, most), _rows(w, most), bias, _rows(residual, most)


@torch.library.custom_op("nanogpt::linear_act", mutates_args=())
def linear_act_op(x: Tensor, w: Tensor, bias: Tensor | None, residual: Tensor | None, activation: str, keep_pre: bool) -> tuple[Tensor, Tensor]:
    """-> (out, pre): pre [.., N] = x @ w.T + bias if keep_pre (which needs an activation), else empty."""
    act = _linear_shapes(x, w, bias, residual, activation)
    _same_gpu(x, w, bias, residual)
    assert act or not keep_pre, "keep_pre: without an activation the backward needs no pre-activation"
    shape = (*x.shape[:-1], w.shape[0])
    if x.numel() == 0 or w.numel() == 0:
        assert x.shape[-1] > 0, "linear_act: a contraction of length 0"
        out = x.new_empty(shape)
        return out, out.new_empty(shape if keep_pre else 0)
    out, pre = _b().linear_raw(*_linear_usable(x, w, bias, residual), act, keep_pre)
    return out, out.new_empty(0) if pre is None else pre


@linear_act_op.register_fake
def _(x, w, bias, residual, activation, keep_pre):
    _linear_shapes(x, w, bias, residual, activation)
    out = x.new_empty((*x.shape[:-1], w.shape[0]))
    return out, torch.empty_like(out) if keep_pre else x.new_empty(0)


@torch.library.custom_op("nanogpt::linear_act_backward", mutates_args=())
def linear_act_backward_op(dout: Tensor, x: Tensor, w: Tensor, pre: Tensor | None, activation: str, need_dx: bool, need_dw: bool,
                           need_dbias: bool) -> tuple[Tensor, Tensor, Tensor]:
    """-> (dx, dw, dbias), empty where not wanted.  (The residual's gradient is dout.)"""
    act = ACTIVATIONS[activation]
    assert dout.shape == (*x.shape[:-1], w.shape[0]) and dout.dtype == x.dtype == w.dtype == torch.bfloat16
    assert not act or pre is not None and pre.shape == dout.shape, "the backward of an activation needs the forward's pre-activation"
    _same_gpu(x, w, dout, pre)
    if x.numel() == 0 or w.numel() == 0:
        shapes = (need_dx, x.shape), (need_dw, w.shape), (need_dbias, w.shape[:1])
        return tuple(x.new_zeros(shape if want else 0) for want, shape in shapes)
    x, w, _, _ = _linear_usable(x, w, None, None)
    r = _b().linear_backward_raw(dout, x, w, _contiguous(pre) if act else None, act, need_dx, need_dw, need_dbias)
    return tuple(dout.new_empty(0) if t is None else t for t in r)


@linear_act_backward_op.register_fake
def _(dout, x, w, pre, activation, need_dx, need_dw, need_dbias):
    e = lambda want, *shape: x.new_empty(shape if want else (0,))
    return e(need_dx, *x.shape), e(need_dw, *w.shape), e(need_dbias, w.shape[0])


def _linear_setup(ctx, inputs, output):
    x, w, bias, residual, activation, keep_pre = inputs
    ctx.save_for_backward(x, w, output[1] if keep_pre else None)
    ctx.activation = activation
    ctx.set_materialize_grads(False)


def _linear_backward(ctx, dout, _dpre):
    x, w, pre = ctx.saved_tensors
    if dout is None:
        return None, None, None, None, None, None
    need = ctx.needs_input_grad
    if not any(need[:3]):               # the residual alone: there is no pre-activation then
        return None, None, None, dout, None, None
    dx, dw, db = torch.ops.nanogpt.linear_act_backward(dout, x, w, pre, ctx.activation, need[0], need[1], need[2])
    return (dx if need[0] else None, dw if need[1] else None, db if need[2] else None, dout if need[3] else None, None, None)


linear_act_op.register_autograd(_linear_backward, setup_context=_linear_setup)


def linear_act(x: Tensor, w: Tensor, bias: Tensor | None = None, residual: Tensor | None = None, activation: str = "none") -> Tensor:
    """residual + act(x @ w.T + bias) for bf16 x [..., K], w [N, K], bias [N], residual [..., N]; fp32 accumulation, bias, activation
    and residual applied to the fp32 sums, one rounding.  `activation`: "none", "relu2" (max(z, 0)^2), "gelu", "gelu_tanh", "silu".
    Any sizes (2^29 rows, 2^21 values in one).  Rows of x, w and residual are read in place if they are contiguous and evenly spaced, at most
    2^21 values apart; other layouts are copied.  Differentiable in x, w, bias and residual; an activation's backward keeps
    the bf16 pre-activation and rounds its gradient to bf16 for the two products."""
    if not is_dynamo_compiling():       # straight to the binding, which takes ordinary tensors in usable form
        act = ACTIVATIONS.get(activation)
        if act is not None:
            out = (_binding or _b()).linear_act(x, w, bias, residual, act)
            if out is not None:
                return out
    if _plain(x, w, bias, residual):
        act = _linear_shapes(x, w, bias, residual, activation)
        if _direct(x, w, bias, residual):
            _same_gpu(x, w, bias, residual)
            if x.numel() and w.numel():
                return _launched(_b().linear_act(*_linear_usable(x, w, bias, residual), act), "linear_act")
    keep = activation != "none" and torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, w, bias))
    return torch.ops.nanogpt.linear_act(x, w, bias, residual, activation, keep)[0]


# ------------------------------------------------------------------------------------------------
# qk_norm_rope

def _rope_shapes(q: Tensor, k: Tensor, cos: Tensor, sin: Tensor, positions: Tensor | None, q_weight: Tensor | None, k_weight: Tensor | None) -> None:
    assert q.ndim in (3, 4) and k.ndim == q.ndim and q.shape[:-2] == k.shape[:-2] and q.shape[-1] == k.shape[-1], (
        f"q {tuple(q.shape)} and k {tuple(k.shape)}: [T, H, D] or [B, T, H, D] with the same tokens and head size")
    assert q.dtype in _FLOATS and k.dtype == q.dtype, f"q {q.dtype} and k {k.dtype}: both bfloat16 or both float32"
    assert cos.ndim == 2 and cos.shape == sin.shape and cos.dtype == sin.dtype and cos.dtype in _FLOATS, (
        "cos and sin: [positions, rotated / 2], both bfloat16 or both float32")
    tokens = tuple(q.shape[:-2])
    assert positions is None or (positions.dtype in (torch.int32, torch.int64) and tuple(positions.shape) in (tokens, tokens[-1:])), (
        f"positions: int32 or int64, of shape {tokens} or {tokens[-1:]}")
    for w in (q_weight, k_weight):
        assert w is None or (w.shape == (q.shape[-1],) and w.dtype == q.dtype), "weights: one value per head element, in the heads' type"


def _rope_usable(q, k, cos, sin, positions, q_weight, k_weight):
    heads = lambda t: t if t.stride(-1) == 1 else t.contiguous()
    return heads(q), heads(k), cos.contiguous(), sin.contiguous(), positions, _contiguous(q_weight), _contiguous(k_weight)


@torch.library.custom_op("nanogpt::qk_norm_rope", mutates_args=())
def qk_norm_rope_op(q: Tensor, k: Tensor, cos: Tensor, sin: Tensor, positions: Tensor | None, q_weight: Tensor | None, k_weight: Tensor | None,
                    eps: float, interleaved: bool) -> tuple[Tensor, Tensor]:
    tensors = (q, k, cos, sin, positions, q_weight, k_weight)
    _rope_shapes(*tensors)
    _same_gpu(*tensors)
    if q.numel() == 0 and k.numel() == 0:
        return q.new_empty(q.shape), k.new_empty(k.shape)
    with torch.no_grad():
        return _launched(_b().qk_norm_rope(*_rope_usable(*tensors), eps, interleaved), "qk_norm_rope")


@qk_norm_rope_op.register_fake
def _(q, k, cos, sin, positions, q_weight, k_weight, eps, interleaved):
    _rope_shapes(q, k, cos, sin, positions, q_weight, k_weight)
    return q.new_empty(q.shape), k.new_empty(k.shape)


@torch.library.custom_op("nanogpt::qk_norm_rope_backward", mutates_args=())
def qk_norm_rope_backward_op(dq_out: Tensor, dk_out: Tensor, q: Tensor, k: Tensor, cos: Tensor, sin: Tensor, positions: Tensor | None,
                             q_weight: Tensor | None, k_weight: Tensor | None, eps: float, interleaved: bool, need_dq_weight: bool,
                             need_dk_weight: bool) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """-> (dq, dk, dq_weight, dk_weight), the weights' empty where not wanted."""
    tensors = (q, k, cos, sin, positions, q_weight, k_weight)
    _rope_shapes(*tensors)
    _same_gpu(*tensors, dq_out, dk_out)
    assert dq_out.shape == q.shape and dk_out.shape == k.shape and dq_out.dtype == q.dtype and dk_out.dtype == k.dtype
    D = q.shape[-1]
    if q.numel() == 0 and k.numel() == 0:
        return q.new_empty(q.shape), k.new_empty(k.shape), q.new_zeros(D if need_dq_weight else 0), q.new_zeros(D if need_dk_weight else 0)
    r = _b().rope_backward_raw(dq_out, dk_out, *_rope_usable(*tensors), eps, interleaved, need_dq_weight, need_dk_weight)
    return tuple(q.new_empty(0) if t is None else t for t in r)


@qk_norm_rope_backward_op.register_fake
def _(dq_out, dk_out, q, k, cos, sin, positions, q_weight, k_weight, eps, interleaved, need_dq_weight, need_dk_weight):
    D = q.shape[-1]
    return q.new_empty(q.shape), k.new_empty(k.shape), q.new_empty(D if need_dq_weight else 0), q.new_empty(D if need_dk_weight else 0)


def _rope_setup(ctx, inputs, output):
    q, k, cos, sin, positions, q_weight, k_weight, eps, interleaved = inputs
    ctx.save_for_backward(q, k, cos, sin, positions, q_weight, k_weight)
    ctx.params = eps, interleaved


def _rope_backward(ctx, dq_out, dk_out):
    q, k, cos, sin, positions, q_weight, k_weight = ctx.saved_tensors
    need = ctx.needs_input_grad
    dq, dk, dqw, dkw = torch.ops.nanogpt.qk_norm_rope_backward(dq_out, dk_out, q, k, cos, sin, positions, q_weight, k_weight, *ctx.params,
                                                               need[5], need[6])
    return dq, dk, None, None, None, dqw if need[5] else None, dkw if need[6] else None, None, None


qk_norm_rope_op.register_autograd(_rope_backward, setup_context=_rope_setup)


def qk_norm_rope(q: Tensor, k: Tensor, cos: Tensor, sin: Tensor, positions: Tensor | None = None, q_weight: Tensor | None = None,
                 k_weight: Tensor | None = None, eps: float | None = None, interleaved: bool = False) -> tuple[Tensor, Tensor]:
    """(rot(norm(q)), rot(norm(k))) for q [T, Hq, D] or [B, T, Hq, D] and k likewise with its own number of heads, bf16 or fp32; views of
    a packed projection are read in place.  norm is over each head's D values (eps None: the machine epsilon of fp32), times the weight
    [D] if given.  The first R values of a head are rotated, R / 2 = cos.shape[1]: pairs (i, i + R / 2), or (2 i, 2 i + 1) if
    interleaved, (a, b) -> (a cos - b sin, b cos + a sin) with row `positions[token]` of cos and sin (None: the token's index in its
    sequence).  A position outside the tables makes that token's heads NaN.  2 <= D <= 512.  Differentiable in q, k and the weights."""
    eps = RMS_EPS if eps is None else float(eps)
    tensors = (q, k, cos, sin, positions, q_weight, k_weight)
    if not is_dynamo_compiling():
        out = (_binding or _b()).qk_norm_rope(*tensors, eps, interleaved)
        if out is not None:
            return out
    if _plain(*tensors):
        _rope_shapes(*tensors)
        if _direct(*tensors):
            _same_gpu(*tensors)
            if q.numel() or k.numel():
                return _launched(_b().qk_norm_rope(*_rope_usable(*tensors), eps, interleaved), "qk_norm_rope")
    return torch.ops.nanogpt.qk_norm_rope(*tensors, eps, interleaved)


# ------------------------------------------------------------------------------------------------
# distill_topk

def _distill_shapes(logits, ids, teacher, teacher_lse, row_weight) -> None:
    assert logits.ndim == 2 and logits.dtype in _FLOATS, f"logits {tuple(logits.shape)} {logits.dtype}: [T, V], bfloat16 or float32"
    T = logits.shape[0]
    assert ids.ndim == 2 and ids.shape[0] == T and ids.dtype in (torch.int32, torch.int64), f"ids {tuple(ids.shape)} {ids.dtype}: [T, K] int32 or int64"
    assert teacher.shape == ids.shape and teacher.dtype == torch.float32, f"teacher {tuple(teacher.shape)} {teacher.dtype}: float32, one logit per id"
    for name, t in (("teacher_lse", teacher_lse), ("row_weight", row_weight)):
        assert t is None or (t.shape == (T,) and t.dtype == torch.float32), f"{name}: [T] float32"


def _distill_usable(logits, ids, teacher, teacher_lse, row_weight):
    return _rows(logits), ids.contiguous(), teacher.contiguous(), _contiguous(teacher_lse), _contiguous(row_weight)


def _nothing_listed(logits, ids) -> bool:
    return logits.numel() == 0 or ids.numel() == 0


@torch.library.custom_op("nanogpt::distill_topk", mutates_args=())
def distill_topk_op(logits: Tensor, ids: Tensor, teacher: Tensor, teacher_lse: Tensor | None, row_weight: Tensor | None, temperature: float,
                    A: float, B: float, C: float) -> tuple[Tensor, Tensor]:
    """-> (losses [T], stats [T, 4] for the backward).  C = 0: no softcap."""
    tensors = (logits, ids, teacher, teacher_lse, row_weight)
    _distill_shapes(*tensors)
    _same_gpu(*tensors)
    if _nothing_listed(logits, ids):
        return logits.new_zeros(logits.shape[0], dtype=torch.float32), logits.new_zeros((logits.shape[0], 4), dtype=torch.float32)
    return _b().distill_raw(*_distill_usable(*tensors), temperature, A, B, C)


@distill_topk_op.register_fake
def _(logits, ids, teacher, teacher_lse, row_weight, temperature, A, B, C):
    _distill_shapes(logits, ids, teacher, teacher_lse, row_weight)
    T = logits.shape[0]
    return logits.new_empty(T, dtype=torch.float32), logits.new_empty((T, 4), dtype=torch.float32)


@torch.library.custom_op("nanogpt::distill_topk_backward", mutates_args=())
def distill_topk_backward_op(dlosses: Tensor, logits: Tensor, ids: Tensor, teacher: Tensor, teacher_lse: Tensor | None, row_weight: Tensor | None,
                             stats: Tensor, temperature: float, A: float, B: float, C: float) -> Tensor:
    tensors = (logits, ids, teacher, teacher_lse, row_weight)
    _distill_shapes(*tensors)
    _same_gpu(*tensors, dlosses, stats)
    assert dlosses.shape == logits.shape[:1] and dlosses.dtype == torch.float32
    if _nothing_listed(logits, ids):
        return logits.new_zeros(logits.shape)
    return _b().distill_backward_raw(dlosses, *_distill_usable(*tensors), stats, temperature, A, B, C)


@distill_topk_backward_op.register_fake
def _(dlosses, logits, ids, teacher, teacher_lse, row_weight, stats, temperature, A, B, C):
    return logits.new_empty(logits.shape)


@torch.library.custom_op("nanogpt::distill_topk_fwd_bwd", mutates_args=())
def distill_topk_fwd_bwd_op(logits: Tensor, ids: Tensor, teacher: Tensor, teacher_lse: Tensor | None, row_weight: Tensor | None, temperature: float,
                            A: float, B: float, C: float, grad_scale: float) -> tuple[Tensor, Tensor]:
    tensors = (logits, ids, teacher, teacher_lse, row_weight)
    _distill_shapes(*tensors)
    _same_gpu(*tensors)
    if _nothing_listed(logits, ids):
        return logits.new_zeros(logits.shape[0], dtype=torch.float32), logits.new_zeros(logits.shape)
    return _launched(_b().distill_fused(*_distill_usable(*tensors), temperature, A, B, C, grad_scale), "distill_topk_fwd_bwd")


@distill_topk_fwd_bwd_op.register_fake
def _(logits, ids, teacher, teacher_lse, row_weight, temperature, A, B, C, grad_scale):
    _distill_shapes(logits, ids, teacher, teacher_lse, row_weight)
    return logits.new_empty(logits.shape[0], dtype=torch.float32), logits.new_empty(logits.shape)


def _distill_setup(ctx, inputs, output):
    logits, ids, teacher, teacher_lse, row_weight, *params = inputs
    ctx.save_for_backward(logits, ids, teacher, teacher_lse, row_weight, output[1])
    ctx.params = params
    ctx.set_materialize_grads(False)


def _distill_backward(ctx, dlosses, _dstats):
    grad = None
    if dlosses is not None:
        logits, ids, teacher, teacher_lse, row_weight, stats = ctx.saved_tensors
        grad = torch.ops.nanogpt.distill_topk_backward(dlosses, logits, ids, teacher, teacher_lse, row_weight, stats, *ctx.params)
    return grad, None, None, None, None, None, None, None, None


distill_topk_op.register_autograd(_distill_backward, setup_context=_distill_setup)


def _softcap(softcap) -> tuple[float, float, float]:
    if softcap is None:
        return 0.0, 0.0, 0.0
    A, B, C = (float(v) for v in softcap)
    assert A > 0 and C > 0, f"softcap {softcap}: A sigmoid((l + B) / C) needs A, C > 0"
    return A, B, C


def distill_topk(logits: Tensor, ids: Tensor, teacher: Tensor, teacher_lse: Tensor | None = None, row_weight: Tensor | None = None,
                 temperature: float = 1.0, softcap: tuple[float, float, float] | None = None) -> Tensor:
    """losses [T] fp32 of the student's logits [T, V] (bf16 or fp32) against a teacher's logits `teacher` [T, K] fp32 of the columns `ids`
    [T, K] (int32 or int64), K <= 512, V <= 2^24, A / temperature <= 80.  With z = softcap(logits) / temperature, softcap(l) = A sigmoid((l + B) / C) for
    softcap = (A, B, C), and q = softmax(z) over all V columns,

        losses = row_weight temperature^2 sum_j p_j (log p_j - log q[ids_j]),    p = softmax(teacher / temperature) over the list,

    or, with teacher_lse [T] (the teacher's log-sum-exp over all its columns at this temperature), p = exp(teacher / temperature -
    teacher_lse) and the rest of the teacher's mass against the rest of the student's as one more term.  Entries whose id is not a
    column (-1 pads a list) count for nothing; a row without entries, or of weight 0, has loss 0 and gradient 0.
    Differentiable in logits only."""
    tensors = (logits, ids, teacher, teacher_lse, row_weight)
    params = (float(temperature), *_softcap(softcap))
    if not is_dynamo_compiling():
        losses = (_binding or _b()).distill_topk(*tensors, *params)
        if losses is not None:
            return losses
    if _plain(*tensors):
        _distill_shapes(*tensors)
        if _direct(*tensors):
            _same_gpu(*tensors)
            if not _nothing_listed(logits, ids):
                return _launched(_b().distill_topk(*_distill_usable(*tensors), *params), "distill_topk")
    return torch.ops.nanogpt.distill_topk(*tensors, *params)[0]


def distill_topk_fwd_bwd(logits: Tensor, ids: Tensor, teacher: Tensor, teacher_lse: Tensor | None = None, row_weight: Tensor | None = None,
                         temperature: float = 1.0, softcap: tuple[float, float, float] | None = None,
                         grad_scale: float = 1.0) -> tuple[Tensor, Tensor]:
    """(losses, grad) of distill_topk, grad = grad_scale * d sum(losses) / d logits in the logits' type: one pass over the logits where a
    row fits a workgroup's registers (53744 columns), two beyond.  Not differentiable itself."""
    tensors = (logits, ids, teacher, teacher_lse, row_weight)
    params = (float(temperature), *_softcap(softcap), float(grad_scale))
    if not is_dynamo_compiling():
        out = (_binding or _b()).distill_fused(*tensors, *params)
        if out is not None:
            return out
    if _plain(*tensors):
        _distill_shapes(*tensors)
        if _direct(*tensors):
            _same_gpu(*tensors)
            if not _nothing_listed(logits, ids):
                return _launched(_b().distill_fused(*_distill_usable(*tensors), *params), "distill_topk_fwd_bwd")
    return torch.ops.nanogpt.distill_topk_fwd_bwd(*tensors, *params)

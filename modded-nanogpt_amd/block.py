"""Operators around the attention and MLP of a block, and the loss against a teacher:

    linear_act             out = residual + act(x @ w.T + bias), differentiable in all four
    qk_norm_rope           per-head rms norm of queries and keys and the position rotation in one pass, differentiable
    distill_topk           distillation loss against a teacher's top logits, differentiable in the student's logits
    distill_topk_fwd_bwd   the same loss and its gradient at once, reading the logits once

The functions launch the kernels of libngpt_fp8.so directly; under `torch.compile` or with fake tensors they go through the registered
operators nanogpt::linear_act, qk_norm_rope, distill_topk (and their *_backward), which do the same.  All tensors of a call live
on one GPU; work is enqueued on that GPU's current stream.  There is no CPU implementation.
"""
from __future__ import annotations

import ctypes
import functools

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import _p, _workspace

# the current stream's handle without the Stream object around it
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)       # (a tensor on a GPU is there: CUDA is initialised)

ACTIVATIONS = {"none": 0, "relu2": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
RMS_EPS = 1.1920928955078125e-07          # machine epsilon of fp32, what the other norms of this package add
_DTYPES = {torch.bfloat16: _lib.DT_BF16, torch.float32: _lib.DT_F32}


def _same_gpu(first: Tensor, *others: Tensor | None) -> int:
    """Index of the GPU that holds all of them."""
    index = first.get_device()
    if index < 0:
        raise RuntimeError("nanogpt operators run on the GPU only (got a CPU tensor); there is no CPU fallback")
    for t in others:
        if t is not None and t.get_device() != index:
            if not t.is_cuda:
                raise RuntimeError("nanogpt operators run on the GPU only (got a CPU tensor); there is no CPU fallback")
            raise AssertionError(f"tensors on {first.device} and {t.device}")
    return index


_entry_points: dict = {}


def _launch(index: int, what: str, *args) -> None:
    """Calls an entry point on GPU `index` and its current stream."""
    fn = _entry_points.get(what)
    if fn is None:
        fn = _entry_points[what] = getattr(_lib.load(), what)
    if index == _current_device():
        code = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            code = fn(*args, _raw_stream(index))
    if code:
        _lib.check(code, what)


def _plain(*tensors: Tensor | None) -> bool:
    """Ordinary tensors outside of a trace: the kernels can be launched here."""
    for t in tensors:
        if t is not None and type(t) is not Tensor and type(t) is not torch.nn.Parameter:
            return False
    return not torch.compiler.is_compiling()


def _needs_grad(*tensors: Tensor | None) -> bool:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


# ------------------------------------------------------------------------------------------------
# linear_act

def _linear_shapes(x: Tensor, w: Tensor, bias: Tensor | None, residual: Tensor | None, activation: str) -> int:
    act = ACTIVATIONS.get(activation)
    assert act is not None, f"activation {activation!r}: one of {', '.join(ACTIVATIONS)}"
    xs, ws = x.shape, w.shape
    assert len(ws) == 2 and len(xs) >= 1 and xs[-1] == ws[1], f"x {tuple(xs)} and w {tuple(ws)}: x is [..., K], w [N, K]"
    bf16 = torch.bfloat16
    assert x.dtype == bf16 and w.dtype == bf16, f"linear_act takes bfloat16, got {x.dtype} and {w.dtype}"
    if bias is not None:
        assert bias.shape == ws[:1], f"bias {tuple(bias.shape)}: one value per row of w"
        assert bias.dtype == bf16, f"linear_act takes bfloat16, got a bias of {bias.dtype}"
    if residual is not None:
        assert residual.shape == xs[:-1] + ws[:1], f"residual {tuple(residual.shape)}: the shape of the result"
        assert residual.dtype == bf16, f"linear_act takes bfloat16, got a residual of {residual.dtype}"
    return act


def _ld(t: Tensor) -> int:
    """Row stride of a matrix; that of a single row says nothing."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _matrix(t: Tensor) -> Tensor:
    """[..., K] as a matrix whose rows are contiguous and do not overlap: a view where there is one."""
    if t.ndim != 2:
        t = t.reshape(-1, t.shape[-1])
    if t.is_contiguous():
        return t
    return t if (t.stride(1) == 1 or t.shape[1] == 1) and _ld(t) >= t.shape[1] else t.contiguous()


def _linear_fwd(x: Tensor, w: Tensor, bias: Tensor | None, residual: Tensor | None, activation: str, keep_pre: bool) -> tuple[Tensor, Tensor | None]:
    act = _linear_shapes(x, w, bias, residual, activation)
    assert act or not keep_pre, "keep_pre: without an activation the backward needs no pre-activation"
    gpu = _same_gpu(x, w, bias, residual)
    N, K = w.shape
    out = x.new_empty(x.shape[:-1] + (N,))
    pre = torch.empty_like(out) if keep_pre else None
    if out.numel() == 0:
        return out, pre
    if K == 0:
        raise RuntimeError("linear_act: contraction of length 0")
    xr, wr = _matrix(x), _matrix(w)
    if bias is not None and (bias.stride(0) != 1 or bias.data_ptr() % 16):
        bias = bias.clone(memory_format=torch.contiguous_format)
    res = None if residual is None else _matrix(residual)
    _launch(gpu, "ngpt_linear_act_fwd", xr.data_ptr(), _ld(xr), wr.data_ptr(), _ld(wr), None if bias is None else bias.data_ptr(),
            None if res is None else res.data_ptr(), 0 if res is None else _ld(res), xr.shape[0], N, K, act, out.data_ptr(),
            None if pre is None else pre.data_ptr())
    return out, pre


def _linear_bwd(dout: Tensor, x: Tensor, w: Tensor, pre: Tensor | None, activation: str, need_dx: bool, need_dw: bool,
                need_dbias: bool) -> tuple[Tensor | None, Tensor | None, Tensor | None]:
    act = ACTIVATIONS[activation]
    assert dout.shape == (*x.shape[:-1], w.shape[0]) and dout.dtype == torch.bfloat16
    assert act == 0 or pre is not None, "the backward of an activation needs the forward's pre-activation"
    gpu = _same_gpu(x, w, dout, pre)
    N, K = w.shape
    new = lambda *shape: torch.empty(shape, dtype=torch.bfloat16, device=x.device)
    dx = new(*x.shape) if need_dx else None
    dw = new(N, K) if need_dw else None
    db = new(N) if need_dbias else None
    if not (need_dx or need_dw or need_dbias):
        return dx, dw, db
    M = dout.numel() // N if N else 0
    if M == 0 or N == 0 or K == 0:
        for t in (dx, dw, db):
            if t is not None:
                t.zero_()
        return dx, dw, db
    dout = dout.contiguous()
    pre = None if pre is None else pre.contiguous()
    xr, wr = _matrix(x), _matrix(w)
    ws = _workspace(_lib.load().ngpt_linear_act_bwd_workspace_bytes(M, N, K), x.device)
    _launch(gpu, "ngpt_linear_act_bwd", _p(dout), _p(pre), _p(xr), _ld(xr), _p(wr), _ld(wr), M, N, K, act, _p(dx), _p(dw), _p(db), _p(ws), ws.numel())
    return dx, dw, db


@torch.library.custom_op("nanogpt::linear_act", mutates_args=())
def linear_act_op(x: Tensor, w: Tensor, bias: Tensor | None, residual: Tensor | None, activation: str, keep_pre: bool) -> tuple[Tensor, Tensor]:
    """-> (out, pre): pre [.., N] = x @ w.T + bias if keep_pre, else empty."""
    out, pre = _linear_fwd(x, w, bias, residual, activation, keep_pre)
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
    return tuple(dout.new_empty(0) if t is None else t for t in _linear_bwd(dout, x, w, pre, activation, need_dx, need_dw, need_dbias))


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
    dx, dw, db = torch.ops.nanogpt.linear_act_backward(dout, x, w, pre, ctx.activation, need[0], need[1], need[2])
    return (dx if need[0] else None, dw if need[1] else None, db if need[2] else None, dout if need[3] else None, None, None)


linear_act_op.register_autograd(_linear_backward, setup_context=_linear_setup)


class LinearActFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, residual, activation):
        keep = activation != "none" and any(ctx.needs_input_grad[:3])
        out, pre = _linear_fwd(x, w, bias, residual, activation, keep)
        ctx.save_for_backward(x, w, pre)
        ctx.activation = activation
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        x, w, pre = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dw, db = _linear_bwd(dout, x, w, pre, ctx.activation, need[0], need[1], need[2])
        return dx, dw, db, dout if need[3] else None, None


def linear_act(x: Tensor, w: Tensor, bias: Tensor | None = None, residual: Tensor | None = None, activation: str = "none") -> Tensor:
    """residual + act(x @ w.T + bias) for bf16 x [..., K], w [N, K], bias [N], residual [..., N]; fp32 accumulation, bias, activation
    and residual applied to the fp32 sums, one rounding.  `activation`: "none", "relu2" (max(z, 0)^2), "gelu", "gelu_tanh", "silu".
    Any sizes; rows of x, w and residual may be strided.  Differentiable in x, w, bias and residual; an activation's backward keeps
    the bf16 pre-activation."""
    if not _plain(x, w, bias, residual):
        keep = activation != "none" and _needs_grad(x, w, bias)
        return torch.ops.nanogpt.linear_act(x, w, bias, residual, activation, keep)[0]
    if _needs_grad(x, w, bias, residual):
        return LinearActFunction.apply(x, w, bias, residual, activation)
    return _linear_fwd(x, w, bias, residual, activation, False)[0]


# ------------------------------------------------------------------------------------------------
# qk_norm_rope

def _rope_shapes(q: Tensor, k: Tensor, cos: Tensor, sin: Tensor, positions: Tensor | None, q_weight: Tensor | None, k_weight: Tensor | None) -> None:
    qs, ks, dtype = q.shape, k.shape, q.dtype
    assert len(qs) in (3, 4) and len(ks) == len(qs) and qs[:-2] == ks[:-2] and qs[-1] == ks[-1], (
        f"q {tuple(qs)} and k {tuple(ks)}: [T, H, D] or [B, T, H, D] with the same tokens and head size")
    assert dtype in _DTYPES and k.dtype == dtype, f"q {dtype} and k {k.dtype}: both bfloat16 or both float32"
    assert cos.ndim == 2 and cos.shape == sin.shape and cos.dtype == sin.dtype and cos.dtype in _DTYPES, (
        "cos and sin: [positions, rotated / 2], both bfloat16 or both float32")
    if positions is not None:
        assert positions.dtype in (torch.int32, torch.int64) and (positions.shape == qs[:-2] or positions.shape == qs[-3:-2]), (
            f"positions: int32 or int64, of shape {tuple(qs[:-2])} or {tuple(qs[-3:-2])}")
    for w in (q_weight, k_weight):
        assert w is None or (w.shape == qs[-1:] and w.dtype == dtype), "weights: one value per head element, in the heads' type"


def _heads(t: Tensor) -> Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


@functools.lru_cache(maxsize=1024)
def _strides(*s: int):
    """The strides as a C array (read only, so one per value will do)."""
    return (ctypes.c_int64 * len(s))(*s)


def _head_strides(t: Tensor):
    s = t.stride()
    return _strides(0 if t.ndim == 3 else s[0], s[-3], s[-2])


def _rope_common(q, k, cos, sin, positions, q_weight, k_weight, eps, interleaved):
    """(tensors to keep alive, leading arguments shared by both directions)"""
    B = q.shape[0] if q.ndim == 4 else 1
    T, Hq, D = q.shape[-3:]
    cos, sin = cos.contiguous(), sin.contiguous()
    pos_strides = None
    if positions is not None:
        s = positions.stride()
        pos_strides = _strides(s[0] if positions.ndim == 2 else 0, s[-1])
    q_weight = None if q_weight is None else q_weight.contiguous()
    k_weight = None if k_weight is None else k_weight.contiguous()
    args = (_DTYPES[q.dtype], B, T, Hq, k.shape[-2], D, 2 * cos.shape[1], _p(cos), _p(sin), _DTYPES[cos.dtype], cos.shape[0],
            _p(positions), int(positions is not None and positions.dtype == torch.int64), pos_strides, _p(q_weight), _p(k_weight),
            eps, int(interleaved))
    return (cos, sin, q_weight, k_weight), args


def _rope_fwd(q, k, cos, sin, positions, q_weight, k_weight, eps, interleaved) -> tuple[Tensor, Tensor]:
    _rope_shapes(q, k, cos, sin, positions, q_weight, k_weight)
    gpu = _same_gpu(q, k, cos, sin, positions, q_weight, k_weight)
    q_out, k_out = q.new_empty(q.shape), k.new_empty(k.shape)
    if q.numel() == 0 and k.numel() == 0:
        return q_out, k_out
    q, k = _heads(q), _heads(k)
    keep, args = _rope_common(q, k, cos, sin, positions, q_weight, k_weight, eps, interleaved)
    _launch(gpu, "ngpt_qk_norm_rope", _p(q), _head_strides(q), _p(k), _head_strides(k), *args, _p(q_out), _p(k_out))
    return q_out, k_out


def _rope_bwd(dq_out, dk_out, q, k, cos, sin, positions, q_weight, k_weight, eps, interleaved, need_dqw, need_dkw):
    """-> dq, dk, dq_weight or None, dk_weight or None"""
    gpu = _same_gpu(q, k, cos, sin, positions, q_weight, k_weight, dq_out, dk_out)
    assert dq_out.shape == q.shape and dk_out.shape == k.shape and dq_out.dtype == q.dtype and dk_out.dtype == k.dtype
    dq, dk = q.new_empty(q.shape), k.new_empty(k.shape)
    dqw = torch.empty_like(q_weight, memory_format=torch.contiguous_format) if need_dqw else None
    dkw = torch.empty_like(k_weight, memory_format=torch.contiguous_format) if need_dkw else None
    if q.numel() == 0 and k.numel() == 0:
        for t in (dqw, dkw):
            if t is not None:
                t.zero_()
        return dq, dk, dqw, dkw
    q, k, dq_out, dk_out = _heads(q), _heads(k), _heads(dq_out), _heads(dk_out)
    keep, args = _rope_common(q, k, cos, sin, positions, q_weight, k_weight, eps, interleaved)
    nws = _lib.load().ngpt_qk_norm_rope_bwd_workspace_bytes(q.shape[-1]) if need_dqw or need_dkw else 0
    ws = _workspace(nws, q.device) if nws else None
    _launch(gpu, "ngpt_qk_norm_rope_bwd", _p(dq_out), _head_strides(dq_out), _p(dk_out), _head_strides(dk_out), _p(q), _head_strides(q), _p(k),
            _head_strides(k), *args, _p(dq), _p(dk), _p(dqw), _p(dkw), _p(ws), nws)
    return dq, dk, dqw, dkw


@torch.library.custom_op("nanogpt::qk_norm_rope", mutates_args=())
def qk_norm_rope_op(q: Tensor, k: Tensor, cos: Tensor, sin: Tensor, positions: Tensor | None, q_weight: Tensor | None, k_weight: Tensor | None,
                    eps: float, interleaved: bool) -> tuple[Tensor, Tensor]:
    return _rope_fwd(q, k, cos, sin, positions, q_weight, k_weight, eps, interleaved)


@qk_norm_rope_op.register_fake
def _(q, k, cos, sin, positions, q_weight, k_weight, eps, interleaved):
    _rope_shapes(q, k, cos, sin, positions, q_weight, k_weight)
    return q.new_empty(q.shape), k.new_empty(k.shape)


@torch.library.custom_op("nanogpt::qk_norm_rope_backward", mutates_args=())
def qk_norm_rope_backward_op(dq_out: Tensor, dk_out: Tensor, q: Tensor, k: Tensor, cos: Tensor, sin: Tensor, positions: Tensor | None,
                             q_weight: Tensor | None, k_weight: Tensor | None, eps: float, interleaved: bool, need_dq_weight: bool,
                             need_dk_weight: bool) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """-> (dq, dk, dq_weight, dk_weight), the weights' empty where not wanted."""
    r = _rope_bwd(dq_out, dk_out, q, k, cos, sin, positions, q_weight, k_weight, eps, interleaved, need_dq_weight, need_dk_weight)
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


class QKNormRopeFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, cos, sin, positions, q_weight, k_weight, eps, interleaved):
        ctx.save_for_backward(q, k, cos, sin, positions, q_weight, k_weight)
        ctx.params = eps, interleaved
        return _rope_fwd(q, k, cos, sin, positions, q_weight, k_weight, eps, interleaved)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq_out, dk_out):
        need = ctx.needs_input_grad
        dq, dk, dqw, dkw = _rope_bwd(dq_out, dk_out, *ctx.saved_tensors, *ctx.params, need[5], need[6])
        return dq, dk, None, None, None, dqw, dkw, None, None


def qk_norm_rope(q: Tensor, k: Tensor, cos: Tensor, sin: Tensor, positions: Tensor | None = None, q_weight: Tensor | None = None,
                 k_weight: Tensor | None = None, eps: float | None = None, interleaved: bool = False) -> tuple[Tensor, Tensor]:
    """(rot(norm(q)), rot(norm(k))) for q [T, Hq, D] or [B, T, Hq, D] and k likewise with its own number of heads, bf16 or fp32; views of
    a packed projection are read in place.  norm is over each head's D values (eps None: the machine epsilon of fp32), times the weight
    [D] if given.  The first R values of a head are rotated, R / 2 = cos.shape[1]: pairs (i, i + R / 2), or (2 i, 2 i + 1) if
    interleaved, (a, b) -> (a cos - b sin, b cos + a sin) with row `positions[token]` of cos and sin (None: the token's index in its
    sequence).  A position outside the tables makes that token's heads NaN.  Differentiable in q, k and the weights."""
    eps = RMS_EPS if eps is None else float(eps)
    args = (q, k, cos, sin, positions, q_weight, k_weight, eps, interleaved)
    if not _plain(*args[:7]):
        return torch.ops.nanogpt.qk_norm_rope(*args)
    if _needs_grad(q, k, q_weight, k_weight):
        return QKNormRopeFunction.apply(*args)
    return _rope_fwd(*args)


# ------------------------------------------------------------------------------------------------
# distill_topk

def _distill_shapes(logits, ids, teacher, teacher_lse, row_weight) -> None:
    assert logits.ndim == 2 and logits.dtype in _DTYPES, f"logits {tuple(logits.shape)} {logits.dtype}: [T, V], bfloat16 or float32"
    T = logits.shape[0]
    assert ids.ndim == 2 and ids.shape[0] == T and ids.dtype in (torch.int32, torch.int64), f"ids {tuple(ids.shape)} {ids.dtype}: [T, K] int32 or int64"
    assert teacher.shape == ids.shape and teacher.dtype == torch.float32, f"teacher {tuple(teacher.shape)} {teacher.dtype}: float32, one logit per id"
    for name, t in (("teacher_lse", teacher_lse), ("row_weight", row_weight)):
        assert t is None or (t.shape == (T,) and t.dtype == torch.float32), f"{name}: [T] float32"


def _distill_args(logits, ids, teacher, teacher_lse, row_weight, temperature, A, B, C):
    _distill_shapes(logits, ids, teacher, teacher_lse, row_weight)
    gpu = _same_gpu(logits, ids, teacher, teacher_lse, row_weight)
    keep = [_matrix(logits)] + [None if t is None else t.contiguous() for t in (ids, teacher, teacher_lse, row_weight)]
    lg, i, t, l, w = keep
    T, V = lg.shape
    return gpu, keep, (_p(lg), _DTYPES[lg.dtype], _ld(lg), _p(i), int(i.dtype == torch.int64), _p(t), _p(l), _p(w), T, V, i.shape[1],
                  temperature, A, B, C)


def _distill_fwd(logits, ids, teacher, teacher_lse, row_weight, temperature, A, B, C, keep_stats: bool) -> tuple[Tensor, Tensor | None]:
    gpu, keep, args = _distill_args(logits, ids, teacher, teacher_lse, row_weight, temperature, A, B, C)
    losses = torch.empty(logits.shape[0], dtype=torch.float32, device=logits.device)
    stats = torch.empty((logits.shape[0], 4), dtype=torch.float32, device=logits.device) if keep_stats else None
    if losses.numel() == 0:
        return losses, stats
    if ids.shape[1] == 0:
        return losses.zero_(), None if stats is None else stats.zero_()
    _launch(gpu, "ngpt_distill_fwd", *args, _p(losses), _p(stats))
    return losses, stats


def _distill_bwd(dlosses, logits, ids, teacher, teacher_lse, row_weight, stats, temperature, A, B, C) -> Tensor:
    assert dlosses.shape == (logits.shape[0],) and dlosses.dtype == torch.float32
    _same_gpu(logits, dlosses, stats)
    gpu, keep, args = _distill_args(logits, ids, teacher, teacher_lse, row_weight, temperature, A, B, C)
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    if grad.numel() == 0:
        return grad
    if ids.shape[1] == 0:
        return grad.zero_()
    _launch(gpu, "ngpt_distill_bwd", *args, _p(stats), _p(dlosses), dlosses.stride(0), _p(grad), _ld(grad))
    return grad


def _distill_fused(logits, ids, teacher, teacher_lse, row_weight, temperature, A, B, C, grad_scale) -> tuple[Tensor, Tensor]:
    lib = _lib.load()
    if logits.numel() == 0 or ids.ndim != 2 or ids.shape[1] == 0 or logits.shape[1] > lib.ngpt_distill_fused_max_cols(_DTYPES.get(logits.dtype, 0)):
        # a row longer than a workgroup's registers: two passes over the logits
        losses, stats = _distill_fwd(logits, ids, teacher, teacher_lse, row_weight, temperature, A, B, C, True)
        scale = torch.full((1,), grad_scale, dtype=torch.float32, device=logits.device).expand(logits.shape[0])
        return losses, _distill_bwd(scale, logits, ids, teacher, teacher_lse, row_weight, stats, temperature, A, B, C)
    gpu, keep, args = _distill_args(logits, ids, teacher, teacher_lse, row_weight, temperature, A, B, C)
    losses = torch.empty(logits.shape[0], dtype=torch.float32, device=logits.device)
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    _launch(gpu, "ngpt_distill_fwd_bwd", *args, grad_scale, _p(losses), _p(grad), _ld(grad))
    return losses, grad


@torch.library.custom_op("nanogpt::distill_topk", mutates_args=())
def distill_topk_op(logits: Tensor, ids: Tensor, teacher: Tensor, teacher_lse: Tensor | None, row_weight: Tensor | None, temperature: float,
                    A: float, B: float, C: float) -> tuple[Tensor, Tensor]:
    """-> (losses [T], stats [T, 4] for the backward).  C = 0: no softcap."""
    return _distill_fwd(logits, ids, teacher, teacher_lse, row_weight, temperature, A, B, C, True)


@distill_topk_op.register_fake
def _(logits, ids, teacher, teacher_lse, row_weight, temperature, A, B, C):
    _distill_shapes(logits, ids, teacher, teacher_lse, row_weight)
    T = logits.shape[0]
    return logits.new_empty(T, dtype=torch.float32), logits.new_empty((T, 4), dtype=torch.float32)


@torch.library.custom_op("nanogpt::distill_topk_backward", mutates_args=())
def distill_topk_backward_op(dlosses: Tensor, logits: Tensor, ids: Tensor, teacher: Tensor, teacher_lse: Tensor | None, row_weight: Tensor | None,
                             stats: Tensor, temperature: float, A: float, B: float, C: float) -> Tensor:
    return _distill_bwd(dlosses, logits, ids, teacher, teacher_lse, row_weight, stats, temperature, A, B, C)


@distill_topk_backward_op.register_fake
def _(dlosses, logits, ids, teacher, teacher_lse, row_weight, stats, temperature, A, B, C):
    return logits.new_empty(logits.shape)


@torch.library.custom_op("nanogpt::distill_topk_fwd_bwd", mutates_args=())
def distill_topk_fwd_bwd_op(logits: Tensor, ids: Tensor, teacher: Tensor, teacher_lse: Tensor | None, row_weight: Tensor | None, temperature: float,
                            A: float, B: float, C: float, grad_scale: float) -> tuple[Tensor, Tensor]:
    return _distill_fused(logits, ids, teacher, teacher_lse, row_weight, temperature, A, B, C, grad_scale)


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


class DistillTopKFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, teacher, teacher_lse, row_weight, *params):
        losses, stats = _distill_fwd(logits, ids, teacher, teacher_lse, row_weight, *params, True)
        ctx.save_for_backward(logits, ids, teacher, teacher_lse, row_weight, stats)
        ctx.params = params
        return losses

    @staticmethod
    @once_differentiable
    def backward(ctx, dlosses):
        logits, ids, teacher, teacher_lse, row_weight, stats = ctx.saved_tensors
        return _distill_bwd(dlosses, logits, ids, teacher, teacher_lse, row_weight, stats, *ctx.params), *([None] * 8)


def _softcap(softcap) -> tuple[float, float, float]:
    if softcap is None:
        return 0.0, 0.0, 0.0
    A, B, C = (float(v) for v in softcap)
    assert A > 0 and C > 0, f"softcap {softcap}: A sigmoid((l + B) / C) needs A, C > 0"
    return A, B, C


def distill_topk(logits: Tensor, ids: Tensor, teacher: Tensor, teacher_lse: Tensor | None = None, row_weight: Tensor | None = None,
                 temperature: float = 1.0, softcap: tuple[float, float, float] | None = None) -> Tensor:
    """losses [T] fp32 of the student's logits [T, V] (bf16 or fp32) against a teacher's logits `teacher` [T, K] fp32 of the columns `ids`
    [T, K] (int32 or int64), K <= 512.  With z = softcap(logits) / temperature, softcap(l) = A sigmoid((l + B) / C) for
    softcap = (A, B, C), and q = softmax(z) over all V columns,

        losses = row_weight temperature^2 sum_j p_j (log p_j - log q[ids_j]),    p = softmax(teacher / temperature) over the list,

    or, with teacher_lse [T] (the teacher's log-sum-exp over all its columns at this temperature), p = exp(teacher / temperature -
    teacher_lse) and the rest of the teacher's mass against the rest of the student's as one more term.  Entries whose id is not a
    column (-1 pads a list) count for nothing; a row without entries, or of weight 0, has loss 0 and gradient 0.
    Differentiable in logits only."""
    args = (logits, ids, teacher, teacher_lse, row_weight, float(temperature), *_softcap(softcap))
    if not _plain(*args[:5]):
        return torch.ops.nanogpt.distill_topk(*args)[0]
    if _needs_grad(logits):
        return DistillTopKFunction.apply(*args)
    return _distill_fwd(*args, False)[0]


def distill_topk_fwd_bwd(logits: Tensor, ids: Tensor, teacher: Tensor, teacher_lse: Tensor | None = None, row_weight: Tensor | None = None,
                         temperature: float = 1.0, softcap: tuple[float, float, float] | None = None,
                         grad_scale: float = 1.0) -> tuple[Tensor, Tensor]:
    """(losses, grad) of distill_topk, grad = grad_scale * d sum(losses) / d logits in the logits' type: one pass over the logits where a
    row fits a workgroup's registers (57328 columns), two beyond."""
    args = (logits, ids, teacher, teacher_lse, row_weight, float(temperature), *_softcap(softcap), float(grad_scale))
    if not _plain(*args[:5]):
        return torch.ops.nanogpt.distill_topk_fwd_bwd(*args)
    return _distill_fused(*(t.detach() if isinstance(t, Tensor) else t for t in args))

"""Calls of linear_act, qk_norm_rope and distill_topk beside the sizes of test_gpu_block.py: layouts, modes of torch, values at the edge of the
formulas.  Bounds are that file's, which count roundings."""
import pytest
import torch

from test_gpu_block import BF, D, F32, act64, check_distill, check_linear, close, rnd, teacher_rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def amd():
    import modded_nanogpt_amd
    modded_nanogpt_amd._lib.load()
    return modded_nanogpt_amd


def single_rows(seed, n, dtype=BF):
    """[1, n] whose values are not side by side: a column, every second value, the last of a time axis, one value throughout"""
    return [rnd(seed, n, 24, dtype=dtype).t()[5:6], rnd(seed + 1, 1, 2 * n, dtype=dtype)[:, ::2], rnd(seed + 2, 1, n, 7, dtype=dtype).transpose(1, 2)[:, -1],
            rnd(seed + 3, 1, 1, dtype=dtype).expand(1, n)]


@pytest.mark.parametrize("N,K", [(40, 72), (264, 1024)])
def test_linear_act_single_rows_of_any_stride(amd, N, K):
    w, b, dout = rnd(1, N, K, scale=K ** -0.5), rnd(2, N), rnd(3, 1, N)
    for i, (x, r) in enumerate(zip(single_rows(10, K), single_rows(20, N))):
        check_linear(amd, x, w, b, r, "silu", dout, ("x, residual", i))
        assert torch.equal(amd.linear_act(x[0], w, b, r[0]), amd.linear_act(x.contiguous(), w, b, r.contiguous())[0])
    for i, w1 in enumerate(single_rows(30, K)):              # a weight of one row, for one row and for many
        for M in (1, 50):
            check_linear(amd, rnd(4, M, K), w1, rnd(5, 1), rnd(6, M, 1), "gelu", rnd(7, M, 1), ("w", i, M))
    for i, d in enumerate(single_rows(40, N)):               # an incoming gradient of one row
        check_linear(amd, rnd(8, 1, K), w, b, None, "none", d, ("dout", i))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_distill_a_single_row_of_any_stride(amd, dtype):
    V, K = 1003, 9
    for tail in (False, True):
        ids, teacher, lse = teacher_rows(1, 1, V, K, 1.0 if tail else None)
        for i, logits in enumerate(single_rows(50, V, dtype)):
            check_distill(amd, logits, ids, teacher, lse, None, 1.0, None, (i, tail))


def capped64(logits, ids, teacher, lse, cap, tau, up):
    """losses and gradient with their bounds, for lists of distinct columns; cap[0] / tau and |logits| are moderate"""
    A, B, C = cap
    l = logits.double()
    s = torch.sigmoid((l + B) / C)
    z = A * s / tau
    logq = z - torch.logsumexp(z, 1, keepdim=True)
    q = logq.exp()
    t = teacher.double() / tau
    logp = t - (torch.logsumexp(t, 1) if lse is None else lse.double())[:, None]
    p = logp.exp()
    loss = (p * (logp - logq.gather(1, ids))).sum(1)
    sum_p = p.sum(1)
    rest, ratio, log_others = torch.zeros_like(sum_p), torch.zeros_like(sum_p), torch.zeros_like(sum_p)
    if lse is not None and ids.shape[1] < logits.shape[1]:
        rest = (1 - sum_p).clamp_min(0)
        log_others = logq.scatter(1, ids, -torch.inf).logsumexp(1)
        loss = loss + rest * (rest.log() - log_others)
        ratio = rest / log_others.exp()
    listed = torch.zeros_like(q).scatter(1, ids, 1.0)
    pv = torch.zeros_like(q).scatter(1, ids, p)
    f = (sum_p + rest)[:, None] - ratio[:, None] * (1 - listed)
    slope = A / C * s * (1 - s)
    base = (tau * up.double())[:, None]
    # Roundings E of a term: its exponent of |k1 l + k0| < 6 to 12 E, sigma then to 13 E, times A / tau, and the exponential's own 2 E.  Sums: 56
    # values a thread, 24 levels of a tree; places of -inf that are subtracted again (at most 7 beside the row, or the listed columns, each the
    # smallest term there is) weigh 8 times as much.  The loss takes each sum twice and the listed columns' exponents once more.
    E = 2.0 ** -24
    rel = (26 * A / tau + 160) * E
    size = 1 + (p * logp.abs()).sum(1) + (p * (z.gather(1, ids) - z.gather(1, ids).max(1, keepdim=True)[0]).abs()).sum(1) + rest * log_others.abs()
    lbound = tau * tau * (rel * (sum_p + 2 * rest) + 8 * E * size)
    grad = base * (q * f - pv) * slope
    fabs = (sum_p + rest + ratio)[:, None]
    gbound = base.abs() * ((q * fabs * 3 * rel + pv * 8 * E) * slope + (q * fabs + pv) * 16 * E * A / C * s) + (2.0 ** -8 if logits.dtype == BF else E) * grad.abs()
    return (tau * tau * loss, lbound), (grad, gbound)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("tail", [False, True], ids=["list", "rest"])
@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 57, 100, 256, 1003, 16401])
def test_distill_with_a_small_cap(amd, dtype, tail, V):
    """the cap's smallest term is no longer negligible: what is read outside a row, or of listed columns, must not reach its sum"""
    for T in (3, 600):                                   # no more rows than compute units, and more
        for i, (A, tau) in enumerate(((0.5, 1.0), (1.0, 1.0), (4.0, 2.0), (5.0, 1.0))):
            cap = (A, 5.0, 7.5)
            for K in {1, min(max(1, V // 3), 512), min(V - 1, 512) or 1}:
                ids, teacher, lse = teacher_rows(V + i, 8, V, K, tau if tail else None)
                rows = lambda t: None if t is None else t.repeat(T // 8 + 1, *[1] * (t.ndim - 1))[:T].contiguous()
                logits = rows(rnd(V + i + 1, 8, V, dtype=dtype, scale=3.0))
                ids, teacher, lse = rows(ids), rows(teacher), rows(lse)
                up = torch.rand(T, generator=torch.Generator().manual_seed(i)).to(D) + 0.5
                what = (V, T, A, tau, K)
                loss, grad = capped64(logits, ids, teacher, lse, cap, tau, up)
                kw = dict(teacher_lse=lse, temperature=tau, softcap=cap)
                leaf = logits.clone().requires_grad_()
                got = amd.distill_topk(leaf, ids, teacher, **kw)
                close(got.detach(), *loss, (what, "loss"))
                close(torch.autograd.grad(got, [leaf], up)[0], *grad, (what, "grad"))
                fused = amd.distill_topk_fwd_bwd(logits, ids, teacher, grad_scale=0.25, **kw)
                close(fused[0], *loss, (what, "fused loss"))
                close(fused[1], *capped64(logits, ids, teacher, lse, cap, tau, torch.full((T,), 0.25, device=D))[1], (what, "fused grad"))


def test_distill_with_a_small_cap_on_rows_that_start_anywhere(amd):
    T, V, K = 5, 39, 3
    for dtype in (BF, F32):
        big = rnd(2, T, V + 29, dtype=dtype, scale=3.0)
        for tail in (False, True):
            ids, teacher, lse = teacher_rows(1, T, V, K, 1.0 if tail else None)
            for off in range(9):
                logits = big[:, off:off + V]
                up = torch.full((T,), 0.25, device=D)
                loss, grad = capped64(logits, ids, teacher, lse, (1.0, 5.0, 7.5), 1.0, up)
                got = amd.distill_topk_fwd_bwd(logits, ids, teacher, teacher_lse=lse, softcap=(1.0, 5.0, 7.5), grad_scale=0.25)
                close(got[0], *loss, (off, "loss"))
                close(got[1], *grad, (off, "grad"))


def every_call(amd):
    """(name, function, its tensors) of the four functions with every tensor that they take"""
    M, K, N, V, C = 12, 64, 72, 300, 5
    from test_gpu_block import tables
    cos, sin = tables(M, 24)
    ids, teacher, lse = teacher_rows(5, M, V, C, 1.0)
    weight = torch.rand(M, generator=torch.Generator().manual_seed(1)).to(D)
    yield "linear_act", lambda x, w, b, r: amd.linear_act(x, w, b, r, "gelu"), [rnd(1, M, K), rnd(2, N, K, scale=0.1), rnd(3, N), rnd(4, M, N)]
    yield "qk_norm_rope", lambda q, k, c, s, g, h: amd.qk_norm_rope(q, k, c, s, None, g, h), [rnd(6, M, 4, 24), rnd(7, M, 2, 24), cos, sin, rnd(8, 24), rnd(9, 24)]
    yield "distill_topk", lambda l, t, e, w: amd.distill_topk(l, ids, t, e, w), [rnd(10, M, V), teacher, lse, weight]
    yield "distill_topk_fwd_bwd", lambda l, t, e, w: amd.distill_topk_fwd_bwd(l, ids, t, e, w), [rnd(10, M, V), teacher, lse, weight]


def test_forward_mode_is_refused_for_every_tensor_in_every_mode(amd):
    from torch.autograd import forward_ad
    for name, f, tensors in every_call(amd):
        for i, t in enumerate(tensors):
            for spread in (False, True):                       # in usable form, and one that is copied first
                for mode in (torch.no_grad(), torch.enable_grad()):
                    with forward_ad.dual_level(), mode:
                        if spread:
                            base = torch.empty(*t.shape, 2, dtype=t.dtype, device=D)
                            dual = forward_ad.make_dual(base.copy_(t.unsqueeze(-1)), torch.ones_like(base))[..., 0]
                        else:
                            dual = forward_ad.make_dual(t, torch.ones_like(t))
                        args = [dual if j == i else u for j, u in enumerate(tensors)]
                        with pytest.raises(RuntimeError, match="forward-mode"):
                            f(*args)


def test_forward_mode_is_refused_by_the_registered_operators(amd):
    from torch.autograd import forward_ad
    ops = torch.ops.nanogpt
    (_, _, lin), (_, _, rope), (_, _, dist), _ = every_call(amd)
    ids = teacher_rows(5, 12, 300, 5)[0]
    calls = [(lambda x: ops.linear_act(x, lin[1], None, None, "none", False), lin[0]),
             (lambda q: ops.qk_norm_rope(q, *rope[1:4], None, None, None, 1e-6, False), rope[0]),
             (lambda l: ops.distill_topk(l, ids, dist[1], None, None, 1.0, 0.0, 0.0, 0.0), dist[0]),
             (lambda l: ops.distill_topk_fwd_bwd(l, ids, dist[1], None, None, 1.0, 0.0, 0.0, 0.0, 1.0), dist[0])]
    for f, t in calls:
        with forward_ad.dual_level(), torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            f(forward_ad.make_dual(t, torch.ones_like(t)))


def test_a_forward_mode_incoming_gradient_is_refused(amd):
    from torch.autograd import forward_ad
    for name, f, tensors in every_call(amd):
        if name == "distill_topk_fwd_bwd":
            continue
        leaf = tensors[0].clone().requires_grad_()
        out = f(leaf, *tensors[1:])
        out = out if torch.is_tensor(out) else out[0]
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(out, [leaf], forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out)))


def test_linear_act_gradient_of_the_residual_alone(amd):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Pass(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    x, w, b, dout = rnd(1, 9, 64), rnd(2, 24, 64), rnd(3, 24), rnd(4, 9, 24)
    for act in ("none", "gelu"):
        r = rnd(5, 9, 24).requires_grad_()
        f = lambda r: amd.linear_act(x, w, b, r, act)
        (eager,) = torch.autograd.grad(f(r), [r], dout)
        with Pass():
            (mode,) = torch.autograd.grad(f(r), [r], dout)
        (traced,) = torch.autograd.grad(torch.compile(f, backend="aot_eager", fullgraph=True, dynamic=False)(r), [r], dout)
        for g in (eager, mode, traced):
            assert torch.equal(g, dout), act


@pytest.mark.parametrize("M,N,K", [(128, 64, 64), (4096, 768, 768), (4032, 768, 760), (1000, 250, 333), (33, 72, 100)])
def test_linear_act_backward_stays_inside_its_workspace(amd, M, N, K):
    """every combination of wanted outputs and layouts with the bytes that the query names, between two marked areas; the same bits as with plenty"""
    import itertools
    lib, stream = amd._lib.load(), torch.cuda.current_stream().cuda_stream
    w, mark, guard = rnd(2, N, K, scale=0.1), 0xA5, 1 << 16
    for act, off_d, off_x in itertools.product((0, 3), (0, 1), (0, 1)):
        dout, x, pre = rnd(3, M * N + 8)[off_d:off_d + M * N], rnd(1, M * K + 8)[off_x:off_x + M * K], rnd(4, M, N) if act else None
        ptr = lambda t: None if t is None else t.data_ptr()

        def call(want, ws, n):
            outs = [torch.empty(*s, dtype=BF, device=D) if k else None for k, s in zip(want, ((M, K), (N, K), (N,)))]
            code = lib.ngpt_linear_act_bwd(ptr(dout), ptr(pre), ptr(x), K, ptr(w), K, M, N, K, act, *map(ptr, outs), ws, n, stream)
            assert code == 0, (code, lib.ngpt_last_error())
            return outs

        most = lib.ngpt_linear_act_bwd_workspace_bytes(M, N, K)
        plenty = torch.empty(most, dtype=torch.uint8, device=D)
        want_all = call((1, 1, 1), plenty.data_ptr(), most)
        for want in itertools.product((0, 1), repeat=3):
            n = lib.ngpt_linear_act_bwd_workspace_bytes_for(ptr(dout), ptr(x), K, M, N, K, act, *want)
            assert n <= most
            area = torch.full((n + 2 * guard,), mark, dtype=torch.uint8, device=D)
            outs = call(want, area.data_ptr() + guard if n else None, n)
            assert (area[:guard] == mark).all() and (area[guard + n:] == mark).all(), (act, off_d, off_x, want)
            for a, b in zip(outs, want_all):
                assert a is None or torch.equal(a, b), (act, off_d, off_x, want)


def test_linear_act_backward_memory(amd):
    """a projection without an activation reads dout and x in place: beside its results it needs w^T and the parts of split tiles"""
    M, N, K = 49152, 768, 768
    x, w, dout = rnd(1, M, K).requires_grad_(), rnd(2, N, K, scale=0.1).requires_grad_(), rnd(3, M, N)
    out = amd.linear_act(x, w)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    dx, dw = torch.autograd.grad(out, [x, w], dout)
    extra = torch.cuda.max_memory_allocated() - before - (M + N) * K * 2
    assert extra < 80 << 20, extra          # 1.2 MB and at most one 256 KiB part a compute unit (64 MiB); dz and a copy of x would be 151 MB


def test_linear_act_rows_far_apart(amd):
    """x, w and residual of more than 2^21 values between rows: copied, like other layouts that cannot be read in place"""
    M, N, K, far = 5, 24, 72, (1 << 21) + 8
    spread = lambda seed, rows, n: torch.zeros(rows, far, dtype=BF, device=D)[:, 3:3 + n].copy_(rnd(seed, rows, n))
    x, w, r = spread(1, M, K), spread(2, N, K), spread(3, M, N)
    for i, (a, b, c) in enumerate(((x, w.contiguous(), None), (x.contiguous(), w, None), (x.contiguous(), w.contiguous(), r), (x, w, r))):
        check_linear(amd, a, b, None, c, "gelu", rnd(4, M, N), i)
    assert torch.equal(torch.ops.nanogpt.linear_act(x, w, None, r, "none", False)[0], amd.linear_act(x.contiguous(), w.contiguous(), None, r.contiguous()))


def test_linear_act_last_position_of_every_sequence(amd):
    """[B, 1, K] out of [B, T, K]: evenly spaced rows, read in place"""
    B, T, N, K = 7, 5, 40, 96
    h, r, w = rnd(1, B, T, K), rnd(2, B, T, N), rnd(3, N, K, scale=0.1)
    x, res = h[:, -1:], r[:, -1:]
    want = amd.linear_act(x.contiguous(), w, None, res.contiguous(), "silu")
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    got = amd.linear_act(x, w, None, res, "silu")
    peak = torch.cuda.max_memory_allocated() - before          # (ahead of the comparison, which allocates)
    assert torch.equal(got, want) and got.shape == (B, 1, N)
    assert peak <= 512 * -(-B * N * 2 // 512)                  # the result, no copies
    check = amd.linear_act(h[:, -1].requires_grad_(), w, None, r[:, -1], "silu")
    assert torch.equal(check, want[:, 0])


def test_lazily_negated_tensors(amd):
    """the imaginary part of a conjugate shares its memory with the number and is negated when read"""
    for name, f, tensors in every_call(amd):
        tensors = [t.contiguous() for t in tensors]
        for i, t in enumerate(tensors):
            lazy = torch._neg_view((-t).contiguous())
            assert lazy.is_neg() and lazy.is_contiguous()
            got, want = f(*[lazy if j == i else u for j, u in enumerate(tensors)]), f(*tensors)
            for a, b in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, tuple) else (want,)):
                assert torch.equal(a, b), (name, i)
        if name == "distill_topk_fwd_bwd":
            continue
        lazy = torch._neg_view((-tensors[0]).contiguous())
        grads = []
        for leaf in (tensors[0].detach().requires_grad_(), lazy.detach().requires_grad_()):
            out = f(leaf, *tensors[1:])
            out = out if torch.is_tensor(out) else out[0]
            dout = rnd(3, *out.shape, dtype=out.dtype)
            grads += [torch.autograd.grad(out, [leaf], d, retain_graph=True)[0] for d in (dout, torch._neg_view(-dout))]
        assert all(torch.equal(g, grads[0]) for g in grads), name
    _, f, tensors = list(every_call(amd))[2]
    leaf = tensors[0].clone().requires_grad_()
    losses = f(leaf, *tensors[1:])
    (g,) = torch.autograd.grad(torch.complex(torch.zeros_like(losses), losses).conj().imag.sum(), [leaf], retain_graph=True)
    assert torch.equal(g, torch.autograd.grad(-losses.sum(), [leaf])[0])


@pytest.mark.parametrize("act", ["none", "relu2", "gelu", "gelu_tanh", "silu"])
def test_activations_and_slopes_at_every_bf16_value(amd, act):
    """the type's lowest value, what masks are made of, among them; a NaN stays one"""
    v = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).to(D).view(BF)
    one, w, z = torch.ones(1, 1, dtype=BF, device=D), v[:, None].contiguous(), v.double()
    y64, s64, _ = act64(z, act)
    for M in (1, 40):                      # both kernels of small sizes
        y = amd.linear_act(one.expand(M, 1), w, None, None, act)[-1]
        bound = 2.0 ** -8 * y64.abs() + 8 * 2.0 ** -24 * z.abs() + 1e-37                  # the store; a few fp32 operations; no denormals
        ok = (y == y64.to(BF)) | ((y.double() - y64).abs() <= bound)
        assert ok[v.isfinite()].all() and y[v.isnan()].isnan().all(), (act, M, v[v.isfinite() & ~ok][:4])
    if act == "none":
        return
    db = torch.ops.nanogpt.linear_act_backward(torch.ones(1, 1 << 16, dtype=BF, device=D), one, w, v[None], act, False, False, True)[2]
    bound = 2.0 ** -8 * s64.abs() + 16 * 2.0 ** -24 * (1 + z.abs().clamp_max(100))        # (beyond 100 a smooth slope is 0 or 1)
    ok = (db == s64.to(BF)) | ((db.double() - s64).abs() <= bound)
    assert ok[v.isfinite()].all() and db[v.isnan()].isnan().all(), (act, v[v.isfinite() & ~ok][:4])

"""linear_act, qk_norm_rope and distill_topk on the GPU against plain formulas in 64 bits.

Tolerances count roundings: a value stored as bf16 is off by at most 2^-8 of itself, an fp32 operation by 2^-24; a sum of n terms by n 2^-24 of the
sum of their magnitudes.  Each reference function returns, beside its values, the bound that follows for the kernel's arithmetic."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
U = {BF: 2.0 ** -8, F32: 2.0 ** -24}
E = 2.0 ** -24
D = "cuda"


@pytest.fixture(scope="module")
def amd():
    import modded_nanogpt_amd
    modded_nanogpt_amd._lib.load()
    return modded_nanogpt_amd


def rnd(seed, *shape, dtype=BF, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g, dtype=F64) * scale).to(dtype).to(D)


def close(got, ref, bound, what):
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    err = (got.double() - ref).abs()
    same = (got.double() == ref) | (got.isnan() & ref.isnan())
    bad = ~same & ~(err <= bound)
    assert not bad.any(), (what, int(bad.sum()), float(err[bad].max()), float((err / bound)[bad].max()), bad.nonzero()[:4].tolist())


# ------------------------------------------------------------------------------------------------ linear_act

def act64(z, act):
    """(value, slope, largest curvature)"""
    if act == "none":
        return z, torch.ones_like(z), 0.0
    if act == "relu2":
        r = z.clamp_min(0)
        return r * r, 2 * r, 2.0
    if act == "gelu":
        cdf, pdf = 0.5 * torch.erfc(-z / math.sqrt(2)), torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        return z * cdf, cdf + z * pdf, 0.8
    if act == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        u = c * (z + 0.044715 * z ** 3)
        t = torch.tanh(u)
        return z * (1 + t) / 2, (1 + t) / 2 + z * (1 - t * t) / 2 * c * (1 + 3 * 0.044715 * z * z), 0.85
    s = torch.sigmoid(z)
    return z * s, s * (1 + z * (1 - s)), 0.5


def linear64(x, w, bias, residual, act, dout=None):
    """values and bounds of out, dx, dw, dbias"""
    x, w = x.double(), w.double()
    b = torch.zeros(w.shape[0], dtype=F64, device=x.device) if bias is None else bias.double()
    r = torch.zeros(x.shape[0], w.shape[0], dtype=F64, device=x.device) if residual is None else residual.double()
    M, K, N = x.shape[0], x.shape[1], w.shape[0]
    z = x @ w.t() + b
    zerr = (K + 2) * E * (x.abs() @ w.abs().t() + b.abs())          # fp32 accumulation and the bias
    y, slope, curv = act64(z, act)
    # the activation: its argument's error, and a few fp32 operations (z times a factor at most 1, the factor to 2^-21)
    yerr = slope.abs() * zerr + curv * zerr ** 2 + 8 * E * (y.abs() + z.abs() * (act not in ("none", "relu2")))
    out = y + r
    res = {"out": (out, U[BF] * out.abs() + (1 + U[BF]) * yerr + 2 * E * (out.abs() + r.abs()))}
    if dout is None:
        return res
    g = dout.double()
    dz = g * slope
    # slope at the stored pre-activation (bf16, of the fp32 sum), then dz in bf16 for the products
    serr = curv * (U[BF] * z.abs() + (1 + U[BF]) * zerr) + (16 * E * (1 + z.abs()) if act != "none" else 0)
    derr = g.abs() * serr
    if act == "none":
        derr = torch.zeros_like(derr)
    pz = derr + (U[BF] * (dz.abs() + derr) if act != "none" else 0)
    dx, dw, db = dz @ w, dz.t() @ x, dz.sum(0)
    mag = dz.abs() + pz
    res["dx"] = (dx, pz @ w.abs() * (1 + U[BF]) + U[BF] * dx.abs() + (N + 66) * E * (mag @ w.abs()))
    res["dw"] = (dw, pz.t() @ x.abs() * (1 + U[BF]) + U[BF] * dw.abs() + (M + 66) * E * (mag.t() @ x.abs()))
    res["dbias"] = (db, (1 + U[BF]) * derr.sum(0) + U[BF] * db.abs() + (M + 2) * E * mag.sum(0))
    return res


def check_linear(amd, x, w, bias, residual, act, dout, what):
    ref = linear64(x, w, bias, residual, act, dout)
    leaves = {n: t.detach().requires_grad_() for n, t in (("x", x), ("w", w), ("bias", bias), ("residual", residual)) if t is not None}
    plain = amd.linear_act(x, w, bias, residual, act)
    out = amd.linear_act(leaves["x"], leaves["w"], leaves.get("bias"), leaves.get("residual"), act)
    assert torch.equal(plain, out)
    close(out, *ref["out"], (what, "out"))
    grads = dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), dout)))
    for n in ("x", "w", "bias"):
        if n in grads:
            close(grads[n], *ref["d" + n], (what, "d" + n))
    if residual is not None:
        assert torch.equal(grads["residual"], dout)


LINEAR_SIZES = [(1, 1, 1), (1, 8, 64), (1, 1024, 768), (2, 3, 5), (3, 129, 64), (5, 4096, 256), (8, 260, 1000), (16, 300, 136), (17, 129, 65), (33, 2304, 768),
                (64, 256, 128), (100, 64, 4096), (128, 512, 72), (255, 257, 100), (300, 72, 1000), (512, 1024, 256), (777, 768, 768), (1030, 300, 776),
                (2048, 2304, 192), (4096, 130, 67)]


@pytest.mark.parametrize("i,M,N,K", [(i, *s) for i, s in enumerate(LINEAR_SIZES)])
def test_linear_act_sizes(amd, i, M, N, K):
    acts = ["none", "relu2", "gelu", "gelu_tanh", "silu"]
    for j, act in enumerate(acts):
        has_bias, has_res = (i + j) % 3 != 0, (i + j) % 2 == 0
        x, w = rnd(100 * i + j, M, K), rnd(100 * i + j + 1, N, K, scale=K ** -0.5)
        check_linear(amd, x, w, rnd(7, N) if has_bias else None, rnd(8, M, N) if has_res else None, act, rnd(9 + j, M, N), (M, N, K, act))


@pytest.mark.parametrize("M,N,K", [(1, 264, 128), (13, 264, 192), (200, 264, 128)])
def test_linear_act_strides_and_leading_dimensions(amd, M, N, K):
    big = rnd(1, M, K + 24)
    w_big = rnd(2, N, K + 40, scale=K ** -0.5)
    res_big = rnd(3, M, N + 13)
    cases = [(big[:, 8:8 + K], w_big[:, 16:16 + K], res_big[:, :N]), (big[:, 3:3 + K], w_big[:, 5:5 + K], res_big[:, 7:7 + N]),
             (rnd(4, K, M).t(), rnd(5, K, N, scale=K ** -0.5).t(), rnd(6, N, M).t()), (rnd(4, 1, K).expand(M, K), w_big[:, :K], rnd(6, N).expand(M, N))]
    for i, (x, w, res) in enumerate(cases):
        bias = rnd(9, N + 3)[3:]
        dout = rnd(10, N).expand(M, N) if i == 3 else rnd(11, M, N + 1)[:, 1:]
        check_linear(amd, x, w, bias, res, "silu", dout, i)
    x3, r3 = rnd(12, 2, M, K), rnd(13, 2, M, N)
    assert torch.equal(amd.linear_act(x3, w_big[:, :K], None, r3, "gelu").view(-1, N),
                       amd.linear_act(x3.view(-1, K), w_big[:, :K], None, r3.view(-1, N), "gelu"))
    assert amd.linear_act(x3[0, 0], w_big[:, :K]).shape == (N,)


def test_linear_act_special_values_stay_in_their_row(amd):
    for M, N, K in ((1, 72, 64), (9, 72, 100), (200, 520, 192)):
        x, w = rnd(1, M, K), rnd(2, N, K)
        x[-1, 3], x[-1, 4] = float("inf"), float("nan")
        w[5] = 0
        got = amd.linear_act(x, w, None, None, "none")
        assert got[-1].isnan().all()
        if M > 1:
            close(got[:-1], *[t[:-1] for t in linear64(x, w, None, None, "none")["out"]], (M, N, K))
        # an infinite residual and bias arrive as they are
        x = rnd(1, M, K)
        bias, res = rnd(3, N), rnd(4, M, N)
        bias[1], res[0, 2] = float("-inf"), float("inf")
        got = amd.linear_act(x, w, bias, res, "none")
        assert (got[:, 1] == float("-inf")).all() and got[0, 2] == float("inf") and got[:, 3:].isfinite().all()


def test_linear_act_empty(amd):
    w = rnd(1, 24, 64).requires_grad_()
    x = torch.empty(0, 64, dtype=BF, device=D, requires_grad=True)
    out = amd.linear_act(x, w, None, None, "gelu")
    assert out.shape == (0, 24)
    dx, dw = torch.autograd.grad(out, [x, w], torch.empty_like(out))
    assert dx.shape == (0, 64) and (dw == 0).all()


def test_linear_act_gradients_that_are_asked_for(amd):
    x, w, b = rnd(1, 70, 96), rnd(2, 40, 96), rnd(3, 40)
    dout = rnd(4, 70, 40)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    full = torch.autograd.grad(amd.linear_act(*leaves, None, "silu"), leaves, dout)
    for i in range(3):
        only = [t.detach().requires_grad_(j == i) for j, t in enumerate((x, w, b))]
        (g,) = torch.autograd.grad(amd.linear_act(*only, None, "silu"), [only[i]], dout)
        assert torch.equal(g, full[i])


# ------------------------------------------------------------------------------------------------ qk_norm_rope

EPS = 1.1920928955078125e-07


def tables(P, R, dtype=F32):
    a = torch.arange(P, dtype=F64)[:, None] * (1e-4 ** (torch.arange(R // 2, dtype=F64) * 2 / R))
    return a.cos().to(dtype).to(D), a.sin().to(dtype).to(D)


def rope64(x, w, cos, sin, pos, interleaved, eps, dy=None):
    """x [B, T, H, D]; values and bounds of y, dx, dw"""
    dt, Dh, R = x.dtype, x.shape[-1], 2 * cos.shape[1]
    x = x.double()
    c, s = cos.double()[pos].unsqueeze(-2), sin.double()[pos].unsqueeze(-2)
    wd = torch.ones(Dh, dtype=F64, device=x.device) if w is None else w.double()

    def turn(v, sign):
        a, b = (v[..., 0:R:2], v[..., 1:R:2]) if interleaved else (v[..., :R // 2], v[..., R // 2:R])
        p, q = a * c - sign * b * s, b * c + sign * a * s
        rot = torch.stack((p, q), -1).flatten(-2) if interleaved else torch.cat((p, q), -1)
        return torch.cat((rot, v[..., R:]), -1)

    def reach(v):       # largest value the rotation can give an element
        a, b = (v[..., 0:R:2], v[..., 1:R:2]) if interleaved else (v[..., :R // 2], v[..., R // 2:R])
        m = a.abs() * c.abs() + b.abs() * s.abs(), b.abs() * c.abs() + a.abs() * s.abs()
        rot = torch.stack(m, -1).flatten(-2) if interleaved else torch.cat(m, -1)
        return torch.cat((rot, v[..., R:].abs()), -1)

    n = (Dh + 32) * E
    r = (x.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    xn = x * r
    y = turn(xn * wd, 1)
    res = {"y": (y, U[dt] * y.abs() + n * reach(xn * wd))}
    if dy is None:
        return res
    g = turn(dy.double(), -1)
    gmag = reach(dy.double())
    rows = g[..., 0].numel()
    dw = (g * xn).sum((0, 1, 2))
    res["dw"] = (dw, U[dt] * dw.abs() + (rows + Dh + 32) * E * (gmag * xn.abs()).sum((0, 1, 2)))
    gw = g * wd
    dx = r * (gw - xn * (gw * xn).mean(-1, keepdim=True))
    mag = r * (gmag * wd.abs() + xn.abs() * (gmag * wd.abs() * xn.abs()).mean(-1, keepdim=True))
    res["dx"] = (dx, U[dt] * dx.abs() + 4 * n * mag)
    return res


def check_rope(amd, q, k, cos, sin, positions, qw, kw, interleaved, what, eps=None):
    B, T = (q.shape[0], q.shape[1]) if q.ndim == 4 else (1, q.shape[0])
    pos = torch.arange(T, device=D).expand(B, T) if positions is None else positions.long().expand(B, T)
    four = lambda t: t if t.ndim == 4 else t.unsqueeze(0)
    leaves = {n: t.detach().requires_grad_() for n, t in (("q", q), ("k", k), ("qw", qw), ("kw", kw)) if t is not None}
    plain = amd.qk_norm_rope(q, k, cos, sin, positions, qw, kw, eps, interleaved)
    outs = amd.qk_norm_rope(leaves["q"], leaves["k"], cos, sin, positions, leaves.get("qw"), leaves.get("kw"), eps, interleaved)
    dq, dk = rnd(91, *q.shape, dtype=q.dtype), rnd(92, *k.shape, dtype=q.dtype)
    grads = dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), (dq, dk))))
    for n, x, w, out, pl, dy in (("q", q, qw, outs[0], plain[0], dq), ("k", k, kw, outs[1], plain[1], dk)):
        ref = rope64(four(x), w, cos, sin, pos, interleaved, EPS if eps is None else eps, four(dy))
        assert torch.equal(pl, out) and out.dtype == x.dtype and out.is_contiguous()
        close(four(out), *ref["y"], (what, n))
        close(four(grads[n]), *ref["dx"], (what, "d" + n))
        if w is not None:
            close(grads[n + "w"], *ref["dw"], (what, "dw", n))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("Dh,R", [(2, 2), (8, 6), (16, 16), (34, 20), (64, 64), (64, 24), (80, 80), (128, 128), (128, 64), (136, 100), (255, 254), (256, 256), (512, 512)])
def test_qk_norm_rope_head_sizes(amd, dtype, Dh, R):
    cos, sin = tables(40, R)
    for i, (shape_q, shape_k) in enumerate((((1, 1, Dh), (1, 1, Dh)), ((2, 19, 6, Dh), (2, 19, 2, Dh)), ((37, 5, Dh), (37, 3, Dh)))):
        q, k = rnd(1 + i, *shape_q, dtype=dtype), rnd(2 + i, *shape_k, dtype=dtype)
        for interleaved in (False, True):
            w = i != 0
            check_rope(amd, q, k, cos, sin, None, rnd(3, Dh, dtype=dtype) if w else None, rnd(4, Dh, dtype=dtype) if w and i == 1 else None,
                       interleaved, (dtype, Dh, R, i, interleaved))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_qk_norm_rope_packed_views_and_positions(amd, dtype):
    B, T, Hq, Hk, Dh = 3, 33, 6, 2, 64
    cos, sin = tables(5000, Dh)
    qkv = rnd(1, B, T, Hq + 2 * Hk, Dh, dtype=dtype)
    q, k = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk]
    pos = torch.randint(0, 5000, (B, T), generator=torch.Generator().manual_seed(3)).to(D)
    for p in (pos, pos.int(), pos[0].contiguous(), pos.t().contiguous().t(), pos[:, :1].expand(B, T)):
        check_rope(amd, q, k, cos, sin, p, None, None, False, "packed")
    # heads before tokens, odd offsets, an eps that matters, tables in bf16
    qt, kt = rnd(4, B, Hq, T, Dh, dtype=dtype).transpose(1, 2), rnd(5, B, Hk, T, Dh + 2, dtype=dtype).transpose(1, 2)[..., 1:1 + Dh]
    check_rope(amd, qt * 1e-3, kt, cos.to(BF), sin.to(BF), pos, rnd(6, Dh, dtype=dtype), None, True, "transposed", eps=1e-2)
    # one head shared by all tokens of a batch (stride 0)
    check_rope(amd, rnd(7, Hq, Dh, dtype=dtype).expand(T, Hq, Dh), rnd(8, T, 1, Dh, dtype=dtype).expand(T, Hk, Dh), cos, sin, None, None, None, False, "expanded")


def test_qk_norm_rope_many_rows(amd):
    """more rows than the grid holds at once: the walk over items, and the weight sums over every workgroup"""
    cos, sin = tables(6000, 32)
    q, k = rnd(1, 2, 5003, 12, 64, dtype=F32), rnd(2, 2, 5003, 4, 64, dtype=F32)
    check_rope(amd, q, k, cos, sin, None, rnd(3, 64, dtype=F32), rnd(4, 64, dtype=F32), False, "many")
    once = amd.qk_norm_rope(q, k, cos, sin)
    assert all(torch.equal(a, b) for a, b in zip(once, amd.qk_norm_rope(q, k, cos, sin)))


def test_qk_norm_rope_positions_outside_the_tables(amd):
    cos, sin = tables(16, 64)
    for Dh in (64, 66):
        q, k = rnd(1, 5, 4, Dh), rnd(2, 5, 2, Dh)
        pos = torch.tensor([3, -1, 15, 16, 1 << 40], device=D)
        qo, ko = amd.qk_norm_rope(q, k, cos, sin, pos)
        for o in (qo, ko):
            assert o[[1, 3, 4]].isnan().all() and o[[0, 2]].isfinite().all()
        leaf = q.detach().requires_grad_()
        (g,) = torch.autograd.grad(amd.qk_norm_rope(leaf, k, cos, sin, pos)[0], [leaf], rnd(3, 5, 4, Dh))
        assert g[[1, 3, 4]].isnan().all() and g[[0, 2]].isfinite().all()


def test_qk_norm_rope_zero_rows_and_empty(amd):
    cos, sin = tables(16, 64)
    q = torch.zeros(4, 2, 64, dtype=F32, device=D, requires_grad=True)
    k = rnd(1, 4, 2, 64, dtype=F32)
    qo, _ = amd.qk_norm_rope(q, k, cos, sin)
    assert (qo == 0).all()
    (g,) = torch.autograd.grad(qo, [q], torch.ones_like(qo))
    close(g[None], *rope64(q.detach()[None], None, cos, sin, torch.arange(4, device=D)[None], False, EPS, torch.ones(1, 4, 2, 64, device=D))["dx"], "zero rows")
    w = torch.ones(64, dtype=BF, device=D, requires_grad=True)
    e = torch.empty(0, 2, 64, dtype=BF, device=D, requires_grad=True)
    qo, ko = amd.qk_norm_rope(e, e, cos, sin, None, w, w)
    assert qo.shape == (0, 2, 64)
    assert (torch.autograd.grad((qo, ko), [w], (torch.empty_like(qo), torch.empty_like(ko)))[0] == 0).all()


def test_qk_norm_rope_gradient_against_differences(amd):
    cos, sin = tables(8, 48)
    q, k, w = rnd(1, 8, 3, 64, dtype=F32), rnd(2, 8, 1, 64, dtype=F32), rnd(3, 64, dtype=F32)
    cq, ck = rnd(4, 8, 3, 64, dtype=F32), rnd(5, 8, 1, 64, dtype=F32)

    def f(q, w):
        a, b = amd.qk_norm_rope(q, k, cos, sin, None, w, None)
        return (a.double() * cq).sum() + (b.double() * ck).sum()

    ql, wl = q.clone().requires_grad_(), w.clone().requires_grad_()
    gq, gw = torch.autograd.grad(f(ql, wl), [ql, wl])
    vq, vw = rnd(6, 8, 3, 64, dtype=F32), rnd(7, 64, dtype=F32)
    h = 2.0 ** -6
    diff = float(f(q + h * vq, w + h * vw) - f(q - h * vq, w - h * vw)) / (2 * h)
    formula = float((gq.double() * vq).sum() + (gw.double() * vw).sum())
    # central differences: h^2 / 6 of the third derivative (values of order sqrt(8 * 4 * 64) * a few), and 2^-24 roundings over 2 h
    assert abs(diff - formula) < 45 * (h * h * 10 + 2.0 ** -24 * 64 / h), (diff, formula)


# ------------------------------------------------------------------------------------------------ distill_topk

CAP = (23.0, 5.0, 7.5)


def distill64(logits, ids, teacher, lse, weight, tau, cap, up=None):
    """losses and gradient, each with its bound; loops over rows, entry by entry"""
    T, V = logits.shape
    x = logits.double()
    sg = torch.sigmoid((x + cap[1]) / cap[2]) if cap else None
    z = (cap[0] * sg if cap else x) / tau
    losses, lbound = torch.zeros(T, dtype=F64), torch.zeros(T, dtype=F64)
    grad, gbound = torch.zeros(T, V, dtype=F64), torch.zeros(T, V, dtype=F64)
    for t in range(T):
        w = 1.0 if weight is None else float(weight[t])
        if w == 0.0:
            continue
        use = [(int(i), float(v)) for i, v in zip(ids[t], teacher[t]) if 0 <= int(i) < V]
        tz = torch.tensor([v / float(torch.tensor(tau, dtype=F32)) for _, v in use], dtype=F64)
        if not use or (lse is None and tz.max() == -math.inf):
            continue
        col = torch.tensor([i for i, _ in use])
        zt = z[t].cpu() - z[t].cpu().max()         # (first: log V is lost next to 3e38 even in 64 bits)
        logq = zt - torch.logsumexp(zt, 0)
        q = logq.exp()
        logp = tz - (torch.logsumexp(tz, 0) if lse is None else float(lse[t]))
        p = logp.exp()
        terms = torch.where(p == 0, torch.zeros_like(p), p * (logp - logq[col]))
        kl, ratio = terms.sum(), 0.0
        out = torch.ones(V, dtype=torch.bool)
        out[col] = False
        rest_p = max(0.0, 1 - float(p.sum())) if lse is not None and out.any() else 0.0
        logrest = torch.logsumexp(logq[out], 0) if out.any() else None
        if rest_p > 0 and out.any():
            kl = kl + rest_p * (math.log(rest_p) - logrest)
            ratio = rest_p / float(logrest.exp())
        losses[t] = w * tau * tau * kl
        # the sum's terms: V / 1024 per thread and a tree; exponentials whose argument matters are below 2^6; the softcap's sigma to a few 2^-24
        rel = (V / 1024 + 256) * E + (400 * E / tau if cap else 0) + 64 * E / tau
        zfin = torch.where(p == 0, torch.zeros_like(p), (zt[col] - zt[col].max()).abs().nan_to_num(posinf=0))
        size = 1 + (p * logp.abs().nan_to_num(posinf=0)).sum() + (p * zfin).sum() + (rest_p * abs(float(logrest)) if rest_p > 0 and out.any() else 0)
        lbound[t] = abs(w) * tau * tau * (4 * rel * (p.sum() + rest_p) + rel * size) + 4 * E * losses[t].abs()
        if up is not None:
            f = torch.full((V,), float(p.sum()) + rest_p, dtype=F64)
            fabs = f.clone()
            f[out] -= ratio
            fabs[out] += ratio
            pv = torch.zeros(V, dtype=F64).index_add_(0, col, p)
            base = w * float(up[t]) * tau
            slope = (cap[0] / cap[2] * sg[t] * (1 - sg[t])).cpu() if cap else torch.ones(V, dtype=F64)
            grad[t] = base * (q * f - pv) * slope
            gbound[t] = abs(base) * (q * fabs * 8 * rel + pv * 8 * E + 1e-34) * slope.abs() + U[logits.dtype] * grad[t].abs() + 1e-36
            gbound[t] += abs(base) * (q * fabs + pv) * 16 * E * (cap[0] / cap[2] * sg[t].cpu() if cap else 0)       # 1 - sigma near 1
    return (losses.to(D), lbound.to(D)), (grad.to(D), gbound.to(D))


def teacher_rows(seed, T, V, K, tail_at=None):
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(T)]).to(D)
    t = (torch.randn(T, K, generator=g) * 2 + 3).to(D)
    lse = None if tail_at is None else torch.logsumexp(t.double() / tail_at, 1).float() + torch.rand(T, generator=g).to(D) * 0.4 + 1e-3
    return ids, t, lse


def check_distill(amd, logits, ids, teacher, lse=None, weight=None, tau=1.0, cap=None, what=None):
    T = logits.shape[0]
    up = rnd(77, T, dtype=F32)
    (loss, lb), (grad, gb) = distill64(logits, ids, teacher, lse, weight, tau, cap, up)
    kw = dict(teacher_lse=lse, row_weight=weight, temperature=tau, softcap=cap)
    got = amd.distill_topk(logits, ids, teacher, **kw)
    close(got, loss, lb, (what, "loss"))
    leaf = logits.detach().requires_grad_()
    again = amd.distill_topk(leaf, ids, teacher, **kw)
    assert torch.equal(again, got) or (got.isnan() == again.isnan()).all()
    (g,) = torch.autograd.grad(again, [leaf], up)
    assert g.dtype == logits.dtype
    close(g, grad, gb, (what, "grad"))
    losses, fused = amd.distill_topk_fwd_bwd(logits, ids, teacher, grad_scale=0.25, **kw)
    close(losses, loss, lb, (what, "fused loss"))
    _, (grad, gb) = distill64(logits, ids, teacher, lse, weight, tau, cap, torch.full((T,), 0.25))
    close(fused, grad, gb, (what, "fused grad"))


@pytest.mark.parametrize("cap", [None, CAP], ids=["plain", "softcap"])
@pytest.mark.parametrize("tail", [False, True], ids=["list", "rest"])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,V,K", [(1, 1, 1), (2, 7, 3), (5, 100, 7), (3, 1000, 64), (4, 4099, 65), (3, 16384, 200), (2, 16401, 33), (3, 32768, 5), (3, 50304, 64),
                                   (2, 57328, 512), (2, 57341, 10), (2, 70001, 30)])
def test_distill_sizes(amd, cap, tail, dtype, T, V, K):
    tau = (1.0, 2.0, 0.7)[V % 3]
    ids, teacher, lse = teacher_rows(V, T, V, K, tau if tail else None)
    check_distill(amd, rnd(V + 1, T, V, dtype=dtype, scale=3.0), ids if V % 2 else ids.int(), teacher, lse, None, tau, cap, (T, V, K))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_distill_rows_that_start_anywhere(amd, dtype):
    T, V, K = 5, 1237, 9
    ids, teacher, lse = teacher_rows(1, T, V, K, 1.0)
    big = rnd(2, T, V + 29, dtype=dtype, scale=3.0)
    for off in range(0, 9):
        check_distill(amd, big[:, off:off + V], ids, teacher, lse, None, 1.0, None, off)
    check_distill(amd, rnd(3, V, T, dtype=dtype).t(), ids.t().contiguous().t(), teacher.t().contiguous().t(), lse, None, 1.0, CAP, "transposed")


@pytest.mark.parametrize("cap", [None, CAP], ids=["plain", "softcap"])
@pytest.mark.parametrize("tail", [False, True], ids=["list", "rest"])
def test_distill_lists_with_holes_and_repetitions(amd, cap, tail):
    T, V, K = 9, 300, 40
    ids, teacher, lse = teacher_rows(1, T, V, K, 1.0 if tail else None)
    ids[0, 3:] = -1                       # a short list
    ids[1] = -1                           # an empty one
    ids[2, 5], ids[2, 6] = V, 1 << 40     # not columns
    ids[3, 10:20] = ids[3, 9]             # one column eleven times
    ids[4] = 17                           # the same column throughout
    ids[5, 1] = ids[5, 0] = V - 1
    teacher[6, 4:] = -math.inf            # entries of no mass
    teacher[7] = -math.inf
    if tail:
        lse = torch.logsumexp(teacher.double(), 1).float().nan_to_num(neginf=0.0) + 0.2
        lse[3:5] += 2.0
        lse[0] = teacher[0, :3].logsumexp(0) - 0.01       # more than the whole mass listed: no rest
    weight = torch.tensor([1, 0.5, 1, 2, 1, 0, 1, 1, 3.0], device=D)
    logits = rnd(2, T, V, dtype=F32, scale=3.0)
    check_distill(amd, logits, ids, teacher, lse, weight, 1.0, cap, "holes")
    # a row of weight 0 may hold anything
    logits[5] = float("nan")
    losses, grad = amd.distill_topk_fwd_bwd(logits, ids, teacher, teacher_lse=lse, row_weight=weight, softcap=cap)
    assert losses[5] == 0 and (grad[5] == 0).all() and grad.isfinite().all() and losses.isfinite().all()
    leaf = logits.requires_grad_()
    loss = amd.distill_topk(leaf, ids, teacher, teacher_lse=lse, row_weight=weight, softcap=cap)
    (g,) = torch.autograd.grad(loss.sum(), [leaf])
    assert loss[5] == 0 and (g[5] == 0).all() and g.isfinite().all()
    assert loss[1] == 0 and (g[1] == 0).all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("tail", [False, True], ids=["list", "rest"])
def test_distill_masked_logits(amd, dtype, tail):
    T, V, K = 6, 5000, 20
    ids, teacher, lse = teacher_rows(1, T, V - 100, K, 1.0 if tail else None)
    logits = rnd(2, T, V, dtype=dtype, scale=3.0)
    logits[:, V - 100:] = -math.inf
    logits[1, V - 100:] = torch.finfo(dtype).min
    logits[2] = logits[2] + 1000
    logits[3] = torch.finfo(dtype).min                         # everything at the lowest value: a uniform row
    logits[4, :2500] = -math.inf
    ids[4] = torch.arange(2600, 2600 + K, device=D)
    check_distill(amd, logits, ids, teacher, lse, None, 1.0, None, "masked")
    # a listed column that the student rules out: infinite loss; every column listed: no rest
    logits[0, ids[0, 0]] = -math.inf
    assert amd.distill_topk(logits, ids, teacher, lse)[0] == math.inf
    small = rnd(3, 3, 12, dtype=dtype)
    ids, teacher, lse = teacher_rows(4, 3, 12, 12, 1.0)
    check_distill(amd, small, ids, teacher, lse, None, 1.0, None, "all listed")
    nan = rnd(5, 3, 500, dtype=dtype)
    nan[1, 77] = float("nan")
    ids, teacher, lse = teacher_rows(6, 3, 500, 4, 1.0 if tail else None)
    losses, grad = amd.distill_topk_fwd_bwd(nan, ids, teacher, teacher_lse=lse)
    assert losses[1].isnan() and grad[1].isnan().any() and losses[[0, 2]].isfinite().all() and grad[[0, 2]].isfinite().all()


def test_distill_many_rows_and_repeatable(amd):
    T, V, K = 700, 3001, 16
    ids, teacher, lse = teacher_rows(1, T, V, K, 1.0)
    logits = rnd(2, T, V, dtype=F32, scale=2.0)
    up = torch.full((T,), 1.0)
    (loss, lb), (grad, gb) = distill64(logits, ids.cpu(), teacher.cpu(), lse.cpu(), None, 1.0, None, up)
    a = amd.distill_topk_fwd_bwd(logits, ids, teacher, lse)
    b = amd.distill_topk_fwd_bwd(logits, ids, teacher, lse)
    close(a[0], loss, lb, "loss")
    close(a[1], grad, gb, "grad")
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    leaf = logits.requires_grad_()
    (g,) = torch.autograd.grad(amd.distill_topk(leaf, ids, teacher, lse).sum(), [leaf])      # an expanded incoming gradient
    close(g, grad, gb, "expanded")


def test_distill_gradient_against_differences(amd):
    T, V, K = 4, 600, 12
    ids, teacher, lse = teacher_rows(1, T, V, K, 2.0)
    logits, v = rnd(2, T, V, dtype=F32, scale=2.0), rnd(3, T, V, dtype=F32)
    for cap in (None, CAP):
        f = lambda l: amd.distill_topk(l, ids, teacher, lse, temperature=2.0, softcap=cap)
        leaf = logits.clone().requires_grad_()
        (g,) = torch.autograd.grad(f(leaf).sum(), [leaf])
        h = 2.0 ** -5
        diff = float((f(logits + h * v).double() - f(logits - h * v).double()).sum()) / (2 * h)
        formula = float((g.double() * v).sum())
        # h^2 / 6 of a third derivative of order (slope |v|)^3, and loss errors of 2^-24 * 600 over h
        assert abs(diff - formula) < T * (h * h * 30 + 600 * E * 10 / h), (cap, diff, formula)


# ------------------------------------------------------------------------------------------------ past 2^32 bytes

def test_linear_act_of_more_than_4_gib(amd):
    """whole numbers small enough that every sum is exact: all results are the rounded true values"""
    M, N, K = 1_200_003, 2048, 64
    whole = lambda seed, *shape: torch.randint(-1, 2, shape, generator=torch.Generator(D).manual_seed(seed), device=D, dtype=torch.int8).to(BF)
    x, w, b, dout = whole(1, M, K), whole(2, N, K), whole(3, N), whole(4, M, N)
    x, w, b = (t.requires_grad_() for t in (x, w, b))
    out = amd.linear_act(x, w, b, None, "relu2")
    dx, dw, db = torch.autograd.grad(out, [x, w, b], dout)
    with torch.no_grad():
        dw64, db64, step = torch.zeros(N, K, device=D, dtype=F64), torch.zeros(N, device=D, dtype=F64), 100_000
        for i in range(0, M, step):
            xs = x[i:i + step].float()
            z = (xs @ w.float().t() + b.float()).clamp_min(0)             # at most 65
            assert torch.equal(out[i:i + step], (z * z).to(BF)), i
            dz = 2 * z * dout[i:i + step].float()                          # at most 130 and even: exact in bf16
            assert torch.equal(dx[i:i + step], (dz @ w.float()).to(BF)), i
            dw64 += dz.t() @ xs
            db64 += dz.sum(0, dtype=F64)
        assert torch.equal(dw, dw64.float().to(BF)) and torch.equal(db, db64.float().to(BF))


def test_qk_norm_rope_of_more_than_4_gib(amd):
    T, H, Dh, tail = 1_100_003, 17, 128, 1000
    cos, sin = tables(4096, Dh)
    pos = torch.arange(T, device=D) % 4096
    q = torch.randn(T, H, Dh, generator=torch.Generator(D).manual_seed(1), device=D, dtype=BF).requires_grad_()
    k = rnd(2, T // 1000 + 1, 1, Dh).repeat(1000, 1, 1)[:T].contiguous().requires_grad_()
    qo, ko = amd.qk_norm_rope(q, k, cos, sin, pos)
    dq, dk = torch.autograd.grad([qo, ko], [q, k], [q.detach(), k.detach()])
    q2, k2 = (t.detach()[-tail:].clone().requires_grad_() for t in (q, k))
    qo2, ko2 = amd.qk_norm_rope(q2, k2, cos, sin, pos[-tail:])
    dq2, dk2 = torch.autograd.grad([qo2, ko2], [q2, k2], [q2.detach(), k2.detach()])
    # (few tokens take another variant: two roundings of nearly the same value)
    for a, e in ((qo, qo2), (ko, ko2), (dq, dq2), (dk, dk2)):
        a, e = a[-tail:].detach().double(), e.detach().double()
        assert bool(((a - e).abs() <= 2.0 ** -7 * e.abs() + 2.0 ** -18 * e.abs().max()).all())


def test_distill_of_more_than_4_gib(amd):
    T, V, K, tail = 44_001, 50304, 8, 64
    ids, teacher, lse = teacher_rows(1, tail, V, K, 1.0)
    rows = lambda t: t.repeat(T // tail + 1, *[1] * (t.ndim - 1))[-T:].contiguous()
    logits = torch.randn(T, V, generator=torch.Generator(D).manual_seed(2), device=D, dtype=BF)
    ids, teacher, lse = rows(ids), rows(teacher), rows(lse)
    losses, grad = amd.distill_topk_fwd_bwd(logits, ids, teacher, lse, softcap=CAP)
    few = amd.distill_topk_fwd_bwd(logits[-tail:], ids[-tail:], teacher[-tail:], lse[-tail:], softcap=CAP)
    assert torch.equal(losses[-tail:], few[0]) and torch.equal(grad[-tail:], few[1])
    del grad
    leaf = logits.requires_grad_()
    (g,) = torch.autograd.grad(amd.distill_topk(leaf, ids, teacher, lse, softcap=CAP), [leaf], torch.ones(T, device=D))
    last = logits.detach()[-tail:].clone().requires_grad_()
    (g2,) = torch.autograd.grad(amd.distill_topk(last, ids[-tail:], teacher[-tail:], lse[-tail:], softcap=CAP), [last], torch.ones(tail, device=D))
    # (few rows take another sweep width: the sums' order differs; a gradient's terms are off by some 2^-20 and the store by 2^-8)
    assert float((g[-tail:].double() - g2.double()).abs().max()) <= 2.0 ** -7 * float(g2.double().abs().max())


# ------------------------------------------------------------------------------------------------ together

def step(fn_linear, fn_rope, fn_loss, p, B, T, H, Hk, Dh):
    """one block and the loss on top: projections, heads, attention written out, output projection, MLP, logits"""
    x = p["x"]
    qkv = fn_linear(x, p["w_qkv"], p["b_qkv"], None, "none").view(B, T, H + 2 * Hk, Dh)
    q, k = fn_rope(qkv[:, :, :H], qkv[:, :, H:H + Hk], p["g_q"], p["g_k"])
    v = qkv[:, :, H + Hk:]
    k, v = (t.repeat_interleave(H // Hk, 2) for t in (k, v))
    s = (q.unsqueeze(2).to(F32 if q.dtype == BF else F64) * k.unsqueeze(1)).sum(-1) / Dh ** 0.5          # [B, T, T, H]
    s = s.masked_fill(torch.ones(T, T, dtype=torch.bool, device=x.device).triu(1)[None, :, :, None], -math.inf)
    a = (s.softmax(2).unsqueeze(-1) * v.unsqueeze(1)).sum(2).to(x.dtype).reshape(B, T, H * Dh)
    x = fn_linear(a, p["w_o"], None, x, "none")
    x = fn_linear(fn_linear(x, p["w_up"], p["b_up"], None, "gelu_tanh"), p["w_down"], None, x, "none")
    return fn_loss(fn_linear(x, p["w_head"], None, None, "none").view(B * T, -1))


def make_step(B=2, T=24, H=4, Hk=2, Dh=32, V=500, K=8):
    dim = H * Dh
    p = {"x": rnd(1, B, T, dim), "w_qkv": rnd(2, (H + 2 * Hk) * Dh, dim, scale=dim ** -0.5), "b_qkv": rnd(3, (H + 2 * Hk) * Dh, scale=0.1),
         "g_q": 1 + rnd(4, Dh, scale=0.1), "g_k": 1 + rnd(5, Dh, scale=0.1), "w_o": rnd(6, dim, dim, scale=dim ** -0.5),
         "w_up": rnd(7, 4 * dim, dim, scale=dim ** -0.5), "b_up": rnd(8, 4 * dim, scale=0.1), "w_down": rnd(9, dim, 4 * dim, scale=dim ** -0.5 / 2),
         "w_head": rnd(10, V, dim, scale=dim ** -0.5)}
    ids, teacher, lse = teacher_rows(11, B * T, V, K, 1.0)
    return p, ids, teacher, lse, (B, T, H, Hk, Dh), tables(T, Dh)


def test_a_block_and_its_loss(amd):
    p, ids, teacher, lse, dims, (cos, sin) = make_step()
    B, T, H, Hk, Dh = dims
    mine = {n: t.detach().requires_grad_() for n, t in p.items()}
    loss = step(amd.linear_act, lambda q, k, gq, gk: amd.qk_norm_rope(q, k, cos, sin, None, gq, gk),
                lambda l: amd.distill_topk(l, ids, teacher, lse, softcap=CAP), mine, *dims).mean()
    grads = torch.autograd.grad(loss, list(mine.values()))

    ref = {n: t.detach().double().requires_grad_() for n, t in p.items()}

    def linear(x, w, b, r, act):
        z = x @ w.t() + (0 if b is None else b)
        y = z if act == "none" else torch.nn.functional.gelu(z, approximate="tanh")
        return y if r is None else y + r

    def rope(q, k, gq, gk):
        def one(x, g):
            y = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * g
            a, b, c, s = y[..., :Dh // 2], y[..., Dh // 2:], cos.double()[:, None], sin.double()[:, None]
            return torch.cat((a * c - b * s, b * c + a * s), -1)
        return one(q, gq), one(k, gk)

    def loss64(l):
        logq = torch.log_softmax(CAP[0] * torch.sigmoid((l + CAP[1]) / CAP[2]), 1)
        logp = teacher.double() - lse.double()[:, None]
        rest = 1 - logp.exp().sum(1)
        others = logq.scatter(1, ids, -math.inf).logsumexp(1)
        return (logp.exp() * (logp - logq.gather(1, ids))).sum(1) + rest * (rest.log() - others)

    want = step(linear, rope, loss64, ref, *dims).mean()
    wgrads = torch.autograd.grad(want, list(ref.values()))
    # a dozen bf16 roundings on the way (2^-8 each, partly independent): 12 * 2^-8 of the value's scale
    assert abs(float(loss) - float(want)) < 12 * 2.0 ** -8 * max(1.0, float(want))
    for n, g, wg in zip(mine, grads, wgrads):
        rel = float((g.double() - wg).norm() / wg.norm())
        assert rel < 12 * 2.0 ** -8, (n, rel)


def test_a_block_on_another_stream_and_repeated(amd):
    p, ids, teacher, lse, dims, (cos, sin) = make_step()

    def run():
        leaves = {n: t.detach().requires_grad_() for n, t in p.items()}
        loss = step(amd.linear_act, lambda q, k, gq, gk: amd.qk_norm_rope(q, k, cos, sin, None, gq, gk),
                    lambda l: amd.distill_topk(l, ids, teacher, lse), leaves, *dims).sum()
        return [loss.detach(), *torch.autograd.grad(loss, list(leaves.values()))]

    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_replays_from_a_hip_graph(amd):
    """forward and gradients of the three operators captured once, replayed on new inputs between eager work"""
    M, K, N, V, C = 200, 192, 264, 700, 6
    cos, sin = tables(M, 32)
    x, w, b, r, dout = rnd(1, M, K), rnd(2, N, K, scale=0.1), rnd(3, N), rnd(4, M, N), rnd(5, M, N)
    q, k, dq, dk = rnd(6, M, 4, 32), rnd(7, M, 2, 32), rnd(8, M, 4, 32), rnd(9, M, 2, 32)
    ids, teacher, lse = teacher_rows(10, M, V, C, 1.0)
    logits = rnd(11, M, V, scale=2.0)
    ops = torch.ops.nanogpt

    def run():
        out, pre = ops.linear_act(x, w, b, r, "silu", True)
        g = ops.linear_act_backward(dout, x, w, pre, "silu", True, True, True)
        few = amd.linear_act(x[:3], w, b, r[:3], "gelu")
        qo, ko = amd.qk_norm_rope(q, k, cos, sin, None, q[0, 0], None)
        h = ops.qk_norm_rope_backward(dq, dk, q, k, cos, sin, None, q[0, 0], None, EPS, False, True, False)
        losses, grad = amd.distill_topk_fwd_bwd(logits, ids, teacher, lse, softcap=CAP)
        l2, stats = ops.distill_topk(logits, ids, teacher, None, None, 1.0, 0.0, 0.0, 0.0)
        g2 = ops.distill_topk_backward(losses, logits, ids, teacher, None, None, stats, 1.0, 0.0, 0.0, 0.0)
        return [out, *g, few, qo, ko, *h[:3], losses, grad, l2, g2]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    for i in range(3):
        for t in (x, dout, q, dq, logits):
            t.copy_(rnd(20 + i, *t.shape))
        eager = [t.clone() for t in run()]
        graph.replay()
        torch.cuda.synchronize()
        for j, (a, e) in enumerate(zip(captured, eager)):
            assert torch.equal(a, e), (i, j)


def test_traces_under_torch_compile(amd):
    M, K, N, V, C = 48, 64, 72, 300, 5
    cos, sin = tables(M, 24)
    x, w, b = rnd(1, M, K).requires_grad_(), rnd(2, N, K, scale=0.1).requires_grad_(), rnd(3, N).requires_grad_()
    head = rnd(4, V, N, scale=0.1)
    ids, teacher, _ = teacher_rows(5, M, V, C)

    def f(x, w, b):
        y = amd.linear_act(x, w, b, None, "silu").view(M, 3, 24)
        q, k = amd.qk_norm_rope(y[:, :2], y[:, 2:], cos, sin)
        h = torch.cat((q, k), 1).reshape(M, N)
        return amd.distill_topk(amd.linear_act(h, head), ids, teacher, softcap=CAP).sum()

    eager = f(x, w, b)
    ge = torch.autograd.grad(eager, [x, w, b])
    traced = torch.compile(f, backend="aot_eager", fullgraph=True, dynamic=False)
    out = traced(x, w, b)
    gt = torch.autograd.grad(out, [x, w, b])
    assert torch.equal(out, eager)
    for a, e in zip(gt, ge):
        assert torch.equal(a, e)


def three_losses(amd):
    """(function of its leaves, the leaves) for each operator"""
    M, K, N, V, C = 48, 64, 72, 300, 5
    cos, sin = tables(M, 24)
    ids, teacher, _ = teacher_rows(5, M, V, C)
    leaves = lambda *ts: [t.requires_grad_() for t in ts]
    yield (lambda x, w, b: (amd.linear_act(x, w, b, None, "gelu").float() * 0.5).sum()), leaves(rnd(1, M, K), rnd(2, N, K, scale=0.1), rnd(3, N))
    yield (lambda q, k, g: sum((t.float() * 0.5).sum() for t in amd.qk_norm_rope(q, k, cos, sin, None, g))), leaves(rnd(6, M, 4, 24), rnd(7, M, 2, 24), rnd(8, 24))
    yield (lambda l: amd.distill_topk(l, ids, teacher).sum()), leaves(rnd(9, M, V))


def test_gradients_are_not_differentiated_again(amd):
    """a graph of the backward pass may be asked for, but going back through it raises"""
    for f, leaves in three_losses(amd):
        plain = torch.autograd.grad(f(*leaves), leaves)
        again = torch.autograd.grad(f(*leaves), leaves, create_graph=True)
        for a, b in zip(plain, again):
            assert torch.equal(a, b) and b.requires_grad
            with pytest.raises(RuntimeError, match="cannot be differentiated again"):
                torch.autograd.grad(b.float().sum(), leaves[0], retain_graph=True)


def test_forward_mode_is_refused(amd):
    from torch.autograd import forward_ad
    for f, leaves in three_losses(amd):
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward"):
            f(forward_ad.make_dual(leaves[0].detach(), torch.ones_like(leaves[0])), *(t.detach() for t in leaves[1:]))


def test_function_transforms_are_refused(amd):
    for f, leaves in three_losses(amd):
        for i in range(len(leaves)):
            with pytest.raises(RuntimeError, match="torch.func"):
                torch.func.grad(f, argnums=i)(*(t.detach() for t in leaves))


def test_saved_tensors_kept_elsewhere(amd):
    for f, leaves in three_losses(amd):
        plain = torch.autograd.grad(f(*leaves), leaves)
        with torch.autograd.graph.save_on_cpu():
            loss = f(*leaves)
        assert all(torch.equal(a, b) for a, b in zip(plain, torch.autograd.grad(loss, leaves)))


def test_an_input_changed_before_the_backward_raises(amd):
    for f, leaves in three_losses(amd):
        loss = f(*leaves)
        with torch.no_grad():
            leaves[0].add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(loss, leaves)


@pytest.mark.parametrize("M", [3, 40])
def test_linear_act_views_of_a_packed_tensor(amd, M):
    B, K, N = 3, 72, 136
    xs, ws, rs = rnd(1, B, M, 3 * K), rnd(2, N, 2 * K, scale=0.1), rnd(3, B, M, 2 * N)
    x, w, r = xs[..., K:2 * K], ws[:, K:], rs[..., N:]
    assert torch.equal(amd.linear_act(x, w, None, r, "silu"), amd.linear_act(x.contiguous(), w.contiguous(), None, r.contiguous(), "silu"))
    x2, w2 = x.transpose(0, 1), w.t().contiguous().t()        # rows that are not evenly spaced, a weight whose rows are not contiguous
    assert torch.equal(amd.linear_act(x2, w2), amd.linear_act(x2.contiguous(), w2.contiguous()))


def test_two_streams_at_once(amd):
    """the same operators on two streams, different inputs, nothing between them"""
    def inputs(seed):
        M, K, N, V = 700, 512, 520, 4000
        return (rnd(seed, M, K), rnd(seed + 1, N, K, scale=0.05).requires_grad_(), rnd(seed + 2, N).requires_grad_(), rnd(seed + 3, M, N),
                rnd(seed + 4, M, V).requires_grad_(), *teacher_rows(seed + 5, M, V, 16)[:2])

    def run(x, w, b, dout, logits, ids, teacher):
        out = amd.linear_act(x, w, b, None, "silu")
        return [out.detach(), *torch.autograd.grad(out, [w, b], dout), *amd.distill_topk_fwd_bwd(logits, ids, teacher)]

    sets = [inputs(10), inputs(30)]
    want = [[t.clone() for t in run(*s)] for s in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(run(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for result in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(result, want[i]))


def test_a_captured_training_step(amd):
    """forward and autograd's backward in one graph; no eager graph of the leaves is alive during the capture"""
    M, K, N, V, C = 200, 64, 96, 700, 6
    cos, sin = tables(M, 32)
    ids, teacher, lse = teacher_rows(10, M, V, C, 1.0)
    ones = torch.ones(M, device="cuda")
    leaves = {"x": rnd(1, M, K), "w": rnd(2, N, K, scale=0.1), "b": rnd(3, N), "g": 1 + rnd(4, 32, scale=0.1), "head": rnd(5, V, N, scale=0.1)}
    leaves = {n: t.detach().requires_grad_() for n, t in leaves.items()}

    def run():
        y = amd.linear_act(leaves["x"], leaves["w"], leaves["b"], None, "silu").view(M, 3, 32)
        h = torch.cat(amd.qk_norm_rope(y[:, :2], y[:, 2:], cos, sin, None, leaves["g"]), 1).view(M, N)
        losses = amd.distill_topk(amd.linear_act(h, leaves["head"]), ids, teacher, lse, softcap=CAP)
        return [losses.detach(), *torch.autograd.grad(losses, list(leaves.values()), ones)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    for i in range(3):
        with torch.no_grad():
            for j, t in enumerate(leaves.values()):
                t.mul_(1 + 0.01 * (i + 1)).add_(rnd(100 + 20 * i + j, *t.shape, scale=0.01))
        eager = [t.clone() for t in run()]
        graph.replay()
        torch.cuda.synchronize()
        for j, (a, e) in enumerate(zip(captured, eager)):
            assert torch.equal(a, e), (i, j)


def test_dispatch_modes_see_the_registered_operators(amd):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Names(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(func.__name__ if hasattr(func, "__name__") else str(func))
            return func(*args, **(kwargs or {}))

    names = ("linear_act", "qk_norm_rope", "distill_topk")
    for name, (f, leaves) in zip(names, three_losses(amd)):
        plain = torch.autograd.grad(f(*leaves), leaves)
        seen = []
        with Names():
            grads = torch.autograd.grad(f(*leaves), leaves)
        assert any(n.startswith(name + ".") for n in seen) and any(n.startswith(name + "_backward") for n in seen), seen
        assert all(torch.equal(a, b) for a, b in zip(plain, grads))
    ids, teacher, _ = teacher_rows(5, 4, 300, 5)
    seen = []
    logits = rnd(1, 4, 300)
    with Names():
        a = amd.distill_topk_fwd_bwd(logits, ids, teacher)
    assert any(n.startswith("distill_topk_fwd_bwd") for n in seen)
    assert all(torch.equal(x, y) for x, y in zip(a, amd.distill_topk_fwd_bwd(logits, ids, teacher)))


def test_a_traced_function_holds_the_registered_operator(amd):
    from torch.fx.experimental.proxy_tensor import make_fx
    x, w = rnd(1, 5, 64), rnd(2, 24, 64)
    g = make_fx(lambda x, w: amd.linear_act(x, w, activation="silu"))(x, w)
    assert "nanogpt.linear_act" in g.code
    y = rnd(3, 5, 64)
    assert torch.equal(g(y, w), amd.linear_act(y, w, activation="silu"))
    h = torch.jit.trace(lambda x, w: amd.linear_act(x, w, activation="silu"), (x, w))
    assert "nanogpt::linear_act" in str(h.graph)
    assert torch.equal(h(y, w), amd.linear_act(y, w, activation="silu"))

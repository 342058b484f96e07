"""Host side of linear_act, qk_norm_rope and distill_topk: argument checks of the C ABI and of the functions, schemas, fake implementations.
Nothing here touches a GPU."""
import ctypes

import pytest
import torch

BF = torch.bfloat16


@pytest.fixture(scope="module")
def amd():
    import modded_nanogpt_amd
    if not modded_nanogpt_amd._lib.LIB_PATH.exists():
        from modded_nanogpt_amd.build import build
        build(verbose=False)
    return modded_nanogpt_amd


def strides(*s):
    return (ctypes.c_int64 * len(s))(*s)


def test_linear_act_refusals(amd):
    lib = amd._lib.load()
    fwd = lambda x=16, ldx=64, w=16, ldw=64, bias=None, res=None, ldr=0, M=4, N=8, K=64, act=0, out=16, pre=None: lib.ngpt_linear_act_fwd(
        x, ldx, w, ldw, bias, res, ldr, M, N, K, act, out, pre, None)
    assert fwd(x=None) == -1 and fwd(w=None) == -1 and fwd(out=None) == -1
    assert fwd(M=0) == -1 and fwd(N=-1) == -1 and fwd(K=0) == -1
    assert fwd(act=5) == -1 and fwd(act=-1) == -1 and fwd(pre=16) == -1
    assert fwd(ldx=63) == -2 and fwd(ldw=32) == -2 and fwd(res=16, ldr=7) == -2
    assert fwd(bias=8) == -2 and b"16 bytes" in lib.ngpt_last_error()
    assert fwd(N=1 << 25) == -4 and fwd(ldx=1 << 22) == -4 and fwd(ldw=1 << 22) == -4 and fwd(res=16, ldr=1 << 22) == -4
    bwd = lambda dout=16, pre=None, x=16, w=16, M=4, N=8, K=64, act=0, dx=16, dw=16, db=16, ws=16, nws=1 << 40: lib.ngpt_linear_act_bwd(
        dout, pre, x, K, w, K, M, N, K, act, dx, dw, db, ws, nws, None)
    assert bwd(dout=None) == -1 and bwd(x=None) == -1 and bwd(w=None) == -1 and bwd(act=2) == -1 and bwd(M=0) == -1
    assert bwd(ws=None) == -3 and bwd(nws=64) == -3
    assert lib.ngpt_linear_act_bwd_workspace_bytes(0, 8, 64) == 0


def test_qk_norm_rope_refusals(amd):
    lib = amd._lib.load()
    s3, s2 = strides(64, 64, 8), strides(4, 1)

    def call(q=16, qs=s3, k=16, dt=0, B=1, T=4, Hq=2, Hk=1, D=8, R=8, cos=16, tdt=1, P=4, pos=None, ps=None, eps=1e-6, qo=16):
        return lib.ngpt_qk_norm_rope(q, qs, k, s3, dt, B, T, Hq, Hk, D, R, cos, 16, tdt, P, pos, 0, ps, None, None, eps, 0, qo, 16, None)

    assert call(q=None) == -1 and call(qs=None) == -1 and call(k=None) == -1 and call(cos=None) == -1 and call(qo=None) == -1
    assert call(dt=2) == -1 and call(tdt=-1) == -1
    for name in ("B", "T", "Hq", "Hk", "P"):
        assert call(**{name: 0}) == -1, name
    assert call(D=1) == -4 and call(D=513) == -4
    assert call(R=0) == -2 and call(R=7) == -2 and call(R=10) == -2
    assert call(T=5) == -4 and b"positions" in lib.ngpt_last_error()
    assert call(T=5, pos=16) == -1                       # positions need their strides
    assert call(eps=-1.0) == -4 and call(eps=float("nan")) == -4
    back = lambda dq=16, dqw=None, ws=None, nws=0: lib.ngpt_qk_norm_rope_bwd(dq, s3, 16, s3, 16, s3, 16, s3, 0, 1, 4, 2, 1, 8, 8, 16, 16, 1, 4, None, 0, s2,
                                                                             None, None, 1e-6, 0, 16, 16, dqw, None, ws, nws, None)
    assert back(dq=None) == -1 and back(dqw=16) == -3 and back(dqw=16, ws=16, nws=100) == -3


def test_distill_refusals(amd):
    lib = amd._lib.load()
    def fwd(logits=16, dt=0, ld=100, ids=16, t=16, T=2, V=100, K=4, tau=1.0, cap=(0.0, 0.0, 0.0), losses=16):
        return lib.ngpt_distill_fwd(logits, dt, ld, ids, 1, t, None, None, T, V, K, tau, *cap, losses, None, None)
    assert fwd(logits=None) == -1 and fwd(ids=None) == -1 and fwd(t=None) == -1 and fwd(losses=None) == -1
    assert fwd(dt=3) == -1 and fwd(T=0) == -1 and fwd(V=0) == -1 and fwd(K=0) == -1
    assert fwd(K=513) == -4 and fwd(ld=99) == -2 and fwd(logits=17) == -2 and fwd(dt=1, logits=18) == -2
    assert fwd(V=(1 << 24) + 1, ld=1 << 25) == -4
    for tau in (0.0, -1.0, float("inf"), float("nan")):
        assert fwd(tau=tau) == -4
    for cap in ((0.0, 5.0, 7.5), (23.0, 5.0, -1.0), (23.0, float("nan"), 7.5), (200.0, 0.0, 7.5), (float("inf"), 0.0, 1.0)):
        assert fwd(cap=cap) == -4, cap
    assert fwd(tau=0.1, cap=(23.0, 5.0, 7.5)) == -4
    assert lib.ngpt_distill_bwd(16, 0, 100, 16, 1, 16, None, None, 2, 100, 4, 1.0, 0.0, 0.0, 0.0, None, 16, 1, 16, 100, None) == -1
    assert lib.ngpt_distill_bwd(16, 0, 100, 16, 1, 16, None, None, 2, 100, 4, 1.0, 0.0, 0.0, 0.0, 16, 16, 1, 16, 99, None) == -2
    most = lib.ngpt_distill_fused_max_cols(0)
    assert most >= 50304
    assert lib.ngpt_distill_fwd_bwd(16, 0, most + 1, 16, 1, 16, None, None, 2, most + 1, 4, 1.0, 0.0, 0.0, 0.0, 1.0, 16, 16, most + 1, None) == -4
    assert lib.ngpt_distill_stats_bytes(10) == 160


def test_functions_check_their_arguments(amd):
    x, w = torch.zeros(4, 64, dtype=BF), torch.zeros(8, 64, dtype=BF)
    with pytest.raises(RuntimeError, match="GPU only"):
        amd.linear_act(x, w)
    with pytest.raises(AssertionError, match="activation"):
        amd.linear_act(x, w, activation="relu")
    with pytest.raises(AssertionError, match="residual"):
        amd.linear_act(x, w, residual=torch.zeros(4, 64, dtype=BF))
    with pytest.raises(AssertionError, match="bias"):
        amd.linear_act(x, w, torch.zeros(64, dtype=BF))
    with pytest.raises(AssertionError, match="bfloat16"):
        amd.linear_act(x, w, torch.zeros(8))
    with pytest.raises(AssertionError):
        amd.linear_act(x[:, :60], w)
    q, k, cos = torch.zeros(4, 2, 8), torch.zeros(4, 1, 8), torch.zeros(4, 4)
    with pytest.raises(RuntimeError, match="GPU only"):
        amd.qk_norm_rope(q, k, cos, cos)
    with pytest.raises(AssertionError, match="same tokens"):
        amd.qk_norm_rope(q, k[:3], cos, cos)
    with pytest.raises(AssertionError, match="both"):
        amd.qk_norm_rope(q, k.to(BF), cos, cos)
    with pytest.raises(AssertionError, match="positions"):
        amd.qk_norm_rope(q, k, cos, cos, torch.zeros(5, dtype=torch.int64))
    with pytest.raises(AssertionError, match="positions"):
        amd.qk_norm_rope(q, k, cos, cos, torch.zeros(4))
    with pytest.raises(AssertionError, match="weights"):
        amd.qk_norm_rope(q, k, cos, cos, None, torch.zeros(4))
    l, i, t = torch.zeros(3, 10), torch.zeros(3, 2, dtype=torch.int64), torch.zeros(3, 2)
    with pytest.raises(RuntimeError, match="GPU only"):
        amd.distill_topk(l, i, t)
    with pytest.raises(RuntimeError, match="GPU only"):
        amd.distill_topk_fwd_bwd(l, i, t)
    with pytest.raises(AssertionError, match="ids"):
        amd.distill_topk(l, i.float(), t)
    with pytest.raises(AssertionError, match="teacher"):
        amd.distill_topk(l, i, t.double())
    with pytest.raises(AssertionError, match="row_weight"):
        amd.distill_topk(l, i, t, row_weight=torch.zeros(2))
    with pytest.raises(AssertionError, match="softcap"):
        amd.distill_topk(l, i, t, softcap=(23.0, 5.0, 0.0))


def test_fake_implementations(amd):
    m = lambda *s, dtype=BF: torch.empty(*s, dtype=dtype, device="meta")
    ops = torch.ops.nanogpt
    out, pre = ops.linear_act(m(2, 5, 64), m(24, 64), m(24), m(2, 5, 24), "gelu", True)
    assert out.shape == pre.shape == (2, 5, 24)
    assert ops.linear_act(m(5, 64), m(24, 64), None, None, "none", False)[1].numel() == 0
    dx, dw, db = ops.linear_act_backward(m(5, 24), m(5, 64), m(24, 64), None, "none", True, False, True)
    assert dx.shape == (5, 64) and dw.numel() == 0 and db.shape == (24,)
    cos = m(9, 16, dtype=torch.float32)
    q, k = ops.qk_norm_rope(m(9, 4, 32), m(9, 2, 32), cos, cos, None, None, None, 1e-6, False)
    assert q.shape == (9, 4, 32) and k.shape == (9, 2, 32)
    dq, dk, dqw, dkw = ops.qk_norm_rope_backward(q, k, q, k, cos, cos, None, m(32), None, 1e-6, False, True, False)
    assert dqw.shape == (32,) and dkw.numel() == 0
    ids, t = m(3, 4, dtype=torch.int32), m(3, 4, dtype=torch.float32)
    losses, stats = ops.distill_topk(m(3, 100), ids, t, None, None, 1.0, 0.0, 0.0, 0.0)
    assert losses.shape == (3,) and losses.dtype == torch.float32 and stats.shape == (3, 4)
    losses, grad = ops.distill_topk_fwd_bwd(m(3, 100), ids, t, None, None, 1.0, 0.0, 0.0, 0.0, 1.0)
    assert grad.shape == (3, 100) and grad.dtype == BF
    # the functions take tensors of the meta device too
    assert amd.linear_act(m(2, 5, 64), m(24, 64), activation="gelu").shape == (2, 5, 24)
    assert [h.shape for h in amd.qk_norm_rope(m(9, 4, 32), m(9, 2, 32), cos, cos)] == [(9, 4, 32), (9, 2, 32)]
    assert amd.distill_topk(m(3, 100), ids, t).shape == (3,) and amd.distill_topk_fwd_bwd(m(3, 100), ids, t)[1].shape == (3, 100)


def test_autograd_wiring_under_fake_tensors(amd):
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x, w, b, r = (torch.empty(*s, dtype=BF, requires_grad=True) for s in ((6, 64), (24, 64), (24,), (6, 24)))
        y = amd.linear_act(x, w, b, r, "silu")
        q, k = amd.qk_norm_rope(y.view(6, 3, 8)[:, :2], y.view(6, 3, 8)[:, 2:], torch.empty(6, 4), torch.empty(6, 4))
        loss = amd.distill_topk(torch.cat((q, k), 1).flatten(1), torch.empty(6, 2, dtype=torch.int64), torch.empty(6, 2))
        grads = torch.autograd.grad(loss.sum(), [x, w, b, r])
        assert [g.shape for g in grads] == [t.shape for t in (x, w, b, r)]


def test_sizes_past_32_bit_offsets_are_refused(amd):
    lib = amd._lib.load()
    for M, N, K in (((1 << 29) + 1, 8, 64), (4, (1 << 21) + 1, 64), (4, 8, (1 << 21) + 1)):
        assert lib.ngpt_linear_act_fwd(16, K, 16, K, None, None, 0, M, N, K, 0, 16, None, None) == -4
        assert lib.ngpt_linear_act_bwd(16, None, 16, K, 16, K, M, N, K, 0, 16, 16, 16, 16, 1 << 60, None) == -4
        assert lib.ngpt_linear_act_bwd_workspace_bytes(M, N, K) == 0
    for ldx, ldw in ((1 << 22, 64), (64, 1 << 22)):
        assert lib.ngpt_linear_act_bwd(16, None, 16, ldx, 16, ldw, 4, 8, 64, 0, 16, 16, 16, 16, 1 << 60, None) == -4
    assert lib.ngpt_distill_fwd(16, 0, 8, 16, 0, 16, None, None, (1 << 30) + 1, 8, 2, 1.0, 0.0, 0.0, 0.0, 16, None, None) == -4

"""Calls of linear_act, qk_norm_rope and distill_topk beside the sizes of test_gpu_block.py: layouts, modes of torch, values at the edge of the
formulas.  Bounds are that file's, which count roundings."""
import pytest
import torch

from test_gpu_block import BF, D, F32, check_distill, check_linear, rnd, teacher_rows

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

"""Which layouts the block operators read in place: the binding's rule on CPU tensors, whose sizes and strides alone it looks at."""
import itertools

import pytest
import torch


@pytest.fixture(scope="module")
def rows_in_place():
    import modded_nanogpt_amd
    if not modded_nanogpt_amd._lib.BINDING_PATH.exists():
        from modded_nanogpt_amd.build import build
        build(verbose=False)
    return modded_nanogpt_amd._lib.load_torch().rows_in_place


def offsets(t):
    """where each value of t lies in its storage, as [rows, values of a row]"""
    at = torch.zeros(t.shape, dtype=torch.int64)
    for d in range(t.ndim):
        shape = [1] * t.ndim
        shape[d] = t.shape[d]
        at = at + (torch.arange(t.shape[d]) * t.stride(d)).view(shape)
    return at.reshape(-1, t.shape[-1]) if t.shape[-1] else at.reshape(0, 0)


def readable(t):
    """one start, one distance: row r is at r * distance, value by value, and no two rows overlap"""
    at = offsets(t)
    if at.numel() == 0:
        return True
    n, length = at.shape
    apart = int(at[1, 0]) if n > 1 else length
    return apart >= length and bool((at == torch.arange(n)[:, None] * apart + torch.arange(length)).all())


def test_a_single_row_of_another_stride_is_not_read_in_place(rows_in_place):
    m = torch.zeros(64, 48)
    for t in (m[:, 3], m.t()[3], m.t()[:1], m[:1, ::2], m[0, ::2], torch.zeros(1, 48, 5)[:, :, -1], torch.zeros(1, 48, 5).transpose(1, 2)[:, -1],
              torch.zeros(1).expand(48), torch.zeros(1, 1).expand(1, 48), torch.zeros(1, 1, 1).expand(1, 1, 48)):
        assert not readable(t) and not rows_in_place(t), (t.shape, t.stride())
    for t in (m[5], m[5:6], m[5:6, 7:20], m[5, 7:20], m[:1, :1], m[:, :1][3], torch.zeros(1, 5, 48)[:, -1], m[:, 3][:1], torch.zeros(1, 1).expand(1, 1)):
        assert readable(t) and rows_in_place(t), (t.shape, t.stride())


def test_what_is_read_in_place_is_where_the_kernels_look(rows_in_place):
    base, taken = torch.zeros(4 * 5 * 6 * 7), 0
    for shape in ((7,), (1,), (0,), (3, 4), (1, 4), (4, 1), (1, 1), (3, 0), (0, 3), (2, 3, 4), (1, 3, 4), (2, 1, 4), (2, 3, 1), (1, 1, 4), (2, 0, 4), (1, 3, 1)):
        for strides in itertools.product((0, 1, 2, 4, 5, 8, 12, 15, 24), repeat=len(shape)):
            t = base.as_strided(shape, strides)
            if rows_in_place(t):
                taken += 1
                assert readable(t), (shape, strides)
    assert taken > 100


def test_the_backward_of_linear_act_reserves_what_it_uses():
    import modded_nanogpt_amd
    lib = modded_nanogpt_amd._lib.load()
    M, N, K = 4096, 768, 768
    need = lambda act=0, dout=16, x=16, ldx=K, dx=1, dw=1, db=1, M=M: lib.ngpt_linear_act_bwd_workspace_bytes_for(dout, x, ldx, M, N, K, act, dx, dw, db)
    dz, wt, xc, most = 2 * M * N, 2 * N * K, 2 * M * K, lib.ngpt_linear_act_bwd_workspace_bytes(M, N, K)
    assert need(db=0, dw=0) == wt and need(dx=0, dw=0) < 2048 * 4 * N + 256          # nothing but w^T; nothing but column sums
    assert need(dx=0, dw=0, db=0) == 0
    assert need(act=1, dw=0, db=0) == dz + wt and need(dout=8, dw=0, db=0) == dz + wt
    parts = need(dx=0, db=0)                                                         # (by the device: none without one)
    assert need(dx=0, db=0, x=8) == xc + parts == need(dx=0, db=0, ldx=K + 4)
    assert need(dx=0, db=0, M=M - 1) == dz + xc + lib.ngpt_linear_act_bwd_workspace_bytes_for(16, 16, K, M, N, K, 0, 0, 1, 0)
    for act in (0, 3):
        for flags in itertools.product((0, 1), repeat=3):
            for dout, x in itertools.product((16, 2), repeat=2):
                assert need(act, dout, x, K, *flags) <= most
    assert lib.ngpt_linear_act_bwd_workspace_bytes_for(16, 16, 64, 0, 8, 64, 0, 1, 1, 1) == 0
    # what is asked for is what is refused below
    bwd = lambda nws, dx=16, dw=16, db=16: lib.ngpt_linear_act_bwd(16, None, 16, K, 16, K, M, N, K, 0, dx, dw, db, 16, nws, None)
    assert bwd(need() - 1) == -3 and bwd(need(dw=0, db=0) - 1, dw=None, db=None) == -3


def test_rows_too_far_apart_are_copied(rows_in_place):
    import modded_nanogpt_amd
    most = modded_nanogpt_amd._lib.load_torch().LINEAR_MAX_STRIDE
    t = torch.empty(3, most + 64, device="meta")
    assert rows_in_place(t[:, :64]) and not rows_in_place(t[:, :64], most) and rows_in_place(t[:1, :64], most)
    assert rows_in_place(t, most)              # contiguous: a copy would not help
    assert rows_in_place(t[:, 64:].new_empty(3, most)[:, 3:], most)


def test_dimensions_of_size_one_do_not_make_rows_uneven(rows_in_place):
    t = torch.zeros(4, 9, 6, 48)
    for v in (t[:, -1:, 0], t[:, -1:, :1], t[:, :, :1, 5:20], t[:, -1, :1], t[:1, :, :1], t[:, :, :, 3:], t[:, 0, None, 2]):
        assert readable(v) and rows_in_place(v), (v.shape, v.stride())
    for v in (t[:, :2, 0], t[:, -1:, :, 3:], t[:, :1].expand(4, 3, 6, 48), t[:, :1, :5], t.transpose(0, 1)[:, :, :1]):
        assert not rows_in_place(v), (v.shape, v.stride())


def test_distill_constants_outside_32_bit_floats_are_refused():
    import modded_nanogpt_amd
    lib = modded_nanogpt_amd._lib.load()
    call = lambda tau, cap: lib.ngpt_distill_fwd(16, 0, 100, 16, 1, 16, None, None, 2, 100, 4, tau, *cap, 0, None, None)     # (no losses: -1 once these pass)
    assert call(1.0, (0.0, 0.0, 0.0)) == -1 and call(1e-30, (0.0, 0.0, 0.0)) == -1 and call(1.0, (23.0, 5.0, 7.5)) == -1
    assert call(1e-40, (0.0, 0.0, 0.0)) == -4 and b"reciprocal" in lib.ngpt_last_error()
    assert call(1.0, (23.0, 5.0, 1e-40)) == -4 and call(1.0, (23.0, 1e38, 1e-3)) == -4 and call(1.0, (50.0, 0.0, 1e-38)) == -4

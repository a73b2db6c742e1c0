"""CPU: what the packed attention, the vocabulary loss and the many-tensor update do before anything touches a device, at the edges of
what they take."""
import pytest
import torch

from image_captioning_amd import _native as N, ops


def test_linear_ce_loss_forward_refuses():
    lib = N.load()
    good = dict(dtype=1, h=16, ldh=64, w=16, ldw=64, b=None, t=16, R=4, E=64, V=100, ign=-100, mean=1, rl=16, lse=16, loss=16, out=16, ws=16, nbytes=1 << 40)
    for kw, code in ((dict(loss=None), 1), (dict(out=None), 1), (dict(out=24), 1), (dict(ws=None), 1), (dict(R=0), 1), (dict(dtype=5), 1), (dict(V=65535 * 64 + 1), 3)):
        assert lib.icap_linear_ce_loss_fwd(*{**good, **kw}.values(), None) == code, kw


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_packed_rows_are_readable_whatever_the_layout(dtype):
    """Strides that are multiples of 16 bytes and within the limits, an aligned address, the same values; in place where that is possible."""
    per = 16 // torch.empty((), dtype=dtype).element_size()
    base = torch.arange(8 * 131 + 64).to(dtype)
    base = base[(-base.data_ptr() % 16) // base.element_size():]
    odd = base[:8 * 131].view(8, 131)[:, :128].unflatten(1, (4, 32))
    wide = base[:8 * 128].view(8, 4, 32)
    cases = [(odd, False), (odd[:3], False), (odd[:1], True), (odd[1:2], False), (odd[4:5], 4 * 131 % per == 0), (odd.split([1, 7])[0], True), (wide, True), (wide[:, 1:3], True),
             (wide[2:3, 1:2], True), (wide[:0], True), (wide.transpose(0, 1), True), (wide[:, :, ::2], False), (wide[:, :, per // 2:per // 2 + 24], False), (wide[:, :, 8:24], True),
             (base.as_strided((9, 1, 16), (16, 17, 1)), True), (base.as_strided((1, 2, 16), ((1 << 24) + 16, 16, 1)), True),
             (base.as_strided((1, 1, 16), (3, 5, 1)), True), (wide[:, :1].expand(8, 6, 32), True), (base[:1].expand(4, 2, 8), False)]
    for t, in_place in cases:
        got = ops._packed_rows(t)
        assert torch.equal(got, t) and (got.data_ptr() == t.data_ptr()) == in_place
        assert got.stride(2) == 1 and got.data_ptr() % 16 == 0 and all(x % per == 0 for x in got.stride()[:2])
        assert got.stride(0) <= 1 << 24 and got.stride(1) * got.size(1) <= 1 << 30


def test_linear_ce_workspace_for_the_tensors_of_a_call():
    """What is read where it lies takes no room, results that are not wanted take none, and nothing takes more than any call of that size."""
    ws, of = N.load().icap_linear_ce_ws_bytes, N.load().icap_linear_ce_ws_bytes_for
    at = 1 << 20
    for dtype in (0, 1, 2):
        for R, E, V in ((1, 8, 1), (3, 2048, 65536), (684, 512, 81), (4864, 512, 6756), (8192, 2048, 65536), (20000, 16, 4100)):
            for h, ld_h, w, ld_w in ((at, E, at, E), (at, E + 3, at + 2, E + 5), (at + 4, E, at, E + 64)):
                assert 0 < of(dtype, h, ld_h, w, ld_w, R, E, V, 0) <= ws(dtype, R, E, V, 0)
                every = of(dtype, h, ld_h, w, ld_w, R, E, V, 7)
                assert every <= ws(dtype, R, E, V, 1)
                for need in range(1, 7):
                    assert 0 < of(dtype, h, ld_h, w, ld_w, R, E, V, need) <= every
    # one row scored over a weight that is read where it lies: its strips; a copy of the weight alone is 268 MB
    assert of(1, at, 2048, at, 2048, 1, 2048, 65536, 0) < 1 << 14 and of(1, at, 2048, at + 2, 2048, 1, 2048, 65536, 0) > 1 << 28
    assert of(1, at, 2048, at, 2048, 8192, 2048, 65536, 7) <= of(1, at, 2048, at, 2049, 8192, 2048, 65536, 7) - (1 << 28)
    assert of(1, at, 8, at, 8, 0, 8, 8, 0) == 0
    # too small by one piece of the workspace: refused
    n = of(0, at, 64, at, 64, 4, 64, 100, 2)
    good = dict(dtype=0, h=16, ldh=64, w=16, ldw=64, b=None, t=16, R=4, E=64, V=100, ign=-100, lse=16, out=16, g=16, dh=None, dw=16, db=None, ws=16, nbytes=n - 256)
    assert N.load().icap_linear_ce_bwd(*good.values(), None) == 1
    assert N.load().icap_linear_ce_bwd(*{**good, "dw": None, "nbytes": 0, "ws": None}.values(), None) == 0          # nothing is wanted


def test_attention_refuses_more_key_heads_than_a_launch_takes():
    """One token has no stride that would bound its heads."""
    lib = N.load()
    fwd = dict(dtype=1, q=16, k=16, v=16, out=16, lse=None, cu_q=4, cu_k=4, seqs=1, tq=1, tk=1, h=(1 << 23) + 1, kv=(1 << 23) + 1, d=8, qt=0, qh=8, kt=0, kh=8, vt=0, vh=8,
               scale=0.1, causal=1, ws=None, nbytes=0)
    assert lib.icap_attention_packed_fwd(*fwd.values(), None) == 3 and b"key heads" in lib.icap_last_error()
    bwd = dict(dtype=1, dout=16, q=16, k=16, v=16, out=16, lse=16, dq=16, dk=16, dv=16, cu_q=4, cu_k=4, seqs=1, tq=1, tk=1, h=1 << 24, kv=1 << 24, d=8, gt=0, gh=8,
               qt=0, qh=8, kt=0, kh=8, vt=0, vh=8, scale=0.1, causal=1, ws=16)
    assert lib.icap_attention_packed_bwd(*bwd.values(), None) == 3

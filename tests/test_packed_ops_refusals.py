"""CPU: what the packed attention, the vocabulary loss and the many-tensor update refuse, and the sizes their entry points give,
before anything touches a device."""
import ctypes as C

import pytest
import torch

from image_captioning_amd import _native as N, ops, train_ops as T, training


def attn_fwd(**kw):
    a = dict(dtype=1, q=16, k=16, v=16, out=16, lse=None, cu_q=4, cu_k=4, seqs=2, tq=8, tk=8, h=4, kv=2, d=64, qt=256, qh=64, kt=128, kh=64, vt=128, vh=64,
             scale=0.1, causal=1, ws=None, nbytes=0)
    a.update(kw)
    return N.load().icap_attention_packed_fwd(*a.values(), None), N.load().icap_last_error().decode()


@pytest.mark.parametrize("kw,code", [(dict(dtype=3), 1), (dict(dtype=-1), 1), (dict(q=None), 1), (dict(v=None), 1), (dict(cu_q=None), 1), (dict(seqs=0), 1),
                                     (dict(h=5), 1), (dict(kv=0), 1), (dict(tq=-1), 1), (dict(out=None), 1), (dict(d=0), 1), (dict(d=136), 3), (dict(d=60), 3),
                                     (dict(scale=0.0), 1), (dict(scale=-1.0), 1), (dict(scale=float("nan")), 1), (dict(k=24), 2), (dict(qt=252), 2), (dict(vh=68), 2), (dict(tq=1 << 29), 3), (dict(out=24), 1),
                                     (dict(seqs=1, tq=1, tk=4096, h=8, kv=8), 1)])      # the last one: split keys without a workspace
def test_attention_forward_refuses(kw, code):
    rc, msg = attn_fwd(**kw)
    assert rc == code and msg


def test_attention_forward_of_nothing_is_fine():
    assert attn_fwd(tq=0, q=None, out=None)[0] == 0


def test_attention_backward_refuses():
    lib = N.load()
    good = dict(dtype=0, dout=16, q=16, k=16, v=16, out=16, lse=16, dq=16, dk=16, dv=16, cu_q=4, cu_k=4, seqs=2, tq=8, tk=8, h=4, kv=2, d=32, gt=128, gh=32,
                qt=128, qh=32, kt=64, kh=32, vt=64, vh=32, scale=0.1, causal=1, ws=16)
    for kw, code in ((dict(dout=None), 1), (dict(lse=None), 1), (dict(dk=None), 1), (dict(ws=None), 1), (dict(dq=20), 2), (dict(gt=126), 2), (dict(h=3), 1), (dict(d=12), 3)):
        assert lib.icap_attention_packed_bwd(*{**good, **kw}.values(), None) == code, kw


def test_attention_workspace():
    ws = N.load().icap_attention_packed_ws_bytes
    assert ws(8, 8 * 300, 8 * 300, 8, 8, 64) == 0                       # prompts: no split
    one = ws(1, 1, 8192, 8, 8, 64)                                      # one new token over a long cache
    assert one > 0 and one % (8 * 65 * 4) == 0 and 1 < one // (8 * 65 * 4) <= 32
    assert ws(4096, 4096, 4096 * 512, 8, 8, 64) == 0                    # enough sequences to fill the card
    assert ws(1, 1, 100, 8, 8, 64) == 0 and ws(0, 1, 1, 1, 1, 8) == 0


def ce_fwd(**kw):
    a = dict(dtype=1, h=16, ldh=64, w=16, ldw=64, b=None, t=16, R=4, E=64, V=100, ign=-100, mean=1, rl=16, lse=16, out=16, ws=16, nbytes=1 << 40)
    a.update(kw)
    return N.load().icap_linear_ce_fwd(*a.values(), None)


@pytest.mark.parametrize("kw,code", [(dict(dtype=7), 1), (dict(h=None), 1), (dict(t=None), 1), (dict(R=0), 1), (dict(V=0), 1), (dict(ldh=63), 1), (dict(ldw=10), 1),
                                     (dict(ws=None), 1), (dict(ws=24), 1), (dict(nbytes=8), 1), (dict(lse=None), 1), (dict(R=65535 * 64 + 1), 3), (dict(V=65535 * 64 + 1), 3),
                                     (dict(E=(1 << 20) + 1, ldh=1 << 21, ldw=1 << 21), 3), (dict(R=1 << 22, V=1 << 21), 3), (dict(R=1 << 22, E=1 << 20, ldh=1 << 20, ldw=1 << 20), 3)])
def test_linear_ce_forward_refuses(kw, code):
    assert ce_fwd(**kw) == code


def test_linear_ce_backward_refuses():
    lib = N.load()
    good = dict(dtype=0, h=16, ldh=64, w=16, ldw=64, b=None, t=16, R=4, E=64, V=100, ign=-100, lse=16, out=16, g=16, dh=16, dw=16, db=None, ws=16, nbytes=1 << 40)
    for kw, code in ((dict(g=None), 1), (dict(lse=None), 1), (dict(nbytes=0), 1), (dict(dh=20), 2), (dict(dw=4), 2), (dict(E=0), 1)):
        assert lib.icap_linear_ce_bwd(*{**good, **kw}.values(), None) == code, kw


def test_linear_ce_workspace_is_bounded():
    ws = N.load().icap_linear_ce_ws_bytes
    for dtype, size in ((0, 4), (1, 2), (2, 2)):
        for R, E, V in ((1, 8, 1), (684, 512, 81), (8192, 1024, 65536), (65536, 512, 131072)):
            assert ws(dtype, R, E, V, 0) > 0
            # copies of hidden and weight (twice: rows and transposed), pieces, fp32 partial results, the bias gradient's
            rows = -(-R // 128) * 128
            most = (1 << 29) + 2 * size * ((rows + 64) * (E + 64) + (V + 64) * (E + 64)) + 4 * 33 * rows * E + 4 * 32 * min(V, 70000) * E // 16 + 8 * V * (rows // 128 + 1) + (1 << 20)
            assert ws(dtype, R, E, V, 1) < most
    # the logits of this call in fp32 alone would take 32 GiB
    assert ws(1, 65536, 512, 131072, 1) < 5 << 30
    assert ws(1, 0, 8, 8, 0) == 0


def test_adamw_tensors_refuses():
    lib = N.load()
    one, n, st, ix = (C.c_void_p * 1)(16), (C.c_longlong * 1)(4), (C.c_int * 1)(1), (C.c_int * 1)(0)

    def call(count=1, p=one, g=one, m=one, v=one, ms=None, vs=None, n=n, st=st, ix=ix, pd=0, gd=0, bits=32, step_dev=None):
        return lib.icap_adamw_tensors(count, p, g, m, v, ms, vs, n, st, ix, pd, gd, bits, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1.0, 0, step_dev, None)
    assert call(count=-1) == 1 and call(p=None) == 1 and call(bits=16) == 1 and call(pd=3) == 1 and call(pd=0, gd=1) == 1 and call(pd=1, gd=2) == 1
    assert call(bits=8) == 1                                            # 8-bit states without scales
    assert call(p=(C.c_void_p * 1)(None)) == 1 and call(n=(C.c_longlong * 1)(-1)) == 1 and call(n=(C.c_longlong * 1)((1 << 40) + 1)) == 3
    assert call(st=(C.c_int * 1)(0)) == 1 and call(ix=(C.c_int * 1)(1 << 20)) == 1
    assert call(count=0, p=None, g=None, m=None, v=None, n=None, st=None, ix=None) == 0


def test_tensors_off_the_device_are_refused():
    q, cu = torch.zeros(4, 2, 16), torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(N.IcapError, match="no CPU fallback"):
        ops.attention_packed(q, q, q, cu)
    with pytest.raises(N.IcapError, match="no CPU fallback"):
        T.attention_packed_bwd(q, q, q, q, q, torch.zeros(4, 2), cu)
    with pytest.raises(N.IcapError, match="no CPU fallback"):
        training.packed_attention(q.requires_grad_(), q, q, cu)
    h, w, t = torch.zeros(4, 8), torch.zeros(10, 8), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(N.IcapError, match="no CPU fallback"):
        training.linear_cross_entropy(h, w, None, t)
    with pytest.raises(N.IcapError, match="do not belong together"):
        training.linear_cross_entropy(h, w, None, t[:3])
    with pytest.raises(N.IcapError, match="no CPU fallback"):
        T.adamw_tensors([h], [h], [h], [h], step=1, lr=1e-3)
    with pytest.raises(N.IcapError, match="as many gradients"):
        T.adamw_tensors([h], [], [h], [h], step=1, lr=1e-3)
    with pytest.raises(N.IcapError, match="HIP device"):
        training.AdamWTensors([torch.nn.Parameter(h)])
    with pytest.raises(ValueError, match="8 or 32"):
        training.AdamWTensors([torch.nn.Parameter(h)], state_bits=16)

"""CPU: what the packed attention, the vocabulary loss and the many-tensor update do before anything touches a device, at the edges of
what they take."""
from image_captioning_amd import _native as N


def test_linear_ce_loss_forward_refuses():
    lib = N.load()
    good = dict(dtype=1, h=16, ldh=64, w=16, ldw=64, b=None, t=16, R=4, E=64, V=100, ign=-100, mean=1, rl=16, lse=16, loss=16, out=16, ws=16, nbytes=1 << 40)
    for kw, code in ((dict(loss=None), 1), (dict(out=None), 1), (dict(out=24), 1), (dict(ws=None), 1), (dict(R=0), 1), (dict(dtype=5), 1), (dict(V=65535 * 64 + 1), 3)):
        assert lib.icap_linear_ce_loss_fwd(*{**good, **kw}.values(), None) == code, kw

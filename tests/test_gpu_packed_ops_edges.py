"""GPU: calls of the packed attention, the vocabulary loss and the many-tensor AdamW at the edges of what they take: sizes of one with odd
strides, losses changed in place, gradients far from 1, words of small probability, memory that a call takes."""
import pytest
import torch

from .test_gpu_packed_ops import D, E24, rnd, within

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ words of small probability
def rare_words(R, E, V, lowest, oracle, outlier=1.0):
    """fp32: half of the words are never a target and have probabilities down to exp(lowest) and below.  dweight's rows, each held to a
    bound that is relative to that row's own terms; dhidden and dbias likewise."""
    from image_captioning_amd import train_ops as T
    h, w = rnd(R, E, seed=1), rnd(V, E, seed=2, scale=E ** -0.5)
    h[:, E // 2] *= outlier
    w[:, E // 3] *= outlier
    b = rnd(V, seed=3, scale=0.5)
    b[V // 2:] += torch.linspace(-5.0, lowest, V - V // 2)
    t = torch.randint(0, V // 2, (R,), generator=torch.Generator().manual_seed(4))
    if R > 1:
        t[::5] = -100
    hd, wd, bd, td = (x.to(oracle) for x in (h.double(), w.double(), b.double(), t))
    x = hd @ wd.t() + bd
    A = hd.abs() @ wd.abs().t()
    # two fp16 parts of each operand (2^-22, and 2^-39 of its row's largest value), low products dropped, fp32 sums
    dx = (3 * 2.0 ** -22 + (3 * E + 8) * E24) * A + 4 * E24 * x.abs() + 2.0 ** -38 * (
        hd.abs().amax(1, keepdim=True) * wd.abs().sum(1) + wd.abs().amax(1) * hd.abs().sum(1, keepdim=True))
    lse = torch.logsumexp(x, 1, keepdim=True)
    e_lse = dx.amax(1, keepdim=True) + (V / 64 + 80) * E24 + 4 * E24 * lse.abs()
    on = ((td >= 0) & (td < V))[:, None]
    P = torch.exp(x - lse) * on
    hot = torch.zeros_like(P).scatter_(1, td.clamp(min=0)[:, None], 1.0) * on
    d = P - hot
    e_plain = P * (dx + e_lse + (lse - x).abs() * 3 * E24 + 2.0 ** -21)
    # D as two fp16 values: 22 bits of each value, or as many below the largest of its word
    ed = e_plain + d.abs() * 2.0 ** -22 + 2.0 ** -38 * d.abs().amax(0)
    sc = 1.0 / int(on.sum())

    def bound(a, ea, m, terms, y):
        return sc * (ea @ m.abs() + ((3 * terms + 48) * E24 + 3 * 2.0 ** -22) * (a.abs() @ m.abs())) * 1.01 + 5 * E24 * y.abs() + 1e-44
    dw, db, dh = sc * d.t() @ hd, sc * d.sum(0), sc * d @ wd
    e_dw = bound(d.t(), ed.t(), hd, R, dw) + sc * 2.0 ** -38 * float(hd.abs().max()) * d.abs().sum(0)[:, None]
    e_db = sc * (e_plain.sum(0) + (R + 8) * E24 * d.abs().sum(0)) * 1.01 + 5 * E24 * db.abs() + 1e-44
    # dhidden sums over words: a row is held to its own terms and to 2^-38 of the largest weight for every word
    e_dh = bound(d, ed, wd, V, dh) + sc * V * 2.0 ** -38 * float(wd.abs().max())
    _, _, saved = T.linear_ce_fwd(h.to(D), w.to(D), b.to(D), t.to(D), -100, True)
    got = T.linear_ce_bwd(torch.ones(1, device=D), saved)
    for name, g, y, e in zip(("dh", "dw", "db"), got, (dh, dw, db), (e_dh, e_dw, e_db)):
        within(g, y.cpu(), e.cpu(), name)
    return saved, got


@pytest.mark.parametrize("R,E,V,lowest", [(600, 64, 300, -25.0), (600, 64, 300, -60.0), (1, 8, 10, -30.0), (70, 40, 1000, -30.0), (3300, 64, 4100, -30.0), (40, 4160, 100, -30.0)])
def test_linear_ce_gradients_of_rare_words(R, E, V, lowest):
    rare_words(R, E, V, lowest, "cpu")


def test_linear_ce_gradients_of_rare_words_with_outlying_features():
    """One feature of hidden, and another of the weight, is two hundred times the others."""
    rare_words(300, 512, 200, -30.0, "cpu", outlier=200.0)


def test_linear_ce_gradients_of_rare_words_in_several_pieces():
    from image_captioning_amd import _native as N
    R, E, V = 20000, 16, 4100
    assert N.load().icap_linear_ce_ws_bytes(0, R, E, V, 1) < 4 * R * V
    rare_words(R, E, V, -30.0, D)


def test_linear_ce_gradients_of_rare_words_one_at_a_time():
    """dweight without the others is the same; dhidden alone is within its bound (its words then need no factors)."""
    from image_captioning_amd import train_ops as T
    saved, (dh, dw, db) = rare_words(257, 72, 400, -30.0, "cpu")
    one = torch.ones(1, device=D)
    assert torch.equal(T.linear_ce_bwd(one, saved, need=(False, True, False))[1], dw)
    assert torch.equal(T.linear_ce_bwd(one, saved, need=(False, False, True))[2], db)
    alone = T.linear_ce_bwd(one, saved, need=(True, False, False))[0]
    # two sums of the same products: 3 V roundings of fp32 each, and 22 bits of every operand
    size = float((saved[1].abs().max(0)[0]).max()) / 200
    assert float((alone - dh).abs().max()) <= 2 * (3 * 400 * E24 + 2.0 ** -20) * size

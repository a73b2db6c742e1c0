"""GPU: calls of the packed attention, the vocabulary loss and the many-tensor AdamW at the edges of what they take: sizes of one with odd
strides, losses changed in place, gradients far from 1, words of small probability, memory that a call takes."""
import math

import pytest
import torch

from .test_gpu_packed_ops import BF16, D, E24, F16, F32, TYPES, half_step, offsets, rnd, within

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


# ------------------------------------------------------------------------------------------------ gradients far from 1
def backward_oracle(q, k, v, g, out, lse, causal, scale):
    """The backward formula in 64 bits from the forward call's own results (their rounding is not the backward call's), one text.
    Bounds: P rounded once, 16 bits of each dS, fp32 sums; nothing that grows with the text but the sums' own roundings."""
    u = half_step(q.dtype)
    up, uds = (0.0, 0.0) if q.dtype == F32 else (u, 2.0 ** -16)
    tiny = 2.0 ** -25 if q.dtype == F16 else 0.0
    n, H, dim = q.shape
    K = k.shape[1]
    r = {"dq": torch.zeros(q.shape, dtype=torch.float64), "dk": torch.zeros(k.shape, dtype=torch.float64), "dv": torch.zeros(k.shape, dtype=torch.float64)}
    b = {m: torch.zeros_like(x) for m, x in r.items()}
    q, k, v, g, out, lse = (x.double() for x in (q, k, v, g, out, lse))
    for h in range(H):
        c = h // (H // K)
        Q, KK, V, G, O = q[:, h], k[:, c], v[:, c], g[:, h], out[:, h]
        s = scale * Q @ KK.t()
        P = torch.exp(s - lse[:, h:h + 1])
        if causal:
            P = P.tril()
        e_s = float(scale * (dim + 8) * E24 * (Q.abs() @ KK.abs().t()).max()) + 2.0 ** -21 + 4 * E24 * float(lse[:, h].abs().max())
        dS = P * (G @ V.t() - (G * O).sum(1, keepdim=True))
        E = (uds + 3 * e_s + 4 * E24) * dS.abs() + P * (dim + 8) * E24 * (G.abs() @ V.abs().t() + (G.abs() * O.abs()).sum(1, keepdim=True))
        f = (n + 16) * E24
        r["dq"][:, h] = scale * dS @ KK
        b["dq"][:, h] = scale * ((E + f * dS.abs() + 2.0 ** -32 * dS.abs().amax(1, keepdim=True)) @ KK.abs()) * 1.01
        f = (n * (H // K) + 16) * E24
        r["dk"][:, c] += scale * dS.t() @ Q
        b["dk"][:, c] += scale * ((E + f * dS.abs() + 2.0 ** -32 * dS.abs().amax(0)).t() @ Q.abs()) * 1.01
        r["dv"][:, c] += P.t() @ G
        # weights of fp16 keep their 11 bits down to 2^-28
        b["dv"][:, c] += ((up + f + 3 * e_s) * P + (2.0 ** -39 if tiny else 0.0)).t() @ G.abs() * 1.01
    return {m: (r[m], b[m] + u * r[m].abs() * (1 + 2.0 ** -6) + tiny * 1.01 + 1e-30) for m in r}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,causal", [(1500, False), (1500, True), (70, True), (4096, False)])
@pytest.mark.parametrize("size", [1e-3, 1.0])
def test_attention_gradients_of_small_weights(dtype, n, causal, size):
    """Attention spread over a long text, and small output gradients: every weight, and every dS, is far below 1."""
    from image_captioning_amd import ops, train_ops as T
    H, K, dim = (2, 1, 64) if n < 4000 else (1, 1, 32)
    q, k, v, g = (rnd(n, h, dim, seed=s, scale=c, dtype=dtype) for h, s, c in ((H, 1, 0.5), (K, 2, 0.5), (K, 3, 1.0), (H, 4, size)))
    dev, cu = [x.to(D) for x in (q, k, v)], offsets([n]).to(D)
    out, lse = ops.attention_packed(*dev, cu, causal=causal, want_lse=True)
    got = T.attention_packed_bwd(g.to(D), *dev, out, lse, cu, causal=causal)
    want = backward_oracle(q, k, v, g, out.cpu(), lse.cpu(), causal, dim ** -0.5)
    for name, x in zip(("dq", "dk", "dv"), got):
        within(x, *want[name], name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [70, 1100])
def test_attention_gradients_of_large_values(dtype, n):
    """A large loss scale: dS passes fp16's largest value, the gradients do not."""
    from image_captioning_amd import ops, train_ops as T
    q, k, v, g = (rnd(n, 2, 64, seed=s, scale=c, dtype=dtype) for s, c in ((1, 0.02), (2, 0.02), (3, 4.0), (4, 8e3)))
    dev, cu = [x.to(D) for x in (q, k, v)], offsets([n]).to(D)
    out, lse = ops.attention_packed(*dev, cu, want_lse=True)
    got = T.attention_packed_bwd(g.to(D), *dev, out, lse, cu)
    want = backward_oracle(q, k, v, g, out.cpu(), lse.cpu(), True, 0.125)
    dP = g[:, 0].double() @ v[:, 0].double().t()
    assert float((dP / torch.arange(1, n + 1, dtype=torch.float64)[:, None]).tril().abs().max()) > 65504
    assert max(float(w.abs().max()) for w, _ in want.values()) < 65504
    for name, x in zip(("dq", "dk", "dv"), got):
        within(x, *want[name], name)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_gradients_that_grow_along_a_text(dtype):
    """Output gradients from 1e-6 to 1e3 within one text, and rows that are zeros: what a row or key adds up spans the whole range."""
    from image_captioning_amd import ops, train_ops as T
    n = 700
    q, k, v, g = (rnd(n, 2, 64, seed=s, scale=c, dtype=F32) for s, c in ((1, 0.3), (2, 0.3), (3, 1.0), (4, 1.0)))
    g = g * torch.logspace(-6, 3, n)[:, None, None]
    g[::50] = 0.0
    for order in (torch.arange(n), torch.arange(n - 1, -1, -1)):
        x = [t[order].to(dtype) if i == 3 else t.to(dtype) for i, t in enumerate((q, k, v, g))]
        dev, cu = [t.to(D) for t in x[:3]], offsets([n]).to(D)
        out, lse = ops.attention_packed(*dev, cu, want_lse=True)
        got = T.attention_packed_bwd(x[3].to(D), *dev, out, lse, cu)
        want = backward_oracle(*x, out.cpu(), lse.cpu(), True, 0.125)
        for name, y in zip(("dq", "dk", "dv"), got):
            within(y, *want[name], name)


# ------------------------------------------------------------------------------------------------ keys that are hardly seen
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [40, 512, 1500])
def test_attention_gradients_of_keys_that_are_hardly_seen(dtype, n):
    """Weights down to some 1e-10, in every row, and output gradients of 100: these keys' values get all of their small gradient."""
    from image_captioning_amd import ops, train_ops as T
    q, k, v, g = (rnd(n, 2, 64, seed=s, scale=c, dtype=dtype) for s, c in ((1, 0.3), (2, 0.3), (3, 1.0), (4, 100.0)))
    q[:, :, 0] = 4.0
    k[3::7, :, 0] = -8.0
    k[4::7, :, 0] = -16.0
    k[5::7, :, 0] = -26.0
    dev, cu = [x.to(D) for x in (q, k, v)], offsets([n]).to(D)
    out, lse = ops.attention_packed(*dev, cu, causal=False, want_lse=True)
    got = T.attention_packed_bwd(g.to(D), *dev, out, lse, cu, causal=False)
    want = backward_oracle(q, k, v, g, out.cpu(), lse.cpu(), False, 0.125)
    for name, x in zip(("dq", "dk", "dv"), got):
        within(x, *want[name], name)


# ------------------------------------------------------------------------------------------------ large values of keys that are hardly seen
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [40, 700])
def test_attention_of_large_values_that_are_hardly_seen(dtype, n):
    """Weights of some 1e-7 of values of 6e4: what they add to a row is far above a rounding of it."""
    from image_captioning_amd import ops
    q, k, v = (rnd(n, 2, 64, seed=s, scale=c, dtype=dtype) for s, c in ((1, 0.1), (2, 0.1), (3, 0.01)))
    q[:, :, 0] = 4.0
    k[3::7, :, 0] = torch.linspace(-24.0, -32.0, len(k[3::7]))[:, None].to(dtype)
    v[3::7] = 6e4
    for causal in (False, True):
        cu = offsets([n]).to(D)
        out, lse = ops.attention_packed(*(x.to(D) for x in (q, k, v)), cu, causal=causal, want_lse=True)
        u = half_step(dtype)
        for h in range(2):
            Q, KK, V = (x[:, h].double() for x in (q, k, v))
            s = 0.125 * Q @ KK.t()
            if causal:
                s = s.masked_fill(torch.ones(n, n, dtype=torch.bool).triu(1), -math.inf)
            want = torch.logsumexp(s, 1)
            P = torch.exp(s - want[:, None])
            e_s = float(0.125 * 72 * E24 * (Q.abs() @ KK.abs().t()).max()) + 2.0 ** -21
            # each weight rounded once, and no further than 2^-32 of the row's largest
            bound = ((0.0 if dtype == F32 else u) + (n + 16) * E24 + 3 * e_s) * (P @ V.abs()) + (2.0 ** -32 * V.abs().sum(0) if dtype == F16 else 0.0)
            within(out[:, h], P @ V, bound + u * (P @ V).abs() * (1 + 2.0 ** -6) + (2.0 ** -25 if dtype == F16 else 0.0) + 1e-30, "out")
            within(lse[:, h], want, 2 * e_s + 4 * E24 * want.abs() + (n + 16) * E24, "lse")


# ------------------------------------------------------------------------------------------------ the graph knows of the update
@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_tensors_tells_autograd_that_parameters_changed(bits):
    """A graph kept across a step holds values that are no longer there: its backward pass is refused, as after torch's optimizers."""
    from image_captioning_amd import training
    w, left = (torch.nn.Parameter(rnd(8, 64, seed=s).to(D)) for s in (1, 2))
    opt = training.AdamWTensors([w, left], lr=1e-2, state_bits=bits)
    h, t = rnd(5, 64, seed=3).to(D), torch.tensor([0, 1, 2, 3, 4], device=D)
    kept, other = training.linear_cross_entropy(h, w, None, t), (left * left).sum()
    w.grad = torch.ones_like(w)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept.backward()
    other.backward()                                         # it had no gradient and was left alone
    kept = training.linear_cross_entropy(h, w, None, t)
    opt.advance_recorded(1)                                  # a replay has written the parameters
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept.backward()


# ------------------------------------------------------------------------------------------------ the loss as a tensor of its own
@pytest.mark.parametrize("dtype", TYPES)
def test_linear_cross_entropy_changed_in_place(dtype):
    """loss /= steps, loss *= and loss += before the backward pass, as accumulation loops write them."""
    from image_captioning_amd import training
    h, w = rnd(30, 64, seed=1, dtype=dtype).to(D).requires_grad_(), rnd(90, 64, seed=2, scale=0.2, dtype=dtype).to(D).requires_grad_()
    t = torch.randint(0, 90, (30,), generator=torch.Generator().manual_seed(3)).to(D)
    want = torch.autograd.grad(training.linear_cross_entropy(h, w, None, t) * 0.25, (h, w))
    value = training.linear_cross_entropy(h, w, None, t)
    before = float(value.detach())
    value /= 4
    value += 1.0
    value -= 1.0
    assert abs(float(value.detach()) - before / 4) <= 4 * E24 * (before + 1)
    for x, y in zip(torch.autograd.grad(value, (h, w)), want):
        assert torch.equal(x, y)
    # what a training loop collects keeps one value alive, not what the backward call reads
    assert training.linear_cross_entropy(h, w, None, t).detach().untyped_storage().nbytes() <= 64


def test_loss_on_stored_logits_changed_in_place():
    from image_captioning_amd import training
    x = rnd(6, 5, 40, seed=1).to(D).requires_grad_()
    t = torch.randint(0, 40, (6, 5), generator=torch.Generator().manual_seed(3)).to(D)
    for loss in (lambda: training.compute_loss(x, t, 0), lambda: training.CrossEntropyLoss(ignore_index=0)(x.reshape(-1, 40), t.reshape(-1))):
        want, = torch.autograd.grad(loss() * 0.25, x)
        value = loss()
        value /= 4
        got, = torch.autograd.grad(value, x)
        assert torch.equal(got, want)


# ------------------------------------------------------------------------------------------------ strides of axes of size one
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("at", [slice(0, 1), slice(1, 2), slice(7, 8)])
def test_attention_of_one_token_of_an_odd_projection(dtype, at):
    """One token sliced from rows of an odd width: its token stride is no multiple of 16 bytes, and belongs to an axis of size 1."""
    from image_captioning_amd import ops, train_ops as T
    H, K, dim = 4, 2, 32
    buf = rnd(8, (H + 2 * K) * dim + 3, seed=1, dtype=dtype).to(D)
    q, k, v = (t.unflatten(1, (-1, dim)) for t in buf[:, :(H + 2 * K) * dim].split((H * dim, K * dim, K * dim), 1))
    g = rnd(8, H * dim + 5, seed=2, dtype=dtype).to(D)[:, :H * dim].unflatten(1, (H, dim))
    one, all8 = offsets([1]).to(D), offsets([8]).to(D)
    for args, cu in (((q[at], k[at], v[at]), (one, one)), ((q[at], k, v), (one, all8))):
        dense = [torch.empty(t.shape, device=D, dtype=dtype).copy_(t) for t in args]
        got, want = ops.attention_packed(*args, *cu, want_lse=True), ops.attention_packed(*dense, *cu, want_lse=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        for x, y in zip(T.attention_packed_bwd(g[at], *args, *got, *cu), T.attention_packed_bwd(g[at].clone(memory_format=torch.contiguous_format), *dense, *want, *cu)):
            assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_of_one_head_and_of_rows_far_apart(dtype):
    """One key head of a tensor with an odd head stride; the last token of a text whose rows lie further apart than a stride may be."""
    from image_captioning_amd import ops
    dim, n = 16, 9
    heads = rnd(n * dim + 8, seed=3, dtype=dtype).to(D)
    q = heads.as_strided((n, 1, dim), (dim, dim + 1, 1))
    cu = offsets([n]).to(D)
    dense = torch.empty(q.shape, device=D, dtype=dtype).copy_(q)
    assert torch.equal(ops.attention_packed(q, q, q, cu), ops.attention_packed(dense, dense, dense, cu))
    far = rnd(dim, seed=4, dtype=dtype).to(D).as_strided((1, 1, dim), ((1 << 24) + 16, dim, 1))
    one = offsets([1]).to(D)
    dense = torch.empty(far.shape, device=D, dtype=dtype).copy_(far)
    assert torch.equal(ops.attention_packed(far, far, far, one), ops.attention_packed(dense, dense, dense, one))


# ------------------------------------------------------------------------------------------------ memory of the loss
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_linear_ce_takes_no_memory_for_copies_that_it_does_not_make(dtype):
    """A weight that is read where it lies is not allocated again: one row scored over it takes kilobytes."""
    from image_captioning_amd import train_ops as T
    V, E = 65536, 1024
    w = torch.zeros(V, E, device=D, dtype=dtype)
    h, t = torch.zeros(3, E, device=D, dtype=dtype), torch.tensor([5, 0, V - 1], device=D)
    T.linear_ce_fwd(h, w, None, t, want_grad=False)
    torch.cuda.synchronize()
    used = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    value, _, saved = T.linear_ce_fwd(h, w, None, t)
    assert torch.cuda.max_memory_allocated() - used < 1 << 20
    assert abs(float(value) - math.log(V)) < 1e-5
    used = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    dh, _, _ = T.linear_ce_bwd(torch.ones(1, device=D), saved, need=(True, False, False))
    # D of 64 rows (8 MB), partial results of dhidden; no copy of the weight (128 MB)
    assert torch.cuda.max_memory_allocated() - used < 32 << 20
    assert not dh.any()


# ------------------------------------------------------------------------------------------------ offsets that pass 32 bits
def test_linear_ce_hidden_gradient_over_more_than_2_31_elements():
    """dhidden sums over a weight of 2.2e9 elements: every word's row is found, the last ones among them."""
    from image_captioning_amd import train_ops as T
    R, E, V = 6, 8192, 268500
    h = rnd(R, E, seed=1, dtype=BF16).to(D)
    w = torch.empty(V, E, device=D, dtype=BF16)
    for i, rows in enumerate(w.split(65536)):
        rows.copy_(torch.randn(rows.shape, device=D, generator=torch.Generator(D).manual_seed(i)).mul_(2.0 * E ** -0.5))
    t = torch.tensor([0, V - 1, 140000, V // 2, V - 2, 262145], device=D)
    _, _, saved = T.linear_ce_fwd(h, w, None, t, -100, True)
    dh = T.linear_ce_bwd(torch.ones(1, device=D), saved, need=(True, False, False))[0]
    x = torch.cat([h.double() @ rows.double().t() for rows in w.split(32768)], 1)
    e = 2 * E * E24 * float(max((h.double().abs() @ rows.double().abs().t()).max() for rows in w.split(32768))) + 2.0 ** -20
    d = torch.exp(x - torch.logsumexp(x, 1, keepdim=True))
    size = d.clone()                                         # what is off: the exponentials, and D's one rounding
    d[torch.arange(R), t] -= 1.0
    size = 2 * e * size + 2.0 ** -8 * d.abs()
    want = sum(c @ rows.double() for c, rows in zip(d.split(32768, 1), w.split(32768))) / R
    bound = sum((c + (V + 48) * E24 * a.abs()) @ rows.double().abs() for c, a, rows in zip(size.split(32768, 1), d.split(32768, 1), w.split(32768))) / R
    within(dh, want.cpu(), (bound * 1.01 + 2.0 ** -8 * want.abs()).cpu(), "dh")
    # a target's row that is missing changes every value by some |want|.  The bound is mostly 2 e, 2 E 2^-24 sum |h| |w| = 2 * 8192 * 2^-24 * 115 = 0.11
    # twice, of the terms' sum, which is near |want|: 0.2 to 0.4
    assert float((bound / want.abs().clamp(min=1e-30)).median()) < 0.5


# ------------------------------------------------------------------------------------------------ tensors as programs have them
def test_linear_cross_entropy_of_rows_that_share_memory_and_of_turned_weights():
    from image_captioning_amd import training
    h, w = rnd(1, 64, seed=1).to(D).requires_grad_(), rnd(64, 90, seed=2, scale=0.2).to(D).requires_grad_()
    t = torch.randint(0, 90, (40,), generator=torch.Generator().manual_seed(3)).to(D)
    got = torch.autograd.grad(training.linear_cross_entropy(h.expand(40, 64), w.t(), None, t), (h, w))
    want = torch.autograd.grad(training.linear_cross_entropy(h.repeat(40, 1), w.t().contiguous(), None, t), (h, w))
    for x, y in zip(got, want):
        assert torch.equal(x, y)


# ------------------------------------------------------------------------------------------------ types of one program
def test_linear_cross_entropy_under_autocast():
    """hidden in 16 bits from an autocast layer, weight and bias in fp32: taken as nn.Linear takes them; gradients reach the fp32 leaves."""
    from image_captioning_amd import _native as N, training
    h, w, b = rnd(40, 64, seed=1).to(D).requires_grad_(), rnd(90, 64, seed=2, scale=0.2).to(D).requires_grad_(), rnd(90, seed=3).to(D).requires_grad_()
    t = torch.randint(0, 90, (40,), generator=torch.Generator().manual_seed(3)).to(D)
    for dtype in (BF16, F16):
        with torch.autocast("cuda", dtype=dtype):
            value = training.linear_cross_entropy(h.to(dtype), w, b, t)
        want = training.linear_cross_entropy(h.to(dtype), w.to(dtype), b.to(dtype), t)
        assert torch.equal(value.detach(), want.detach())
        for x, y in zip(torch.autograd.grad(value, (h, w, b)), torch.autograd.grad(want, (h, w, b))):
            assert x.dtype == F32 and torch.equal(x, y)
    with pytest.raises(N.IcapError):
        training.linear_cross_entropy(h.to(BF16), w, b, t)


# ------------------------------------------------------------------------------------------------ recorded, and two at once
@pytest.mark.parametrize("dtype", [F32, F16])
def test_captured_gradients_replay_with_new_inputs(dtype):
    """Loss and attention with their gradients in a HIP graph, replayed with inputs whose sizes differ by powers of ten, eager work between."""
    from image_captioning_amd import ops, train_ops as T
    H, dim, V, lens = 4, 32, 301, [9, 40, 15]
    n, E = sum(lens), H * dim
    cu = offsets(lens).to(D)
    w, b = rnd(V, E, seed=100, scale=E ** -0.5, dtype=dtype).to(D), (rnd(V, seed=101) - torch.linspace(0, 20, V)).to(dtype).to(D)

    def inputs(i):
        return rnd(n, 3 * H, dim, seed=i, dtype=dtype).to(D), torch.randint(0, 100, (n,), generator=torch.Generator().manual_seed(i)).to(D), torch.full((1,), 10.0 ** (2 * i - 3), device=D)

    def step(x, t, g):
        q, k, v = x.split((H, H, H), 1)
        out, lse = ops.attention_packed(q, k, v, cu, want_lse=True)
        value, row, saved = T.linear_ce_fwd(out.view(n, E), w, b, t)
        dh, dw, db = T.linear_ce_bwd(g, saved)
        return (value, row, dh, dw, db, *T.attention_packed_bwd(dh.view(n, H, dim), q, k, v, out, lse, cu))
    x, t, g = inputs(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, t, g)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = step(x, t, g)
    for i in (1, 3, 0, 2):
        new = inputs(i)
        for a, c in zip((x, t, g), new):
            a.copy_(c)
        graph.replay()
        eager = step(*new)
        torch.cuda.synchronize()
        for a, c in zip(recorded, eager):
            assert torch.equal(a, c), f"inputs {i}"


def test_loss_gradients_on_two_streams_at_once():
    from image_captioning_amd import train_ops as T
    h, w, t = rnd(700, 64, seed=4).to(D), rnd(2000, 64, seed=5, scale=0.1).to(D), torch.arange(700, device=D)
    h2, w2, t2 = rnd(300, 128, seed=6).to(D), rnd(900, 128, seed=7, scale=0.1).to(D), torch.arange(300, device=D)
    one = torch.ones(1, device=D)

    def go(*x):
        return T.linear_ce_bwd(one, T.linear_ce_fwd(x[0], x[1], None, x[2])[2])[:2]
    want = go(h, w, t), go(h2, w2, t2)
    torch.cuda.synchronize()
    a, c = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(a):
            x = go(h, w, t)
        with torch.cuda.stream(c):
            y = go(h2, w2, t2)
        torch.cuda.synchronize()
        for got, ref in zip((*x, *y), (*want[0], *want[1])):
            assert torch.equal(got, ref)

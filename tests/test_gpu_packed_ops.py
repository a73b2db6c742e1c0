"""GPU: attention over packed sequences, the vocabulary loss without logits and the many-tensor AdamW against plain formulas in 64
bits.  Every tolerance is an elementwise bound on the error, from the roundings that the kernels make:
u = half a step of the tensors' type (one rounding of P, of dS, of D, of the result), 2^-24 for every fp32 operation in a sum."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
D = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]
E24 = 2.0 ** -24


def half_step(t):
    return torch.finfo(t).eps / 2


def rnd(*shape, seed, scale=1.0, dtype=F32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def offsets(lengths):
    return torch.tensor([0] + list(torch.tensor(lengths).cumsum(0)), dtype=torch.int32)


def within(got, want, bound, what):
    got = got.detach().double().cpu()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - want).abs() - bound
    assert (over <= 0).all(), f"{what}: {float((got - want).abs().max()):.3g} off, {float(((got - want).abs() / bound.clamp(min=1e-300)).max()):.2f} times the bound"


# ------------------------------------------------------------------------------------------------ attention
def attention_oracle(q, k, v, lq, lk, causal, scale, dout=None):
    """Results and elementwise error bounds, sequence by sequence, in 64 bits on the CPU."""
    u = half_step(q.dtype)
    up = 0.0 if q.dtype == F32 else u                        # P and dS are rounded to the tensors' type
    q, k, v = q.double(), k.double(), v.double()
    H, K, dim = q.shape[1], k.shape[1], q.shape[2]
    names = ("out", "lse") + (("dq", "dk", "dv") if dout is not None else ())
    r = {"out": torch.zeros_like(q), "lse": torch.full(q.shape[:2], -math.inf, dtype=torch.float64), "dq": torch.zeros_like(q),
         "dk": torch.zeros_like(k), "dv": torch.zeros_like(v)}
    b = {n: torch.zeros_like(x) for n, x in r.items()}
    q0 = k0 = 0
    for nq, nk in zip(lq, lk):
        seen = torch.ones(nq, nk, dtype=torch.bool)
        if causal:
            seen = torch.arange(nk) <= torch.arange(nq)[:, None] + nk - nq
        for h in range(H if nk and nq else 0):
            g = h // (H // K)
            Q, KK, V = q[q0:q0 + nq, h], k[k0:k0 + nk, g], v[k0:k0 + nk, g]
            s = (scale * Q @ KK.t()).masked_fill(~seen, -math.inf)
            lse = torch.logsumexp(s, 1)
            some = torch.isfinite(lse)
            P = torch.where(some[:, None], torch.exp(s - torch.where(some, lse, torch.zeros_like(lse))[:, None]), torch.zeros_like(s))
            # a score is a dot product of dim terms, the exponent's argument and exp2 itself add a few roundings of it
            ds_ = float(scale * (dim + 8) * E24 * (Q.abs() @ KK.abs().t()).max()) + 2.0 ** -21
            f = (nk + 16) * E24                              # a sum over nk keys
            O = P @ V
            A = P @ V.abs()
            EO = (up + f + 3 * ds_) * A + 1e-30
            r["out"][q0:q0 + nq, h], b["out"][q0:q0 + nq, h] = O, EO + u * O.abs() * (1 + 2 ** -6)
            r["lse"][q0:q0 + nq, h], b["lse"][q0:q0 + nq, h] = lse, 2 * ds_ + 4 * E24 * lse.abs().nan_to_num(posinf=0.0) + f
            if dout is None:
                continue
            G = dout[q0:q0 + nq, h].double()
            fr, fd = (nq * (H // K) + 16) * E24, (dim + 8) * E24
            dP = G @ V.t()
            delta = (G * O).sum(1, keepdim=True)
            dS = P * (dP - delta)
            e_delta = (G.abs() * (EO + u * O.abs())).sum(1, keepdim=True) + fd * (G * O).abs().sum(1, keepdim=True)
            E = (up + 3 * ds_ + 4 * E24) * dS.abs() + P * (fd * (G.abs() @ V.abs().t()) + e_delta)
            x = scale * dS @ KK
            r["dq"][q0:q0 + nq, h] = x
            b["dq"][q0:q0 + nq, h] = scale * ((E + f * dS.abs()) @ KK.abs()) * 1.01 + u * x.abs() * (1 + 2 ** -6) + 1e-30
            r["dk"][k0:k0 + nk, g] += scale * dS.t() @ Q
            b["dk"][k0:k0 + nk, g] += scale * ((E + fr * dS.abs()).t() @ Q.abs()) * 1.01 + 1e-30
            r["dv"][k0:k0 + nk, g] += P.t() @ G
            b["dv"][k0:k0 + nk, g] += ((up + fr + 3 * ds_) * P).t() @ G.abs() * 1.01 + 1e-30
        q0, k0 = q0 + nq, k0 + nk
    for n in ("dk", "dv"):
        b[n] += u * r[n].abs() * (1 + 2 ** -6)
    # fp16's smallest step, of P, dS and of the results
    tiny = 0.0 if q.dtype == F32 or u > 1e-3 else 2.0 ** -25
    return {n: (r[n], b[n] + (tiny * (1 + sum(lk) + sum(lq)) * 4 if n != "lse" else 0.0)) for n in names}


def run_attention(q, k, v, lq, lk, causal, scale=None, dout=None):
    from image_captioning_amd import ops, train_ops as T
    cq, ck = offsets(lq).to(D), offsets(lk).to(D)
    out, lse = ops.attention_packed(q, k, v, cq, ck, causal=causal, scale=scale, want_lse=True)
    got = {"out": out, "lse": lse}
    if dout is not None:
        got["dq"], got["dk"], got["dv"] = T.attention_packed_bwd(dout, q, k, v, out, lse, cq, ck, causal=causal, scale=scale)
    return got


def compare_attention(dtype, lq, lk, H, K, dim, causal, seed=0, scale=None, big=1.0, extra=0):
    """extra: rows behind the last sequence."""
    tq, tk = sum(lq), sum(lk)
    q, k, v = rnd(tq + extra, H, dim, seed=seed, scale=big, dtype=dtype), rnd(tk + extra, K, dim, seed=seed + 1, dtype=dtype), rnd(tk + extra, K, dim, seed=seed + 2, dtype=dtype)
    g = rnd(tq + extra, H, dim, seed=seed + 3, dtype=dtype)
    s = scale if scale is not None else dim ** -0.5
    want = attention_oracle(q, k, v, lq, lk, causal, s, g)
    got = run_attention(q.to(D), k.to(D), v.to(D), lq, lk, causal, scale, g.to(D))
    for n, (w, b) in want.items():
        x = got[n].detach().double().cpu()
        if n == "lse":
            empty = torch.isinf(w)
            assert torch.equal(torch.isinf(x) & (x < 0), empty), "lse of empty rows"
            within(x[~empty], w[~empty], b[~empty], n)
        else:
            within(x, w, b, n)
    if extra:
        for n, used in (("out", tq), ("dq", tq), ("dk", tk), ("dv", tk)):
            assert not got[n][used:].any(), f"{n} behind the last sequence"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [8, 32, 40, 64, 80, 128])
@pytest.mark.parametrize("H,K", [(1, 1), (6, 2), (8, 1)])
def test_attention_shapes(dtype, dim, H, K):
    compare_attention(dtype, [5, 0, 64, 1, 33], [5, 0, 64, 1, 33], H, K, dim, True, seed=dim)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lq,lk", [([1], [1]), ([300], [300]), ([130, 15, 16, 17], [130, 15, 16, 17]),       # tile borders
                                   ([7, 3, 0, 20], [70, 0, 5, 129]),                                         # keys of another length, none, no queries
                                   ([40, 9], [10, 9]), ([65], [1]),                                          # more queries than keys: rows that see nothing
                                   ([127, 129], [257, 63])])
def test_attention_lengths(dtype, causal, lq, lk):
    compare_attention(dtype, lq, lk, 4, 2, 64, causal, seed=len(lq) + 3, extra=3)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_many_sequences(dtype):
    """More sequences than a workgroup has threads: the search for a tile's sequence goes round more than once."""
    lq = [(i * 7) % 13 for i in range(700)]
    compare_attention(dtype, lq, lq, 2, 2, 32, True, seed=5, extra=70)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,K", [(8, 1), (4, 4), (32, 2)])
def test_attention_single_tokens_over_long_caches(dtype, H, K):
    """One new token a text, keys split over workgroups: a long cache, short ones, one of a single token, an empty one."""
    compare_attention(dtype, [1, 1, 1, 1], [3001, 127, 1, 0], H, K, 64, True, seed=H)
    compare_attention(dtype, [1], [129], H, K, 128, True, seed=H + 1, extra=1)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_more_tiles_than_the_card_takes_at_once(dtype):
    """Long sequences whose backward pass does not share a walk between groups of waves: there are enough workgroups."""
    lens = [130] * 15 + [131]
    compare_attention(dtype, lens, lens, 64, 64, 8, True, seed=11)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_large_scores(dtype):
    compare_attention(dtype, [90, 31], [90, 31], 2, 1, 64, True, seed=9, big=20.0)
    compare_attention(dtype, [40], [40], 2, 1, 64, False, seed=10, scale=1e-3)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_of_slices_of_one_projection(dtype):
    """q, k, v as strided slices of a fused [tokens, (heads + 2 kv_heads) dim] projection, and as slices that are not aligned."""
    from image_captioning_amd import ops
    H, K, dim, lens = 4, 2, 32, [50, 14]
    n = sum(lens)
    for pad in (0, 3):                                       # pad 3: rows that are not 16-byte aligned
        x = rnd(n, (H + 2 * K) * dim + pad, seed=4, dtype=dtype).to(D)
        q, k, v = (t.unflatten(1, (-1, dim)) for t in x[:, pad:].split((H * dim, K * dim, K * dim), 1))
        cu = offsets(lens).to(D)
        got = ops.attention_packed(q, k, v, cu)
        assert torch.equal(got, ops.attention_packed(q.contiguous(), k.contiguous(), v.contiguous(), cu))
        heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)
        assert torch.equal(got, ops.attention_packed(heads_first, k, v, cu))


def test_attention_hidden_keys_may_hold_anything():
    """The last key is seen by the last query alone: whatever it holds, the other rows are what they were."""
    from image_captioning_amd import ops
    q, k, v = (rnd(70, 2, 64, seed=s, dtype=BF16).to(D) for s in (1, 2, 3))
    cu = offsets([70]).to(D)
    want = ops.attention_packed(q, k, v, cu)
    for bad in (math.nan, math.inf, torch.finfo(BF16).min):
        k2 = k.clone()
        k2[-1] = bad
        assert torch.equal(ops.attention_packed(q, k2, v, cu)[:-1], want[:-1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("lq,lk,H,K,dim", [([20, 30, 100, 5], [20, 30, 100, 5], 4, 2, 64), ([9, 250, 300], [9, 250, 300], 2, 2, 40), ([1, 1, 1], [900, 1500, 40], 4, 1, 128)])
def test_attention_sequences_do_not_touch_each_other(dtype, bad, lq, lk, H, K, dim):
    """Sequence 1 holds NaN or infinities everywhere: the results of the others, which share its tiles, are the formula's."""
    q, k, v, g = (rnd(sum(n), h, dim, seed=s, dtype=dtype) for n, h, s in ((lq, H, 1), (lk, K, 2), (lk, K, 3), (lq, H, 4)))
    want = attention_oracle(q, k, v, lq, lk, True, dim ** -0.5, g)
    rows, keys = slice(lq[0], lq[0] + lq[1]), slice(lk[0], lk[0] + lk[1])
    for x, at in ((q, rows), (k, keys), (v, keys), (g, rows)):
        x[at] = bad
    got = run_attention(q.to(D), k.to(D), v.to(D), lq, lk, True, None, g.to(D))
    for n, (w, b) in want.items():
        others = torch.ones(len(w), dtype=torch.bool)
        others[keys if n in ("dk", "dv") else rows] = False
        within(got[n].cpu()[others], w[others], b[others], n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("n,dim", [(50, 64), (300, 128)])
def test_attention_values_behind_a_token_do_not_touch_it(dtype, bad, n, dim):
    """The last key and value are seen by the last query alone, the first query's row sees the first key alone."""
    q, k, v, g = (rnd(n, 2, dim, seed=s, dtype=dtype) for s in (5, 6, 7, 8))
    want = attention_oracle(q, k, v, [n], [n], True, dim ** -0.5, g)

    def changed(x, at):
        x = x.clone()
        x[at] = bad
        return x
    got = run_attention(q.to(D), changed(k, -1).to(D), changed(v, -1).to(D), [n], [n], True, None, g.to(D))
    for name in ("out", "lse", "dq"):
        within(got[name].cpu()[:-1], want[name][0][:-1], want[name][1][:-1], name)
    got = run_attention(changed(q, 0).to(D), k.to(D), v.to(D), [n], [n], True, None, changed(g, 0).to(D))
    for name in ("out", "lse", "dq", "dk", "dv"):
        within(got[name].cpu()[1:], want[name][0][1:], want[name][1][1:], name)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_infinite_values_are_the_formulas(dtype):
    """A visible key of the score -inf has the weight zero; a visible infinite value is the rows' result."""
    q, k, v = (rnd(40, 1, 24, seed=s, dtype=dtype) for s in (1, 2, 3))
    q[:, 0, 0] = 1.0
    k2 = k.clone()
    k2[7, 0, 0] = -math.inf
    v2 = v.clone()
    v2[9, 0, 3] = math.inf
    got = run_attention(q.to(D), k2.to(D), v2.to(D), [40], [40], False)["out"].cpu()
    left = torch.arange(40) != 7
    w, b = attention_oracle(q, k[left], v[left], [40], [39], False, 24 ** -0.5)["out"]
    cols = torch.arange(24) != 3
    within(got[:, :, cols], w[:, :, cols], b[:, :, cols], "out")
    assert (got[:, :, 3] == math.inf).all()


def test_attention_over_more_than_2_31_elements():
    """Rows 2^23 elements apart: the last ones lie beyond 2^31 elements, whichever tensor they are of."""
    n, H, K, dim = 290, 2, 1, 32
    wide = torch.empty(n, 1 << 23, device=D, dtype=BF16)
    packed = rnd(n, (2 * H + 2 * K) * dim, seed=1, dtype=BF16).to(D)
    wide[:, -packed.size(1):] = packed

    def parts(x):
        return [t.unflatten(1, (-1, dim)) for t in x.split((H * dim, K * dim, K * dim, H * dim), 1)]
    q, k, v, g = parts(packed)
    far = parts(wide[:, -packed.size(1):])
    assert far[1].stride(0) == 1 << 23
    for lq in ([n], [1]):
        near = run_attention(q[-sum(lq):], k, v, lq, [n], True, None, g[-sum(lq):])
        got = run_attention(far[0][-sum(lq):], far[1], far[2], lq, [n], True, None, far[3][-sum(lq):])
        for name in near:
            assert torch.equal(got[name], near[name]), name


def test_attention_offsets_beyond_the_tensors_are_cut_off():
    from image_captioning_amd import ops
    q, k, v = (rnd(40, 2, 32, seed=s).to(D) for s in (1, 2, 3))
    good = ops.attention_packed(q, k, v, offsets([15, 25]).to(D))
    cut = ops.attention_packed(q, k, v, torch.tensor([0, 15, 400], dtype=torch.int32, device=D))
    assert torch.equal(good, cut)


def test_attention_gradient_against_differences():
    """The autograd function's gradient along a random direction, against a central difference of the 64-bit formula."""
    from image_captioning_amd import training
    lens = [9, 20]
    q, k, v = (rnd(29, h, 32, seed=s) for h, s in ((4, 1), (2, 2), (2, 3)))
    w = rnd(29, 4, 32, seed=4).double()

    def value(*x):
        return float((attention_oracle(*(t.double() for t in x), lens, lens, True, 32 ** -0.5)["out"][0] * w).sum())
    leaves = [t.to(D).requires_grad_() for t in (q, k, v)]
    out = training.packed_attention(*leaves, offsets(lens).to(D))
    (out * w.float().to(D)).sum().backward()
    for i in range(3):
        d = rnd(*leaves[i].shape, seed=7 + i).double()
        plus, minus = [t.double() for t in (q, k, v)], [t.double() for t in (q, k, v)]
        plus[i], minus[i] = plus[i] + 1e-4 * d, minus[i] - 1e-4 * d
        want = (value(*plus) - value(*minus)) / 2e-4
        got = float((leaves[i].grad.double().cpu() * d).sum())
        size = float((leaves[i].grad.double().cpu() * d).abs().sum())
        # fp32 sums of some 100 terms in each product, and the difference's own error (third derivatives times 1e-8)
        assert abs(got - want) <= 200 * E24 * size + 1e-6 * size


# ------------------------------------------------------------------------------------------------ vocabulary loss
def ce_oracle(h, w, b, t, ignore, mean, g):
    u = half_step(h.dtype)
    f32 = h.dtype == F32
    h, w = h.double(), w.double()
    R, E = h.shape
    V = w.shape[0]
    x = h @ w.t() + (b.double() if b is not None else 0.0)
    # fp32 tensors: two fp16 parts each (2^-22, and 2^-39 of the largest magnitude), the products of low parts dropped (2^-22)
    A = h.abs() @ w.abs().t()
    dx = (3 * 2.0 ** -22 if f32 else 0.0) * A + ((3 if f32 else 1) * E + 8) * E24 * A + 4 * E24 * x.abs()
    if f32:
        dx = dx + 2.0 ** -38 * (float(h.abs().max()) * w.abs().sum(1) + float(w.abs().max()) * h.abs().sum(1, keepdim=True))
    mx = dx.max(1, keepdim=True)[0]
    lse = torch.logsumexp(x, 1, keepdim=True)
    e_lse = mx + (V / 64 + 80) * E24 + 4 * E24 * lse.abs()
    on = (t >= 0) & (t < V) & (t != ignore)
    at = torch.where(on, t, torch.zeros_like(t))[:, None]
    row = torch.where(on, (lse - x.gather(1, at))[:, 0], torch.zeros_like(lse[:, 0]))
    e_row = torch.where(on, (e_lse + mx)[:, 0] + 2 * E24 * row.abs(), torch.zeros_like(row))
    n = int(on.sum()) if mean else R
    sc = 1.0 / n if n else 0.0
    P = torch.exp(x - lse)
    d = (P - torch.zeros_like(P).scatter_(1, at, 1.0)) * on[:, None]
    # exp of an argument that is off by dx + e_lse, hardware exp2 (2^-22 with its argument's rounding); one rounding to 16 bits
    ed = (P * (dx + e_lse + (lse - x).abs() * 3 * E24 + 2.0 ** -21) + d.abs() * (2.0 ** -22 if f32 else u) + (0 if u > 1e-3 else 2.0 ** -39)) * on[:, None]
    k = abs(g) * sc
    tiny = 2.0 ** -25 if h.dtype != F32 and u < 1e-3 else 0.0
    tiny = 2.0 ** -25 if (not f32 and u < 1e-3) else 0.0

    def grad(a, ea, m, terms):
        y = g * sc * a @ m
        low = (3 * 2.0 ** -22 * a.abs() @ m.abs() + 2.0 ** -38 * a.abs().sum(1, keepdim=True) * float(m.abs().max())) if f32 else 0.0
        return y, k * (ea @ m.abs() + ((3 if f32 else 1) * terms + 48) * E24 * (a.abs() @ m.abs()) + low) * 1.01 + (u + 4 * E24) * y.abs() * 1.01 + tiny
    db = g * sc * d.sum(0)
    e_plain = (P * (dx + e_lse + (lse - x).abs() * 3 * E24 + 2.0 ** -21) * on[:, None]).sum(0)
    return {"row_loss": (row, e_row), "loss": (row.sum() * sc, e_row.sum() * sc + 4 * E24 * (row.sum() * sc).abs()),
            "dh": grad(d, ed, w, V), "dw": grad(d.t(), ed.t(), h, R),
            "db": (db, k * (e_plain + (R + 8) * E24 * d.abs().sum(0)) * 1.01 + (u + 4 * E24) * db.abs() * 1.01 + tiny)}


def compare_ce(dtype, R, E, V, bias=True, ignore=-100, mean=True, g=1.0, seed=0, targets=None, hidden=None, weight=None, oracle="cpu"):
    from image_captioning_amd import train_ops as T
    h = rnd(R, E, seed=seed, dtype=dtype) if hidden is None else hidden
    w = rnd(V, E, seed=seed + 1, scale=2.0 * E ** -0.5, dtype=dtype) if weight is None else weight
    b = rnd(V, seed=seed + 2, scale=0.5, dtype=dtype) if bias else None
    t = torch.randint(0, V, (R,), generator=torch.Generator().manual_seed(seed + 3)) if targets is None else targets
    want = ce_oracle(*(x.to(oracle) if x is not None else None for x in (h, w, b, t)), ignore, mean, g)
    want = {n: (x.cpu(), e.cpu()) for n, (x, e) in want.items()}
    value, row, saved = T.linear_ce_fwd(h.to(D), w.to(D), b.to(D) if bias else None, t.to(D), ignore, mean)
    dh, dw, db = T.linear_ce_bwd(torch.tensor([g], device=D), saved)
    got = {"loss": value, "row_loss": row, "dh": dh, "dw": dw, "db": db}
    for n, (x, e) in want.items():
        if n == "db" and not bias:
            assert db is None
            continue
        assert got[n].dtype == (F32 if n in ("loss", "row_loss") else dtype)
        within(got[n], x, e, n)
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,E,V", [(1, 8, 1), (1, 64, 81), (3, 40, 7), (57, 512, 81), (129, 72, 257), (300, 64, 1000), (64, 520, 513), (260, 128, 6756)])
def test_linear_ce_sizes(dtype, R, E, V):
    t = torch.randint(0, V, (R,), generator=torch.Generator().manual_seed(R))
    t[R // 2:R // 2 + R // 4] = -100
    if R > 3:
        t[1], t[2] = V, -1                                    # outside the vocabulary: left out, as ce_loss does
    compare_ce(dtype, R, E, V, g=64.0 if dtype == F16 else 1.0, seed=R, targets=t)
    compare_ce(dtype, R, E, V, bias=False, mean=False, g=-2.5, seed=R + 1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf, 1e30])
@pytest.mark.parametrize("E", [64, 40])
def test_linear_ce_left_out_rows_may_hold_anything(dtype, bad, E):
    from image_captioning_amd import train_ops as T
    R, V = 90, 200
    h, w, b = rnd(R, E, seed=1, dtype=dtype), rnd(V, E, seed=2, scale=0.2, dtype=dtype), rnd(V, seed=3, dtype=dtype)
    t = torch.randint(0, V, (R,), generator=torch.Generator().manual_seed(4))
    t[::7], t[3], t[4] = 0, V, -5
    want = ce_oracle(h, w, b, t, 0, True, 2.0)
    h[::7], h[3], h[4] = bad, bad, bad
    h[t == 0] = bad
    value, row, saved = T.linear_ce_fwd(h.to(D), w.to(D), b.to(D), t.to(D), 0, True)
    dh, dw, db = T.linear_ce_bwd(torch.tensor([2.0], device=D), saved)
    for n, x in (("loss", value), ("row_loss", row), ("dh", dh), ("dw", dw), ("db", db)):
        within(x, *want[n], n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf, 1e9])
def test_linear_ce_rows_do_not_touch_each_other(dtype, bad):
    """A row that counts and holds NaN, infinities or huge values: the losses of the others, and their rows of dhidden, are the formula's."""
    from image_captioning_amd import train_ops as T
    R, E, V = 70, 64, 150
    h, w = rnd(R, E, seed=1, dtype=dtype), rnd(V, E, seed=2, scale=0.2, dtype=dtype)
    t = torch.randint(0, V, (R,), generator=torch.Generator().manual_seed(4))
    want = ce_oracle(h, w, None, t, -100, False, 1.0)
    h[33] = bad
    _, row, saved = T.linear_ce_fwd(h.to(D), w.to(D), None, t.to(D), -100, False)
    dh, _, _ = T.linear_ce_bwd(torch.tensor([1.0], device=D), saved)
    others = torch.arange(R) != 33
    for n, x in (("row_loss", row), ("dh", dh)):
        within(x.cpu()[others], want[n][0][others], want[n][1][others], n)


def test_linear_ce_over_more_than_2_31_elements():
    """A weight of 2.2e9 elements, and hidden rows 2^23 elements apart."""
    from image_captioning_amd import train_ops as T
    R, E, V = 290, 8192, 268500
    wide = torch.empty(R, 1 << 23, device=D, dtype=BF16)
    h = wide[:, -E:]
    h.copy_(rnd(R, E, seed=1, dtype=BF16))
    w = torch.empty(V, E, device=D, dtype=BF16)
    for i, rows in enumerate(w.split(65536)):
        rows.copy_(torch.randn(rows.shape, device=D, generator=torch.Generator(D).manual_seed(i)).mul_(E ** -0.5))
    t = torch.randint(0, V, (R,), generator=torch.Generator().manual_seed(2))
    t[-3:] = V - 1
    _, row, saved = T.linear_ce_fwd(h, w, None, t.to(D), -100, True)
    dh, dw, _ = T.linear_ce_bwd(torch.tensor([1.0], device=D), saved)
    hc = h.float()
    x = torch.cat([hc @ rows.float().t() for rows in w.split(65536)], 1).double()
    lse = torch.logsumexp(x, 1)
    # exact products summed in fp32 on both sides: each x is off by at most E 2^-24 of its terms' magnitudes
    e = 2 * E * E24 * float(max((hc.abs() @ rows.float().abs().t()).max() for rows in w.split(65536)))
    assert ((row.double() - (lse - x.gather(1, t.to(D)[:, None])[:, 0])).abs() < 2 * e + 1e-5).all()
    hot = (t.to(D)[:, None] == torch.arange(V - 500, V, device=D)).double()
    d = torch.exp(x[:, -500:] - lse[:, None]) - hot
    want = d.t() @ hc.double() / R
    bound = (2.0 ** -8 + 2 * e) * 1.1 * ((d.abs() + hot).t() @ hc.double().abs() / R) + 2.0 ** -8 * want.abs()     # D and the result rounded
    assert ((dw[-500:].double() - want).abs() <= bound).all()
    assert torch.isfinite(dh).all() and dh.any()


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_ce_large_tiles_and_split_contraction(dtype):
    """Enough rows and words for the 256 x 256 tiles, few enough columns that dh and dw split their contraction."""
    compare_ce(dtype, 3300, 64, 4100, g=512.0 if dtype == F16 else 1.0, seed=3)


def test_linear_ce_in_several_pieces_of_the_vocabulary():
    """So many rows that D of the whole vocabulary would pass the workspace's limit: five pieces, the last one shorter."""
    from image_captioning_amd import _native as N
    R, E, V = 130000, 16, 2501
    assert N.load().icap_linear_ce_ws_bytes(1, R, E, V, 1) < 3 * R * V
    compare_ce(BF16, R, E, V, seed=4, g=8.0, oracle=D)


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_ce_extremes(dtype):
    """No row counts; one row counts; a sure prediction; magnitudes far from 1 (fp32: powers of two are taken out and put back)."""
    all_out = torch.full((9,), -100)
    got = compare_ce(dtype, 9, 32, 50, targets=all_out)
    assert float(got["loss"]) == 0.0 and not got["dh"].any() and not got["dw"].any() and not got["db"].any()
    one = all_out.clone()
    one[4] = 49
    compare_ce(dtype, 9, 32, 50, targets=one, ignore=-100)
    h = torch.zeros(5, 32, dtype=dtype)
    h[:, 0] = 30.0
    w = torch.zeros(50, 32, dtype=dtype)
    w[7, 0] = 30.0
    compare_ce(dtype, 5, 32, 50, bias=False, hidden=h, weight=w, targets=torch.tensor([7, 7, 3, 7, 0]), mean=False)
    if dtype == F32:
        for e in (-30, 30):
            compare_ce(dtype, 33, 48, 90, hidden=rnd(33, 48, seed=1) * 2.0 ** e, weight=rnd(90, 48, seed=2) * 2.0 ** -e * 0.3, seed=6)


def test_linear_ce_strided_rows_and_autograd():
    """hidden as a slice of [captions, steps, width], through autograd, with only some gradients wanted."""
    from image_captioning_amd import train_ops as T, training
    h = rnd(6, 11, 64, seed=1).to(D).requires_grad_()
    w, b = rnd(100, 64, seed=2, scale=0.2).to(D).requires_grad_(), rnd(100, seed=3).to(D)
    t = torch.randint(0, 100, (6, 11), generator=torch.Generator().manual_seed(4)).to(D)
    value = training.linear_cross_entropy(h[:, :-1], w, b, t[:, 1:], ignore_index=5, mean_over_valid=False)
    (3.0 * value).backward()
    flat = h.detach()[:, :-1].reshape(-1, 64)
    want, _, saved = T.linear_ce_fwd(flat, w.detach(), b, t[:, 1:].reshape(-1).contiguous(), 5, False)
    dh, dw, db = T.linear_ce_bwd(torch.tensor([3.0], device=D), saved, need=(True, True, False))
    assert db is None and torch.equal(value.detach(), want)
    assert torch.equal(h.grad[:, :-1].reshape(-1, 64), dh) and not h.grad[:, -1].any() and torch.equal(w.grad, dw)
    wide = torch.zeros(60, 100, device=D)
    wide[:, 8:72] = flat
    assert torch.equal(T.linear_ce_fwd(wide[:, 8:72], w.detach(), b, t[:, 1:].reshape(-1).contiguous(), 5, False)[0], want)


def test_linear_ce_agrees_with_the_loss_on_stored_logits():
    from image_captioning_amd import training
    h, w, b = rnd(48, 20, 64, seed=1).to(D), rnd(811, 64, seed=2, scale=0.2).to(D), rnd(811, seed=3).to(D)
    t = torch.randint(0, 811, (48, 20), generator=torch.Generator().manual_seed(4)).to(D)
    t[:, 15:] = 0
    logits = (h.double() @ w.double().t() + b.double()).float()
    a, c = training.compute_loss(logits, t, 0), training.CrossEntropyLoss(ignore_index=0)(logits.reshape(-1, 811), t.reshape(-1))
    # both are fp32 means of some 1000 row losses near 7, logits from sums of 64 terms
    assert abs(float(a) - float(training.linear_cross_entropy(h, w, b, t, 0, mean_over_valid=False))) < 2e-5
    assert abs(float(c) - float(training.linear_cross_entropy(h, w, b, t, 0))) < 2e-5


# ------------------------------------------------------------------------------------------------ AdamW
def adamw_oracle(p, g, m, v, step, lr=1e-2, b1=0.9, b2=0.99, eps=1e-6, wd=0.1):
    p, g, m, v = (x.double() for x in (p, g, m, v))
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    return p * (1 - lr * wd) - lr / (1 - b1 ** step) * m / ((v / (1 - b2 ** step)).sqrt() + eps), m, v


HYPER = dict(lr=1e-2, beta1=0.9, beta2=0.99, eps=1e-6, weight_decay=0.1)
SIZES = [1, 3, 4, 255, 256, 257, 4095, 4096, 4097, 30011]


@pytest.mark.parametrize("dtype,gdtype", [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize("shift", [0, 1])
def test_adamw_tensors_with_fp32_states(dtype, gdtype, shift):
    """shift 1: views that start one value into their storage, where 16-byte access is not possible."""
    from image_captioning_amd import train_ops as T

    def put(x):
        return torch.cat([x.new_zeros(shift), x]).to(D)[shift:]
    ps = [rnd(n, seed=n, dtype=dtype) for n in SIZES]
    gs = [rnd(n, seed=n + 1, scale=10.0 ** (i % 4 - 2), dtype=gdtype) for i, n in enumerate(SIZES)]
    ms, vs = [rnd(n, seed=n + 2, scale=0.1) for n in SIZES], [rnd(n, seed=n + 3).abs() for n in SIZES]
    dev = [[put(x) for x in xs] for xs in (ps, gs, ms, vs)]
    T.adamw_tensors(*dev, step=3, **HYPER)
    u = half_step(dtype)
    for i, n in enumerate(SIZES):
        p, m, v = adamw_oracle(ps[i], gs[i], ms[i], vs[i], 3)
        # m and v: three roundings of values no larger than |m| + |g| and v + g g; the update: eight more
        em, ev = 4 * E24 * (ms[i].double().abs() + gs[i].double().abs()), 5 * E24 * (vs[i].double() + gs[i].double() ** 2)
        within(dev[2][i], m, em, "m")
        within(dev[3][i], v, ev, "v")
        denom = (v / (1 - 0.99 ** 3)).sqrt() + 1e-6
        size = 1e-2 / (1 - 0.9 ** 3) / denom
        upd = size * m.abs()
        within(dev[0][i], p, size * em + upd * (ev / v.clamp(min=1e-300) + 10 * E24) + 3 * E24 * ps[i].double().abs() + (u + E24) * p.abs() + (2.0 ** -25 if dtype == F16 else 0.0), "p")


def test_adamw_tensors_equals_the_flat_optimizer():
    from image_captioning_amd import training
    shapes = [(3, 5), (7,), (100, 41), (1,)]
    a = [torch.nn.Parameter(rnd(*s, seed=i).to(D)) for i, s in enumerate(shapes)]
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    A = training.AdamW(a, lr=3e-3, weight_decay=0.05)
    B = training.AdamWTensors(b, lr=3e-3, weight_decay=0.05, state_bits=32)
    for step in range(4):
        A.zero_grad()
        B.zero_grad()
        for i in range(len(shapes)):
            if i == 1 and step < 2:
                continue                                     # a parameter that gets its first gradient later
            g = rnd(*shapes[i], seed=10 * step + i).to(D)
            for p in (a[i], b[i]):
                (p * g).sum().backward()
        A.step()
        B.step()
    assert A.param_steps == B.param_steps == [4, 2, 4, 4]
    for p, q in zip(a, b):
        # coefficients rounded from other intermediate types: a few 2^-24 of the four updates of at most 3e-3 each
        assert float((p - q).detach().abs().max()) <= 4 * 3e-3 * 16 * E24 + 4 * E24 * float(p.detach().abs().max())


def decode(codes, scales):
    n = codes.numel()
    return codes.float().cpu().double().reshape(-1) * scales.cpu().double().repeat_interleave(256)[:n]


@pytest.mark.parametrize("dtype,gdtype", [(F32, F32), (BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("shift", [0, 1])
def test_adamw_tensors_with_8_bit_states(dtype, gdtype, shift):
    """Two steps in a row: parameters as from the states' values; codes next to the exact values: the first moment the nearest one,
    the second's root one of its two neighbours and never zero for a value above zero."""
    from image_captioning_amd import train_ops as T
    ps = [rnd(n, seed=n, dtype=dtype) for n in SIZES]
    dev = [torch.cat([p.new_zeros(shift), p]).to(D)[shift:] for p in ps]
    m, v = [T.adamw_state8(p) for p in dev], [T.adamw_state8(p) for p in dev]
    if shift:
        m = [(torch.zeros(p.numel() + 1, dtype=torch.uint8, device=D).view(torch.float8_e4m3fn)[1:], s) for p, (_, s) in zip(dev, m)]
    u = half_step(dtype)
    for step in (1, 2):
        gs = [rnd(n, seed=n + step, scale=10.0 ** (i % 4 - 2), dtype=gdtype) for i, n in enumerate(SIZES)]
        gs = [torch.where(torch.arange(g.numel()) % 11 == 5, g * 2.0 ** -12, g) for g in gs]      # small ones among large ones
        before = [(p.cpu().clone(), decode(*a), decode(*b) ** 2) for p, a, b in zip(dev, m, v)]
        T.adamw_tensors(dev, [torch.cat([g.new_zeros(shift), g]).to(D)[shift:] for g in gs], m, v, step=step, seed=77, **HYPER)
        for i, n in enumerate(SIZES):
            p, mm, vv = adamw_oracle(before[i][0], gs[i], before[i][1], before[i][2], step)
            g64 = gs[i].double()
            em, ev = 5 * E24 * (before[i][1].abs() + g64.abs()), 7 * E24 * (before[i][2] + g64 ** 2)
            size = 1e-2 / (1 - 0.9 ** step) / ((vv / (1 - 0.99 ** step)).sqrt() + 1e-6)
            within(dev[i], p, size * em + size * mm.abs() * (ev / vv.clamp(min=1e-300) + 10 * E24) + 3 * E24 * before[i][0].double().abs() + (u + E24) * p.abs() + (2.0 ** -25 if dtype == F16 else 0.0), "p")
            for (codes, scales), x, ex, at_random in ((m[i], mm, em, False), (v[i], vv.sqrt(), ev / vv.sqrt().clamp(min=1e-300), True)):
                pad = torch.nn.functional.pad(x.abs(), (0, -n % 256)).view(-1, 256)
                most = pad.amax(1)
                assert ((scales.cpu().double() - most / 448).abs() <= 8 * E24 * most / 448 + (ex.max() / 448)).all()
                sc = scales.cpu().double().repeat_interleave(256)[:n]
                y = x / sc
                # spacing of e4m3 around |y|: 2^-3 of its power of two, 2^-9 at the bottom
                step_of = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
                off = (codes.float().cpu().double().reshape(-1) - y).abs()
                slack = (ex / sc) + 16 * E24 * y.abs()
                if not at_random:
                    assert (off <= step_of / 2 + slack).all()
                else:
                    assert (off <= step_of + slack).all()
                    assert ((codes.float().cpu().reshape(-1) > 0) == (vv > 0)).all()


def test_adamw_8_bit_second_moment_moves_on_average():
    """sqrt(v) is rounded at random with the right mean: over 4096 equal values the mean code is the value, to six standard
    deviations of a mean of that many roundings (each at most half a step)."""
    from image_captioning_amd import train_ops as T
    n = 4096
    p, g = torch.zeros(n, device=D), torch.full((n,), 0.3, device=D)
    g[::256] = 1.0                                           # the largest of each block
    m, v = T.adamw_state8(p), T.adamw_state8(p)
    T.adamw_tensors([p], [g], [m], [v], step=1, seed=5, **HYPER)
    x = decode(*v)[torch.arange(n) % 256 != 0]
    want = math.sqrt(0.01) * float(torch.tensor(0.3, dtype=F32))
    step = 2.0 ** (math.floor(math.log2(0.3 * 448)) - 3) * math.sqrt(0.01) / 448
    assert len(x.unique()) == 2
    assert abs(float(x.mean()) - want) < 6 * step / 2 / math.sqrt(len(x))
    # and another seed or step rounds others up
    again, other = T.adamw_state8(p), T.adamw_state8(p)
    T.adamw_tensors([torch.zeros_like(p)], [g], [T.adamw_state8(p)], [again], step=1, seed=5, **HYPER)
    T.adamw_tensors([torch.zeros_like(p)], [g], [T.adamw_state8(p)], [other], step=1, seed=6, **HYPER)
    assert torch.equal(again[0].view(torch.uint8), v[0].view(torch.uint8)) and not torch.equal(other[0].view(torch.uint8), v[0].view(torch.uint8))


def test_adamw_8_bit_zero_and_not_finite_gradients():
    from image_captioning_amd import train_ops as T
    p = torch.ones(600, device=D)
    g = torch.zeros(600, device=D)
    m, v = T.adamw_state8(p), T.adamw_state8(p)
    T.adamw_tensors([p], [g], [m], [v], step=1, lr=1e-2, weight_decay=0.0)
    assert torch.equal(p, torch.ones_like(p)) and not m[0].float().any() and not v[1].any()
    g[300] = math.inf                                        # in the second block of three
    T.adamw_tensors([p], [g], [m], [v], step=2, lr=1e-2, weight_decay=0.0)
    assert torch.equal(p[:256], torch.ones(256, device=D)) and torch.equal(p[512:], torch.ones(88, device=D)) and not torch.isfinite(p[300])
    T.adamw_tensors([p], [torch.zeros_like(g)], [m], [v], step=3, lr=1e-2, weight_decay=0.0)
    assert torch.isfinite(p[:256]).all() and torch.isfinite(p[512:]).all()


def test_adamw_tensors_more_than_one_launch_holds():
    """130 tensors, some without a gradient, some empty: four launches, each tensor as if it were alone with its index."""
    from image_captioning_amd import train_ops as T
    sizes = [(i * 37) % 900 for i in range(130)]
    ps = [rnd(n, seed=i).to(D) for i, n in enumerate(sizes)]
    gs = [None if i % 17 == 3 else rnd(n, seed=200 + i).to(D) for i, n in enumerate(sizes)]
    ms, vs = [T.adamw_state8(p) for p in ps], [T.adamw_state8(p) for p in ps]
    alone = [p.clone() for p in ps]
    ma, va = [T.adamw_state8(p) for p in ps], [T.adamw_state8(p) for p in ps]
    T.adamw_tensors(ps, gs, ms, vs, step=1, seed=9, lr=1e-2)
    for i in range(130):
        T.adamw_tensors([alone[i]], [gs[i]], [ma[i]], [va[i]], step=1, seed=9, lr=1e-2, index=[i])
        assert torch.equal(ps[i], alone[i]) and torch.equal(vs[i][0].view(torch.uint8), va[i][0].view(torch.uint8)) and torch.equal(ms[i][1], ma[i][1])


def test_adamw_tensors_of_more_than_2_31_values():
    from image_captioning_amd import train_ops as T
    n, tail = (1 << 31) + 777, 3000
    p, g = (torch.zeros(n, device=D, dtype=BF16) for _ in range(2))
    m, v = (torch.zeros(n, device=D) for _ in range(2))
    small = [rnd(tail, seed=1, dtype=BF16).to(D), rnd(tail, seed=2, dtype=BF16).to(D), rnd(tail, seed=3).to(D), rnd(tail, seed=4).to(D).abs()]
    for x, y in zip((p, g, m, v), small):
        x[-tail:] = y
    T.adamw_tensors([p], [g], [m], [v], step=3, lr=1e-2)
    T.adamw_tensors(small[:1], small[1:2], small[2:3], small[3:], step=3, lr=1e-2)
    for x, y in zip((p, m, v), (small[0], small[2], small[3])):
        assert torch.equal(x[-tail:], y) and not x[:1000].any()


def test_adamw_tensors_refusals_on_the_device():
    from image_captioning_amd import _native as N, train_ops as T
    p, g, m, v = (torch.zeros(8, device=D) for _ in range(4))
    s8 = T.adamw_state8(p)
    for bad in (dict(params=[p, p], grads=[g, g], exp_avg=[m, m], exp_avg_sq=[v, v]), dict(params=[p], grads=[g.half()], exp_avg=[m], exp_avg_sq=[v]),
                dict(params=[p], grads=[g[:7]], exp_avg=[m], exp_avg_sq=[v]), dict(params=[p], grads=[g], exp_avg=[s8], exp_avg_sq=[v]),
                dict(params=[p], grads=[g], exp_avg=[m.half()], exp_avg_sq=[v]), dict(params=[p[::2]], grads=[g[::2]], exp_avg=[m[::2]], exp_avg_sq=[v[::2]]),
                dict(params=[p.double()], grads=[g], exp_avg=[m], exp_avg_sq=[v]), dict(params=[p], grads=[g], exp_avg=[(s8[0], s8[1][:0])], exp_avg_sq=[s8])):
        with pytest.raises(N.IcapError):
            T.adamw_tensors(**bad, step=1, lr=1e-3)
    with pytest.raises(N.IcapError):
        T.adamw_tensors([p], [g], [m], [v], step=0, lr=1e-3)
    p2, m2, v2, t8 = torch.zeros_like(p), torch.zeros_like(p), torch.zeros_like(p), T.adamw_state8(p)
    for states in (([m, m], [v, v2]), ([m, m2], [v, m]), ([m, p], [v, v2]), ([s8, T.adamw_state8(p)], [t8, s8])):
        with pytest.raises(N.IcapError, match="twice"):
            T.adamw_tensors([p, p2], [g, g], *states, step=1, lr=1e-3)
    e, e2 = torch.zeros(0, device=D), torch.zeros(0, device=D)
    T.adamw_tensors([p, e, e2], [g, e, e2], [m, e, e2], [v, e, e2], step=1, lr=1e-3)          # empty tensors share an address
    assert not p.any()


def test_packed_ops_refusals_on_the_device():
    from image_captioning_amd import _native as N, ops, train_ops as T
    q, cu = torch.zeros(8, 4, 32, device=D), offsets([8]).to(D)
    for args in ((q, q[:, :3], q[:, :3], cu), (q, q, q[:7], cu), (q, q.half(), q, cu), (q.double(), q.double(), q.double(), cu), (q, q, q, cu.long()),
                 (q, q, q, cu[:1]), (q, q, q, cu, offsets([4, 4]).to(D)), (q[..., :12], q[..., :12], q[..., :12], cu), (q[0], q[0], q[0], cu)):
        with pytest.raises(N.IcapError):
            ops.attention_packed(*args)
    for scale in (0.0, -0.1, math.inf, math.nan):
        with pytest.raises(N.IcapError, match="scale"):
            ops.attention_packed(q, q, q, cu, scale=scale)
    out, lse = ops.attention_packed(q, q, q, cu, want_lse=True)
    for args in ((q[:7], q, q, q, out, lse), (q, q, q, q, out[:, :2], lse), (q, q, q, q, out, lse.half()), (q, q, q, q, out, lse.t())):
        with pytest.raises(N.IcapError):
            T.attention_packed_bwd(*args, cu)
    h, w, t = torch.zeros(4, 16, device=D), torch.zeros(9, 16, device=D), torch.zeros(4, dtype=torch.int64, device=D)
    for args in ((h, w[:, :8], None, t), (h, w.half(), None, t), (h, w, torch.zeros(8, device=D), t), (h, w, None, t.int()), (h, w, None, t[:3]), (h.t(), w, None, t)):
        with pytest.raises(N.IcapError):
            T.linear_ce_fwd(*args)


@pytest.mark.parametrize("dtype", TYPES)
def test_empty_and_smallest_calls(dtype):
    from image_captioning_amd import ops, train_ops as T, training
    for lq, lk in (([0], [0]), ([0, 0], [0, 5]), ([3, 0], [0, 0]), ([1], [1])):
        compare_attention(dtype, lq, lk, 2, 1, 8, True, seed=1)
        compare_attention(dtype, lq, lk, 2, 1, 8, False, seed=2)
    for R, E, V in ((1, 1, 1), (2, 1, 300), (65, 3, 2)):
        compare_ce(dtype, R, E, V, seed=R)
    p = torch.nn.Parameter(rnd(5, seed=1, dtype=dtype).to(D))
    none = torch.nn.Parameter(torch.zeros(0, 4, device=D, dtype=dtype))
    for bits in (8, 32):
        opt = training.AdamWTensors([p, none], lr=1e-2, state_bits=bits)
        opt.step()                                            # no gradients: nothing to do
        p.grad, none.grad = torch.ones_like(p), torch.zeros_like(none)
        before = p.detach().clone()
        opt.step()
        assert opt.param_steps == [1, 1] and (p < before).all()
        opt.zero_grad()
    T.adamw_tensors([], [], [], [], step=1, lr=1e-3)
    # a key head for every query head's own copy: what is expanded is read in place, and its gradient is the copies'
    q, k = rnd(20, 4, 16, seed=3, dtype=dtype).to(D), rnd(20, 1, 16, seed=4, dtype=dtype).to(D)
    wide = k.expand(20, 4, 16)
    cu = offsets([13, 7]).to(D)
    out, lse = ops.attention_packed(q, wide, wide, cu, want_lse=True)
    assert torch.equal(out, ops.attention_packed(q, wide.contiguous(), wide.contiguous(), cu))
    for x, y in zip(T.attention_packed_bwd(out, q, wide, wide, out, lse, cu), T.attention_packed_bwd(out, q, wide.contiguous(), wide.contiguous(), out, lse, cu)):
        assert torch.equal(x, y)


# ------------------------------------------------------------------------------------------------ as they are used
class Decoder(torch.nn.Module):
    """One attention layer over packed captions and an output layer."""

    def __init__(self, V, E, H, K, dtype):
        super().__init__()
        self.H, self.K, self.dim = H, K, E // H
        make = lambda *s, i: torch.nn.Parameter(rnd(*s, seed=i, scale=s[-1] ** -0.5).to(dtype))     # noqa: E731
        self.table, self.w_in, self.w_out, self.head, self.bias = make(V, E, i=1), make((H + 2 * K) * self.dim, E, i=2), make(E, E, i=3), make(V, E, i=4), torch.nn.Parameter(torch.zeros(V, dtype=dtype))

    def hidden(self, ids, cu, attend):
        x = self.table[ids]
        q, k, v = (t.unflatten(1, (-1, self.dim)) for t in (x @ self.w_in.t()).split((self.H * self.dim, self.K * self.dim, self.K * self.dim), 1))
        return x + attend(q, k, v, cu).flatten(1) @ self.w_out.t()


def plain_attend(q, k, v, cu):
    cu = cu.tolist()
    outs = []
    for a, b in zip(cu[:-1], cu[1:]):
        g = q.shape[1] // k.shape[1]
        s = torch.einsum("qhd,khd->hqk", q[a:b], k[a:b].repeat_interleave(g, 1)) * q.shape[2] ** -0.5
        s = s.masked_fill(torch.ones(b - a, b - a, dtype=torch.bool).triu(1), -math.inf)
        outs.append(torch.einsum("hqk,khd->qhd", s.softmax(-1), v[a:b].repeat_interleave(g, 1)))
    return torch.cat(outs)


def test_training_steps_of_a_decoder_on_packed_captions():
    """Attention, loss, gradients and the update together, three steps in fp32 against torch in 64 bits on the CPU (its own AdamW):
    losses, first gradients and parameters."""
    from image_captioning_amd import training
    V, E, H, K, lens = 131, 64, 4, 2, [7, 20, 1, 12]
    ids = torch.randint(0, V, (sum(lens),), generator=torch.Generator().manual_seed(1))
    target = torch.randint(0, V, (sum(lens),), generator=torch.Generator().manual_seed(2))
    target[::9] = -100
    cu = offsets(lens)
    ref = Decoder(V, E, H, K, torch.float64)
    net = Decoder(V, E, H, K, F32).to(D)
    net.load_state_dict({k: v.float() for k, v in ref.state_dict().items()})
    ref.load_state_dict({k: v.double().cpu() for k, v in net.state_dict().items()})
    theirs = torch.optim.AdamW(ref.parameters(), lr=1e-3, weight_decay=0.01)
    mine = training.AdamWTensors(net.parameters(), lr=1e-3, weight_decay=0.01, state_bits=32)
    for step in range(3):
        theirs.zero_grad()
        want = torch.nn.functional.cross_entropy(ref.hidden(ids, cu, plain_attend) @ ref.head.t() + ref.bias, target)
        want.backward()
        mine.zero_grad()
        got = training.linear_cross_entropy(net.hidden(ids.to(D), cu.to(D), training.packed_attention), net.head, net.bias, target.to(D))
        got.backward()
        assert abs(float(got.detach()) - float(want.detach())) < 1e-5 * float(want.detach())
        if step == 0:
            for p, r in zip(net.parameters(), ref.parameters()):
                # fp32 chains of sums of at most 131 terms, some ten products deep: 1e-4 of the gradient's size is far above their roundings
                assert float((p.grad.double().cpu() - r.grad).norm()) < 1e-4 * float(r.grad.norm())
        theirs.step()
        mine.step()
    for p, r in zip(net.parameters(), ref.parameters()):
        # where a gradient's size is that of its own rounding the update's sign is open: three steps of 1e-3 bound every value
        assert float((p.detach().double().cpu() - r.detach()).abs().max()) <= 2 * 3 * 1e-3 * 1.05
        assert float((p.detach().double().cpu() - r.detach()).norm()) < 2e-3 * float(r.detach().norm() + 1e-2)


def test_captured_step_replays_with_new_inputs():
    """Forward, gradients and update through the functional forms recorded in a HIP graph, replayed with new inputs and the step
    count in device memory, eager work between the replays: every replay equals the eager calls."""
    from image_captioning_amd import ops, train_ops as T
    H, K, dim, V, lens = 4, 2, 32, 301, [9, 40, 15]
    n, E = sum(lens), H * dim
    cu = offsets(lens).to(D)

    def inputs(i):
        return rnd(n, H + 2 * K, dim, seed=i, dtype=BF16).to(D), torch.randint(0, V, (n,), generator=torch.Generator().manual_seed(i)).to(D)
    w0 = rnd(V, E, seed=100, scale=E ** -0.5, dtype=BF16).to(D)
    one = torch.ones(1, device=D)

    def step(x, t, w, m, v, **count):
        q, k, val = x.split((H, K, K), 1)
        out, lse = ops.attention_packed(q, k, val, cu, want_lse=True)
        value, _, saved = T.linear_ce_fwd(out.view(n, E), w, None, t)
        dh, dw, _ = T.linear_ce_bwd(one, saved)
        grads = T.attention_packed_bwd(dh.view(n, H, dim), q, k, val, out, lse, cu)
        T.adamw_tensors([w], [dw], [m], [v], seed=3, lr=1e-3, **count)
        return (value, *grads)
    w, m, v = w0.clone(), T.adamw_state8(w0), T.adamw_state8(w0)
    x, t = inputs(0)
    count = torch.zeros(1, dtype=torch.int32, device=D)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                            # a first eager pass on clones, on the stream of the recording
        step(x, t, w.clone(), T.adamw_state8(w0), T.adamw_state8(w0), step=1)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        count += 1
        recorded = step(x, t, w, m, v, step=0, step_dev=count)
    we, me, ve = w0.clone(), T.adamw_state8(w0), T.adamw_state8(w0)
    for i in range(4):
        new = inputs(i)
        x.copy_(new[0])
        t.copy_(new[1])
        graph.replay()
        eager = step(*new, we, me, ve, step=i + 1)
        torch.cuda.synchronize()
        for a, b in zip(recorded, eager):
            assert torch.equal(a, b), f"replay {i}"
        assert torch.equal(m[0].view(torch.uint8), me[0].view(torch.uint8)) and torch.equal(v[0].view(torch.uint8), ve[0].view(torch.uint8))
        # the recorded step computes its bias correction from the count on the device, in the same double precision
        assert torch.equal(w, we)


def test_calls_on_two_streams_at_once():
    from image_captioning_amd import ops, train_ops as T
    q, k, v = (rnd(2000, 4, 64, seed=s, dtype=BF16).to(D) for s in (1, 2, 3))
    cu = offsets([700, 1300]).to(D)
    h, w, t = rnd(500, 128, seed=4, dtype=BF16).to(D), rnd(3000, 128, seed=5, scale=0.1, dtype=BF16).to(D), torch.arange(500, device=D)
    want = ops.attention_packed(q, k, v, cu), T.linear_ce_fwd(h, w, None, t)[0]
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(a):
            x = ops.attention_packed(q, k, v, cu)
            y2 = T.linear_ce_fwd(h, w, None, t)[0]
        with torch.cuda.stream(b):
            y = T.linear_ce_fwd(h, w, None, t)[0]
            x2 = ops.attention_packed(q, k, v, cu)
        torch.cuda.synchronize()
        assert torch.equal(x, want[0]) and torch.equal(x2, want[0]) and torch.equal(y, want[1]) and torch.equal(y2, want[1])


def test_optimizer_state_is_saved_and_loaded():
    from image_captioning_amd import training
    def make():
        return [torch.nn.Parameter(rnd(300, seed=1).to(D)), torch.nn.Parameter(rnd(4, 70, seed=2).to(D))]
    a, b = make(), make()
    A, B = training.AdamWTensors(a, lr=1e-2, seed=4), training.AdamWTensors(b, lr=1.0)

    def go(opt, params, i):
        opt.zero_grad()
        for j, p in enumerate(params):
            p.grad = rnd(*p.shape, seed=10 * i + j).to(D)
        opt.step()
    for i in range(2):
        go(A, a, i)
    B.load_state_dict(A.state_dict())
    for p, q in zip(a, b):
        q.data.copy_(p.data)
    for i in range(2, 4):
        go(A, a, i)
        go(B, b, i)
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and A.param_steps == B.param_steps == [4, 4]
    with pytest.raises(ValueError):
        training.AdamWTensors(b, state_bits=32).load_state_dict(A.state_dict())

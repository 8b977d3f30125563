"""Packed attention where scores are large, against the formulas in 64 bits.

Most cases have whole numbers times powers of two as q and k, so that every score is exact in fp32 whatever the order of its sum:
what is left of a probability's error is its exponent, 2^-24 of at most 150 in a few roundings, and the exponential's, below
`ES` = 2^-15 together.  The roundings to bf16 are counted as everywhere: P and dS before their products, the output that
D = rowsum(dO out) is taken from, the results."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BF, ES = 2.0 ** -8, 2.0 ** -15
INF = math.inf


def _ops():
    from image_to_pointcloud_amd import ops
    return ops


def cu(lens):
    return torch.tensor([0] + list(lens), dtype=torch.int32).cumsum(0).to(torch.int32).cuda()


def inputs(kind, e, tq, tk, heads, kv, seed):
    """q, k, v, dout (bf16, on the device).  ties: scores 2^(2e) times whole numbers around zero; low: the same below zero;
    offset, -offset: whole numbers behind +-2^(2e)."""
    gen = torch.Generator().manual_seed(seed)
    q, k = (torch.randint(-1, 2, (t, h, 64), generator=gen).float() for t, h in ((tq, heads), (tk, kv)))
    if kind == "ties":
        q, k = q * 2.0 ** e, k * 2.0 ** e
    elif kind == "low":
        q, k = q.abs(), -k.abs()
        q[..., 0], k[..., 0] = 1, -1
        q, k = q * 2.0 ** e, k * 2.0 ** e
    else:
        q[..., 0], k[..., 0] = 2.0 ** e, 2.0 ** e * (-1 if kind[0] == "-" else 1)
    v, dout = (torch.randn(t, h, 64, generator=gen) for t, h in ((tk, kv), (tq, heads)))
    return tuple(t.to(torch.bfloat16).cuda() for t in (q, k, v, dout))


def reference(q, k, v, ql, kl, causal, scale, dout=None, starts=None, rounded=0.0, es=None):
    """Values and bounds.  rounded: the share of |lse| by which a probability of the backward pass may be off; es: a function of
    the summed magnitudes of a score's terms instead of ES."""
    q, k, v = (t.double().cpu() for t in (q, k, v))
    H, Hk = q.shape[1], k.shape[1]
    names = [("out", q)]
    r = {"lse": torch.full(q.shape[:2], -INF, dtype=torch.float64)}
    if dout is not None:
        dout = dout.double().cpu()
        names += [("dq", q), ("dk", k), ("dv", v)]
    for n, t in names:
        r[n], r[n + "_b"] = torch.zeros_like(t), torch.zeros_like(t)
    r["lse_b"] = torch.zeros_like(r["lse"])
    q0 = k0 = 0
    for b, (a, n) in enumerate(zip(ql, kl)):
        if starts is not None:
            k0 = starts[b]
        for h in range(H if a and n else 0):
            g = h // (H // Hk)
            rows, keys = slice(q0, q0 + a), slice(k0, k0 + n)
            Q, K, V = q[rows, h], k[keys, g], v[keys, g]
            S = scale * (Q @ K.T)
            on = torch.ones(a, n, dtype=torch.bool)
            if causal:
                on = torch.arange(n)[None, :] <= torch.arange(a)[:, None] + n - a
            S = S.masked_fill(~on, -INF)
            top = S.amax(1, keepdim=True)
            top = torch.where(top == -INF, torch.zeros_like(top), top)
            W = torch.exp(S - top)
            total = W.sum(1, keepdim=True)
            P = W / torch.where(total == 0, torch.ones_like(total), total)
            lse = (top + torch.log(total))[:, 0]
            A, O = P @ V.abs(), P @ V
            e = torch.full_like(total, ES) if es is None else es((P * (scale * (Q.abs() @ K.abs().T))).sum(1, keepdim=True))
            r["out"][rows, h], r["lse"][rows, h] = O, lse
            r["out_b"][rows, h] = BF * O.abs() + (BF * 1.02 + 2 * e) * A
            # scale log2(e), its product with the reference, the sum with log2 of the sum, ln 2: a half step each
            r["lse_b"][rows, h] = 2.0 ** -22 * lse.abs().nan_to_num(posinf=0.0, neginf=0.0) + 2.0 ** -18 + e[:, 0]
            if dout is not None:
                e = e + rounded * lse.abs().nan_to_num(posinf=0.0)[:, None]
                G = dout[rows, h]
                r["dv"][keys, g] += P.T @ G
                r["dv_b"][keys, g] += P.T @ ((BF * 1.02 + 2 * e) * G.abs())
                D, dP = (G * O).sum(1, keepdim=True), G @ V.T
                eD = (G.abs() * r["out_b"][rows, h]).sum(1, keepdim=True) * 1.02
                Z = P * (dP - D)
                eZ = 1.02 * (BF * Z.abs() + P * eD + 3 * e * P * (G.abs() @ V.abs().T + D.abs()))
                r["dq"][rows, h] = scale * Z @ K
                r["dq_b"][rows, h] = scale * 1.02 * (eZ @ K.abs() + ES * (Z.abs() @ K.abs()))
                r["dk"][keys, g] += scale * Z.T @ Q
                r["dk_b"][keys, g] += scale * 1.02 * (eZ.T @ Q.abs() + ES * (Z.abs().T @ Q.abs()))
        q0, k0 = q0 + a, k0 + n
    if dout is not None:
        for n in ("dq", "dk", "dv"):
            r[n + "_b"] += BF * r[n].abs()
    return r


def inside(got, r, name, rows=slice(None)):
    got, want, bound = got.detach().double().cpu()[rows], r[name][rows], r[name + "_b"][rows]
    off = (got - want).abs()
    ok = (got == want) | (off <= bound + 1e-30)
    assert ok.all(), (f"{name}: {int((~ok).sum())} of {ok.numel()} values off, worst by {((off - bound)[~ok]).max():.3e} "
                      f"(NaN: {int(got.isnan().sum())})")


# scores of 2^35, 2^28, 2^40 and 2^64 by the operands or the scale; of -2^36 and below; around +-2^19 a few steps apart
KINDS = [("ties", 16, 0.125), ("ties", 0, 2.0 ** 28), ("ties", 0, 2.0 ** 40), ("ties", 0, 2.0 ** 64), ("low", 16, 0.125),
         ("low", 20, 2.0 ** 64), ("offset", 11, 0.125), ("-offset", 11, 0.125)]
IDS = [f"{n}-{e}-{math.log2(s):g}" for n, e, s in KINDS]


@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("kind,e,scale", KINDS, ids=IDS)
def test_large_scores(kind, e, scale, causal):
    """One tile, a pack that fills the chip, keys in shares."""
    ops = _ops()
    for ql, kl, heads, kv in (([200, 31], [200, 31], 2, 2), ([100], [3000], 2, 2), ([3, 17], [400, 30], 4, 2),
                              ([577, 130, 577, 1, 577, 577, 577, 0, 577, 577], None, 26, 26)):
        kl = kl or ql
        q, k, v, _ = inputs(kind, e, sum(ql), sum(kl), heads, kv, heads)
        out, lse = ops.attention_packed(q, k, v, cu(ql), cu(kl), scale=scale, causal=causal)
        r = reference(q, k, v, ql, kl, causal, scale)
        inside(out, r, "out"), inside(lse, r, "lse")


@pytest.mark.parametrize("kind,e,scale", KINDS, ids=IDS)
def test_large_scores_over_a_cache(kind, e, scale):
    """Single tokens and short chunks over slabs, whose keys are walked in shares of unlike numbers of keys."""
    ops = _ops()
    slab = 6200
    for ql, lens in (([1, 1, 1], [300, 6011, 700]), ([1], [300]), ([3, 1, 0, 9], [2000, 1, 40, 5003])):
        q, k, v, _ = inputs(kind, e, sum(ql), slab * len(ql), 8, 2, len(ql))
        out, lse = ops.attention_packed(q, k, v, cu(ql), cu([slab] * len(ql)), k_lens=torch.tensor(lens, dtype=torch.int32).cuda(),
                                        scale=scale, causal=True)
        r = reference(q, k, v, ql, lens, True, scale, starts=[b * slab for b in range(len(ql))])
        inside(out, r, "out"), inside(lse, r, "lse")


@pytest.mark.parametrize("kind,e,scale", KINDS, ids=IDS)
def test_large_scores_before_a_masked_nan(kind, e, scale):
    """The rows that a NaN behind the mask has done again."""
    ops = _ops()
    q, k, v, _ = inputs(kind, e, 180, 180, 2, 1, 5)
    r = reference(q, k, v, [180], [180], True, scale)
    k[179], v[179] = float("nan"), float("nan")
    out, lse = ops.attention_packed(q, k, v, cu([180]), scale=scale, causal=True)
    inside(out, r, "out", slice(0, 179)), inside(lse, r, "lse", slice(0, 179))


def test_scores_beyond_the_largest_float():
    """Scaled scores of about 2^131: the softmax is of their differences, lse is the nearest fp32 has."""
    ops = _ops()
    q, k, v, _ = inputs("low", 32, 70, 70, 1, 1, 3)
    for sign in (1, -1):
        r = reference(q, sign * k, v, [70], [70], False, 2.0 ** 64)
        out, lse = ops.attention_packed(q, sign * k, v, cu([70]), scale=2.0 ** 64)
        inside(out, r, "out")
        # above the largest float infinity; -inf is a query that sees no key
        over = r["lse"].abs() > 2.0 ** 128
        assert over.any() and ((lse.cpu() == INF) if sign < 0 else (lse.cpu() == -torch.finfo(torch.float32).max))[over].all()


@pytest.mark.parametrize("rows,heads", [(1, 8), (70, 2), (577, 40)])
def test_scores_beyond_the_largest_float_behind_minus_infinity(rows, heads):
    """A row whose first scores are all -inf takes the others as they are, however low."""
    ops = _ops()
    q, k, v, _ = inputs("low", 32, rows, 100, heads, heads, 3)
    k[:40, :, 0] = -INF
    for causal in (False, True):
        if causal and rows > 100:
            continue
        r = reference(q, k[40:], v[40:], [rows], [60], causal, 2.0 ** 64)
        out, lse = ops.attention_packed(q, k, v, cu([rows]), cu([100]), scale=2.0 ** 64, causal=causal)
        seen = slice(max(0, rows - 60) if causal else 0, rows)
        inside(out, r, "out", seen)
        assert (lse.cpu()[seen] < -(2.0 ** 126)).all() and torch.isfinite(lse.cpu()[seen]).all()


# ------------------------------------------------------------------ gradients
# besides: lse of 2^13, below the size from which rows are done again, and 2^15, above it
GRAD_KINDS = KINDS + [("offset", 8, 0.125), ("offset", 9, 0.125), ("-offset", 9, 0.125)]
GRAD_IDS = [f"{n}-{e}-{math.log2(s):g}" for n, e, s in GRAD_KINDS]
# Where a probability of the backward pass is exp(S - lse): lse's rounding, those of lse / scale, of its products with the scale and
# log2(e), and the sums of the score's products that start at it
ROUNDED = 2.0 ** -20


def gradients(q, k, v, dout, ql, kl, causal, scale, **kw):
    ops = _ops()
    out, lse = ops.attention_packed(q, k, v, cu(ql), cu(kl), scale=scale, causal=causal)
    got = ops.attention_packed_backward(dout, q, k, v, out, lse, cu(ql), cu(kl), scale=scale, causal=causal)
    r = reference(q, k, v, ql, kl, causal, scale, dout, **kw)
    return dict(zip(("dq", "dk", "dv"), got)), r


@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("kind,e,scale", GRAD_KINDS, ids=GRAD_IDS)
def test_gradients_of_large_scores(kind, e, scale, causal):
    """Few tiles and many, heads of a group apart and together, rows of few keys."""
    for ql, kl, heads, kv in (([200, 31], [200, 31], 2, 2), ([100, 3], [30, 400], 4, 2),
                              ([577, 130, 577, 1, 577, 577, 577, 0, 577, 577], None, 26, 26), ([300] * 12, None, 24, 6)):
        kl = kl or ql
        q, k, v, dout = inputs(kind, e, sum(ql), sum(kl), heads, kv, heads + 1)
        got, r = gradients(q, k, v, dout, ql, kl, causal, scale, rounded=ROUNDED if e == 8 else 0.0)
        for n, t in got.items():
            inside(t, r, n)


@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
def test_gradients_of_large_and_small_scores_together(causal):
    """Rows of either kind in a tile: what the one needs leaves the other's gradients right."""
    q, k, v, dout = inputs("offset", 11, 180, 180, 4, 2, 9)
    q[::3] = 0
    got, r = gradients(q, k, v, dout, [180], [180], causal, 0.125)
    for n, t in got.items():
        inside(t, r, n)


def test_gradients_of_large_scores_before_a_masked_nan():
    ops = _ops()
    q, k, v, dout = inputs("ties", 16, 180, 180, 2, 1, 5)
    c = cu([180])
    out, lse = ops.attention_packed(q, k, v, c, scale=0.125, causal=True)
    r = reference(q, k, v, [180], [180], True, 0.125, dout)
    q2, d2, k2, v2 = (t.clone() for t in (q, dout, k, v))
    q2[20], d2[20], k2[150], v2[150] = (float("nan"),) * 4
    _, dk, dv = ops.attention_packed_backward(d2, q2, k, v, out, lse, c, scale=0.125, causal=True)
    inside(dk, r, "dk", slice(21, 180)), inside(dv, r, "dv", slice(21, 180))
    dq, _, _ = ops.attention_packed_backward(dout, q, k2, v2, out, lse, c, scale=0.125, causal=True)
    inside(dq, r, "dq", slice(0, 150))


@pytest.mark.parametrize("size", [4.0, 8.0, 16.0])
def test_gradients_of_peaked_scores(size):
    """Ordinary values of some size: scores of some hundreds whose sums round, and an lse that rounds as much."""
    gen = torch.Generator().manual_seed(4)
    q, k, v, dout = ((s * torch.randn(195, 2, 64, generator=gen)).to(torch.bfloat16).cuda() for s in (size, size, 1.0, 1.0))
    for causal in (False, True):
        got, r = gradients(q, k, v, dout, [130, 65], [130, 65], causal, 0.125, rounded=ROUNDED,
                           es=lambda mag: ES * (1 + mag))
        for n, t in got.items():
            inside(t, r, n)


@pytest.mark.parametrize("rows", [5, 64, 150])
def test_keys_of_scores_of_minus_infinity_have_no_gradient(rows):
    """Nothing of theirs is in the output: dk and dv are 0, also where a tile ends behind the last query."""
    ops = _ops()
    gen = torch.Generator().manual_seed(4)
    q, k, v, dout = (torch.randn(n, 2, 64, generator=gen).to(torch.bfloat16).cuda() for n in (rows, 100, 100, rows))
    q = q.abs() + 0.5
    k[:70, :, 0] = -INF
    out, lse = ops.attention_packed(q, k, v, cu([rows]), cu([100]))
    _, dk, dv = ops.attention_packed_backward(dout, q, k, v, out, lse, cu([rows]), cu([100]))
    assert not dk[:70].any() and not dv[:70].any()
    r = reference(q, k[70:], v[70:], [rows], [30], False, 0.125, dout, es=lambda mag: ES * (1 + mag))
    inside(dk[70:], r, "dk"), inside(dv[70:], r, "dv")

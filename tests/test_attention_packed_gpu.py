"""Attention over packed sequences and its gradients, against the formulas in 64 bits.

Bounds count roundings, value by value.  The products take bf16 operands and sum in fp32; what is rounded to bf16 (half a
step: 2^-8 of the value) besides the outputs is P before P V and P^T dO, dS before dS K and dS^T Q, and the `out` that
D = rowsum(dO out) is taken from.  `F` = 2^-15 of the summed magnitudes covers the fp32 part: sums of some thousand terms
in blocks of 16, and exponents c (s - m) of size up to 2^6 that are rounded to 2^-24 of their size."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BF, F = 2.0 ** -8, 2.0 ** -15
INF = math.inf


def _ops():
    from image_to_pointcloud_amd import ops
    return ops


def cu(lens):
    return torch.tensor([0] + list(lens), dtype=torch.int32).cumsum(0).to(torch.int32).cuda()


def make(ql, kl=None, heads=2, kv=None, seed=0, layout="rows", extra=(0, 0), size=1.0):
    """q, k, v, dout on the device.  layout: rows [T, H, 64]; heads [H, T, 64] underneath; wide: slices of one buffer."""
    kl = ql if kl is None else kl
    kv = kv or heads
    gen = torch.Generator().manual_seed(seed)
    tq, tk = sum(ql) + extra[0], sum(kl) + extra[1]

    def one(t, h):
        x = (size * torch.randn(t, h, 64, generator=gen)).to(torch.bfloat16).cuda()
        if layout == "heads":
            return x.transpose(0, 1).contiguous().transpose(0, 1)
        if layout == "wide":
            w = torch.full((t, h + 1, 72), 3.0, dtype=torch.bfloat16, device="cuda")
            w[:, :h, :64] = x
            return w[:, :h, :64]
        return x
    return one(tq, heads), one(tk, kv), one(tk, kv), one(tq, heads)


def reference(q, k, v, ql, kl, causal, scale, dout=None, starts=None, short=0):
    """Values and, for each output, the bound on its error; rows behind the sequences are zero.  short: sequences of up to
    that many keys have D from fp32 sums instead of the rounded output."""
    q, k, v = (t.double().cpu() for t in (q, k, v))
    H, Hk = q.shape[1], k.shape[1]
    r = {"out": torch.zeros_like(q), "out_b": torch.zeros_like(q), "lse": torch.full(q.shape[:2], -INF, dtype=torch.float64),
         "lse_b": torch.zeros(q.shape[:2], dtype=torch.float64)}
    if dout is not None:
        dout = dout.double().cpu()
        for n, t in (("dq", q), ("dk", k), ("dv", v)):
            r[n], r[n + "_b"] = torch.zeros_like(t), torch.zeros_like(t)
    q0 = k0 = 0
    for b, (a, n) in enumerate(zip(ql, kl)):
        if starts is not None:
            k0 = starts[b]
        for h in range(H if a and n else 0):
            g = h // (H // Hk)
            rows, keys = slice(q0, q0 + a), slice(k0, k0 + n)
            Q, K, V = q[rows, h], k[keys, g], v[keys, g]
            S = scale * Q @ K.T
            on = torch.ones(a, n, dtype=torch.bool)
            if causal:
                on = torch.arange(n)[None, :] <= torch.arange(a)[:, None] + n - a
            S = S.masked_fill(~on, -INF)
            lse = torch.logsumexp(S, 1)
            P = torch.where(on, torch.exp(S - torch.where(lse == -INF, torch.zeros_like(lse), lse)[:, None]), 0.0)
            mag = scale * (Q.abs() @ K.abs().T)                  # of a score's terms
            A = P @ V.abs()
            O = P @ V
            es = F * (1 + (P * mag).sum(1, keepdim=True))         # relative error of a probability
            r["out"][rows, h], r["lse"][rows, h] = O, lse
            r["out_b"][rows, h] = BF * O.abs() + (BF * 1.02 + 2 * es) * A
            r["lse_b"][rows, h] = 2.0 ** -18 * (1 + (P * mag).sum(1) + lse.abs().nan_to_num(posinf=0.0))
            if dout is not None:
                G = dout[rows, h]
                r["dv"][keys, g] += P.T @ G
                r["dv_b"][keys, g] += P.T @ ((BF * 1.02 + 2 * es) * G.abs())
                D = (G * O).sum(1, keepdim=True)
                eD = (G.abs() * r["out_b"][rows, h]).sum(1, keepdim=True) * 1.02
                if n <= short:
                    eD = 3 * es * (P * (G.abs() @ V.abs().T)).sum(1, keepdim=True)
                dP = G @ V.T
                Z = P * (dP - D)
                eZ = 1.02 * (BF * Z.abs() + P * eD + 3 * es * P * (G.abs() @ V.abs().T + D.abs()))
                r["dq"][rows, h] = scale * Z @ K
                r["dq_b"][rows, h] = scale * 1.02 * (eZ @ K.abs()) + F * scale * (Z.abs() @ K.abs())
                r["dk"][keys, g] += scale * Z.T @ Q
                r["dk_b"][keys, g] += scale * 1.02 * (eZ.T @ Q.abs()) + F * scale * (Z.abs().T @ Q.abs())
        q0, k0 = q0 + a, k0 + n
    if dout is not None:
        for n in ("dq", "dk", "dv"):
            r[n + "_b"] += BF * r[n].abs() + 1e-30
    return r


def inside(got, want, bound, what):
    got = got.detach().double().cpu()
    same = (got == want) | (got.isnan() & want.isnan())
    off = (got - want).abs()
    ok = same | (off <= bound + 1e-30)
    assert ok.all(), f"{what}: {int((~ok).sum())} of {ok.numel()} values off, worst by {((off - bound)[~ok]).max():.3e} (NaN: {int(got.isnan().sum())})"


def check(ql, kl=None, heads=2, kv=None, causal=False, scale=None, seed=0, layout="rows", backward=True, extra=(0, 0), size=1.0):
    ops = _ops()
    q, k, v, dout = make(ql, kl, heads, kv, seed, layout, extra, size)
    kl_ = ql if kl is None else kl
    cq, ck = cu(ql), None if kl is None else cu(kl)
    out, lse = ops.attention_packed(q, k, v, cq, ck, scale=scale, causal=causal)
    ref = reference(q, k, v, ql, kl_, causal, 0.125 if scale is None else scale, dout if backward else None)
    inside(out, ref["out"], ref["out_b"], "out")
    inside(lse, ref["lse"], ref["lse_b"], "lse")
    if backward:
        got = ops.attention_packed_backward(dout, q, k, v, out, lse, cq, ck, scale=scale, causal=causal)
        for n, t in zip(("dq", "dk", "dv"), got):
            inside(t, ref[n], ref[n + "_b"], n)
    return q, k, v, dout, out, lse


@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 257, 577])
def test_one_sequence(n, causal):
    check([n], causal=causal, seed=n)


@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("heads,kv", [(1, 1), (6, 6), (4, 2), (8, 1), (6, 2), (5, 1), (12, 4)])
def test_packs_and_grouped_heads(heads, kv, causal):
    check([1, 70, 0, 33, 129, 64, 0, 2], heads=heads, kv=kv, causal=causal, seed=heads * 7 + kv)


@pytest.mark.parametrize("heads,kv,causal", [(16, 16, False), (26, 26, True), (24, 6, False), (24, 6, True), (24, 12, True)])
def test_many_workgroups(heads, kv, causal):
    """Packs that fill the chip take other tiles than small ones: 128 rows or keys a workgroup, heads of a group apart or
    together."""
    check([577, 577, 130, 577, 1, 577, 33, 577, 0, 577, 577, 577], heads=heads, kv=kv, causal=causal, seed=heads + kv, extra=(40, 40))


def test_chunks_over_slabs():
    """Long chunks at the end of caches, NaN behind the filled slots."""
    ops = _ops()
    ql, lens, slab = [300, 1, 900, 77], [1500, 640, 901, 77], 1600
    q, k, v, _ = make(ql, [slab] * 4, 8, 2, seed=14)
    for b, n in enumerate(lens):
        k[b * slab + n:(b + 1) * slab] = float("nan")
        v[b * slab + n:(b + 1) * slab] = float("nan")
    for causal in (True, False):
        out, lse = ops.attention_packed(q, k, v, cu(ql), cu([slab] * 4), k_lens=torch.tensor(lens, dtype=torch.int32).cuda(),
                                        causal=causal)
        ref = reference(q, k, v, ql, lens, causal, 0.125, starts=[b * slab for b in range(4)])
        inside(out, ref["out"], ref["out_b"], "out")
        inside(lse, ref["lse"], ref["lse_b"], "lse")


def test_more_query_heads_than_a_row_block():
    """40 query heads over one key head: a position's rows lie in two blocks of 32."""
    check([1, 20, 0, 37], heads=40, kv=1, causal=True, seed=3)
    check([90], heads=72, kv=2, seed=4)


def test_heads_that_share_memory():
    """Keys and values broadcast over the heads (head stride 0) are those of one grouped key head, and their gradients are
    the query heads' own."""
    ops = _ops()
    q, k, v, dout = make([70, 9], heads=4, kv=1, seed=8)
    c = cu([70, 9])
    ke, ve = k.expand(79, 4, 64), v.expand(79, 4, 64)
    out, lse = ops.attention_packed(q, ke, ve, c, causal=True)
    ref = reference(q, ke, ve, [70, 9], [70, 9], True, 0.125, dout)
    inside(out, ref["out"], ref["out_b"], "out")
    for n, t in zip(("dq", "dk", "dv"), ops.attention_packed_backward(dout, q, ke, ve, out, lse, c, causal=True)):
        inside(t, ref[n], ref[n + "_b"], n)


def test_one_tensor_as_all_three():
    ops = _ops()
    x, _, _, dout = make([100, 31], heads=2, seed=9)
    c = cu([100, 31])
    a, la = ops.attention_packed(x, x, x, c)
    b, lb = ops.attention_packed(x, x.clone(), x.clone(), c)
    assert torch.equal(a, b) and torch.equal(la, lb)
    for s, t in zip(ops.attention_packed_backward(dout, x, x, x, a, la, c),
                    ops.attention_packed_backward(dout, x, x.clone(), x.clone(), b, lb, c)):
        assert torch.equal(s, t)


@pytest.mark.parametrize("layout", ["heads", "wide"])
def test_strides(layout):
    check([40, 100, 3], heads=4, kv=2, causal=True, layout=layout, seed=5)


def test_slices_of_a_qkv_buffer():
    ops = _ops()
    qkv = torch.randn(150, 3, 3, 64, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    q, k, v = qkv[:, 0], qkv[:, 1], qkv[:, 2]
    c = cu([100, 50])
    out, lse = ops.attention_packed(q, k, v, c)
    o2, l2 = ops.attention_packed(q.contiguous(), k.contiguous(), v.contiguous(), c)
    assert torch.equal(out, o2) and torch.equal(lse, l2)
    # gradients into the slices of a buffer of the same layout
    dqkv = torch.zeros_like(qkv)
    dout = torch.ones_like(out)
    ops.attention_packed_backward(dout, q, k, v, out, lse, c, dq=dqkv[:, 0], dk=dqkv[:, 1], dv=dqkv[:, 2])
    for a, b in zip(ops.attention_packed_backward(dout, q, k, v, out, lse, c), dqkv.unbind(1)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("ql,kl,causal", [([1, 1, 1], [70, 1, 300], True), ([5, 0, 130, 3], [70, 9, 300, 3], True),
                                          ([70, 9], [5, 0], True), ([70, 9, 200], [5, 0, 129], False), ([0, 0], [5, 70], True),
                                          ([300], [3], True), ([129, 40], [100, 41], True)])
def test_other_lengths_of_queries_and_keys(ql, kl, causal):
    """Chunks behind a longer past, queries without a key (causal, fewer keys than queries), keys without a query."""
    check(ql, kl, heads=4, kv=2, causal=causal, seed=sum(ql) + sum(kl))


def test_same_as_the_fixed_length_kernel():
    """Sequences of one length: the networks' attention gives the same values but for its rounding of P."""
    ops = _ops()
    B, T, H = 2, 197, 3
    qkv = torch.randn(B * T, 3, H, 64, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
    out, _ = ops.attention_packed(qkv[:, 0], qkv[:, 1], qkv[:, 2], cu([T] * B))
    fixed = ops.attention(qkv.view(B * T, -1), B, T, H, 0.125).view(B * T, H, 64)
    ref = reference(qkv[:, 0], qkv[:, 1], qkv[:, 2], [T] * B, [T] * B, False, 0.125)
    inside(out.float(), fixed.double().cpu(), 2 * ref["out_b"], "out against attention()")


def test_many_sequences():
    """More sequences than one step of the tile lookup holds, most of them short, some empty."""
    gen = torch.Generator().manual_seed(8)
    lens = torch.randint(0, 6, (4200,), generator=gen).tolist()
    lens[17], lens[4100] = 150, 70
    check(lens, heads=1, causal=True, seed=9)


@pytest.mark.parametrize("scale,size", [(0.5, 1.0), (0.125, 8.0), (1e-3, 1.0)])
def test_scales_and_peaked_scores(scale, size):
    check([130, 65], heads=2, causal=True, scale=scale, size=size, seed=4, backward=size < 4)


def test_scores_that_rise_along_the_keys():
    """Each block of keys far above the ones before it: every block moves the reference."""
    ops = _ops()
    q, k, v, _ = make([200], heads=1, seed=1)
    k = (k.float() * 0.1 + torch.arange(200, device="cuda")[:, None, None] * 0.4 * q[:1].float() / 8).to(torch.bfloat16)
    for causal in (False, True):
        out, lse = ops.attention_packed(q, k, v, cu([200]), causal=causal)
        ref = reference(q, k, v, [200], [200], causal, 0.125)
        inside(out, ref["out"], ref["out_b"], "out")
        inside(lse, ref["lse"], ref["lse_b"], "lse")


@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("batch", [6, 160])
def test_gradients_of_rows_with_few_keys(batch, causal):
    """Their D is not that of the rounded output: nearly all of dP may cancel against it.  (Few and many row tiles.)"""
    ops = _ops()
    ql, kl = [64, 2, 33, 5, 150, 17][:batch] + [60] * (batch - 6), [64, 2, 33, 7, 40, 64][:batch] + [60] * (batch - 6)
    q, k, v, dout = make(ql, kl, heads=8, kv=2, seed=13)
    out, lse = ops.attention_packed(q, k, v, cu(ql), cu(kl), causal=causal)
    got = ops.attention_packed_backward(dout, q, k, v, out, lse, cu(ql), cu(kl), causal=causal)
    ref = reference(q, k, v, ql, kl, causal, 0.125, dout, short=64)
    for n, t in zip(("dq", "dk", "dv"), got):
        inside(t, ref[n], ref[n + "_b"], n)


# ------------------------------------------------------------------ one token over a cache
@pytest.mark.parametrize("heads,kv", [(1, 1), (4, 1), (16, 4), (8, 8), (6, 2), (40, 1)])
@pytest.mark.parametrize("lens", [[1], [64], [777], [0, 5, 300, 64, 65, 1], [3000, 2, 0, 1025]])
def test_one_token_over_slabs(lens, heads, kv):
    ops = _ops()
    slab = 3100
    B = len(lens)
    q, k, v, _ = make([1] * B, [slab] * B, heads, kv, seed=len(lens) + heads)
    # what lies behind a sequence's end in its slab is of no use: here it is NaN and infinite
    for b, n in enumerate(lens):
        k[b * slab + n:(b + 1) * slab] = float("nan")
        v[b * slab + n:(b + 1) * slab] = float("inf")
    starts = [b * slab for b in range(B)]
    out, lse = ops.attention_packed(q, k, v, cu([1] * B), cu([slab] * B), k_lens=torch.tensor(lens, dtype=torch.int32).cuda(),
                                    causal=True)
    ref = reference(q, k, v, [1] * B, lens, True, 0.125, starts=starts)
    inside(out, ref["out"], ref["out_b"], "out")
    inside(lse, ref["lse"], ref["lse_b"], "lse")


def test_a_few_tokens_over_slabs():
    """Short chunks of different lengths at the end of their caches."""
    ops = _ops()
    ql, lens, slab = [3, 1, 0, 40, 7], [700, 64, 9, 1000, 5], 1024
    q, k, v, _ = make(ql, [slab] * 5, 8, 2, seed=12)
    out, lse = ops.attention_packed(q, k, v, cu(ql), cu([slab] * 5), k_lens=torch.tensor(lens, dtype=torch.int32).cuda(), causal=True)
    ref = reference(q, k, v, ql, lens, True, 0.125, starts=[b * slab for b in range(5)])
    inside(out, ref["out"], ref["out_b"], "out")
    inside(lse, ref["lse"], ref["lse_b"], "lse")


def test_lengths_beyond_the_slab_are_held():
    ops = _ops()
    q, k, v, _ = make([1, 1], [100, 100], 2, 2, seed=1)
    a = ops.attention_packed(q, k, v, cu([1, 1]), cu([100, 100]), k_lens=torch.tensor([100, 100], dtype=torch.int32).cuda())
    b = ops.attention_packed(q, k, v, cu([1, 1]), cu([100, 100]), k_lens=torch.tensor([4000, 2 ** 30], dtype=torch.int32).cuda())
    c = ops.attention_packed(q, k, v, cu([1, 1]), cu([100, 100]), k_lens=torch.tensor([-3, 0], dtype=torch.int32).cuda())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert not c[0].any() and (c[1] == -INF).all()


def test_offsets_beyond_32_bits():
    """A sequence whose keys lie more than 4 GiB after their start: every row pitch is 2^22 values, 8 MiB."""
    ops = _ops()
    n, pitch = 600, 1 << 22
    buf = torch.empty(n * pitch, dtype=torch.bfloat16, device="cuda")          # 4.7 GiB, only the rows are written
    k = buf.as_strided((n, 1, 64), (pitch, 64, 1))
    v = buf.as_strided((n, 1, 64), (pitch, 64, 1), 64)
    q, k0, v0, dout = make([n], heads=1, seed=6)
    k.copy_(k0), v.copy_(v0)
    for causal in (False, True):
        out, lse = ops.attention_packed(q, k, v, cu([n]), causal=causal)
        o2, l2 = ops.attention_packed(q, k0, v0, cu([n]), causal=causal)
        assert torch.equal(out, o2) and torch.equal(lse, l2)
        for a, b in zip(ops.attention_packed_backward(dout, q, k, v, out, lse, cu([n]), causal=causal),
                        ops.attention_packed_backward(dout, q, k0, v0, o2, l2, cu([n]), causal=causal)):
            assert torch.equal(a, b)
    one = ops.attention_packed(q[:1], k, v, cu([1]), cu([n]))
    two = ops.attention_packed(q[:1], k0, v0, cu([1]), cu([n]))
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])


# ------------------------------------------------------------------ what is masked has no say
@pytest.mark.parametrize("bad", [float("nan"), INF, -INF])
def test_nonfinite_future_keys(bad):
    """Non-finite rows that a causal mask hides reach no earlier query, and no gradient of an earlier key or query."""
    ops = _ops()
    ql = [150, 90]
    q, k, v, dout = make(ql, heads=4, kv=2, seed=3)
    c = cu(ql)
    ref = reference(q, k, v, ql, ql, True, 0.125)
    for at in (149, 70):                                     # the first sequence's last position, one in its middle
        k2, v2 = k.clone(), v.clone()
        k2[at], v2[at] = bad, bad
        out, lse = ops.attention_packed(q, k2, v2, c, causal=True)
        keep = [i for i in range(240) if not at <= i < 150]
        inside(out[keep], ref["out"][keep], ref["out_b"][keep], f"out {at}")
        inside(lse[keep], ref["lse"][keep], ref["lse_b"][keep], f"lse {at}")
        assert not torch.isfinite(out[at].float()).any()


@pytest.mark.parametrize("bad", [float("nan"), INF])
def test_nonfinite_masked_rows_in_the_gradients(bad):
    ops = _ops()
    ql = [150, 90]
    q, k, v, dout = make(ql, heads=4, kv=2, seed=3)
    c = cu(ql)
    out, lse = ops.attention_packed(q, k, v, c, causal=True)
    ref = reference(q, k, v, ql, ql, True, 0.125, dout)
    # queries before key j do not see it: theirs may be anything
    q2, d2 = q.clone(), dout.clone()
    q2[20], d2[20] = bad, bad
    _, dk, dv = ops.attention_packed_backward(d2, q2, k, v, out, lse, c, causal=True)
    keep = [i for i in range(240) if i > 20]
    inside(dk[keep], ref["dk"][keep], ref["dk_b"][keep], "dk")
    inside(dv[keep], ref["dv"][keep], ref["dv_b"][keep], "dv")
    assert not torch.isfinite(dv[5].float()).any()
    # keys behind query i are not seen by it
    k2, v2 = k.clone(), v.clone()
    k2[120], v2[120] = bad, bad
    dq, _, _ = ops.attention_packed_backward(dout, q, k2, v2, out, lse, c, causal=True)
    keep = [i for i in range(240) if not 120 <= i < 150]
    inside(dq[keep], ref["dq"][keep], ref["dq_b"][keep], "dq")


@pytest.mark.parametrize("heads,kv", [(26, 26), (24, 6)])
def test_nonfinite_masked_rows_in_many_workgroups(heads, kv):
    """The same where a pack fills the chip: NaN keys reach only the queries behind them, NaN queries only the keys before."""
    ops = _ops()
    ql = [577, 577, 130, 577, 1, 577, 33, 577, 577, 577, 577]
    q, k, v, dout = make(ql, heads=heads, kv=kv, seed=5)
    c = cu(ql)
    ref = reference(q, k, v, ql, ql, True, 0.125, dout)
    out, lse = ops.attention_packed(q, k, v, c, causal=True)
    T, first, last = sum(ql), 577 + 300, 2 * 577              # the second sequence from its position 300 on
    k2, v2 = k.clone(), v.clone()
    k2[first], v2[first] = float("nan"), float("nan")
    o2, l2 = ops.attention_packed(q, k2, v2, c, causal=True)
    dq, _, _ = ops.attention_packed_backward(dout, q, k2, v2, out, lse, c, causal=True)
    keep = [i for i in range(T) if not first <= i < last]
    for n, t in (("out", o2), ("lse", l2), ("dq", dq)):
        inside(t[keep], ref[n][keep], ref[n + "_b"][keep], n)
        assert t[first:last].isnan().all()
    q2, d2 = q.clone(), dout.clone()
    q2[first], d2[first] = float("nan"), float("nan")
    _, dk, dv = ops.attention_packed_backward(d2, q2, k, v, out, lse, c, causal=True)
    keep = [i for i in range(T) if not 577 <= i <= first]
    for n, t in (("dk", dk), ("dv", dv)):
        inside(t[keep], ref[n][keep], ref[n + "_b"][keep], n)
        assert t[577:first + 1].isnan().all()


def test_nonfinite_neighbours_in_the_pack():
    """A sequence of NaN beside others, and NaN rows behind the last one: only its own rows are."""
    ops = _ops()
    ql, extra = [33, 40, 65], (19, 19)
    for causal in (False, True):
        q, k, v, dout = make(ql, heads=2, seed=1, extra=extra)
        for t in (q, k, v, dout):
            t[33:73] = float("nan")
            t[138:] = float("nan")
        c = cu(ql)
        out, lse = ops.attention_packed(q, k, v, c, causal=causal)
        grads = ops.attention_packed_backward(dout, q, k, v, out, lse, c, causal=causal)
        for t in (q, k, v, dout):
            t[33:73] = 0
            t[138:] = 0
        ref = reference(q, k, v, ql, ql, causal, 0.125, dout)
        keep = list(range(33)) + list(range(73, 138))
        for n, t in zip(("out", "lse", "dq", "dk", "dv"), (out, lse) + tuple(grads)):
            inside(t[keep], ref[n][keep], ref[n + "_b"][keep], n)
            assert t[33:73].isnan().any()
        assert not out[138:].any() and (lse[138:] == -INF).all()
        for t in grads:
            assert not t[138:].any()


def test_rows_behind_the_last_sequence_are_left():
    ops = _ops()
    ql = [1, 1, 50]
    q, k, v, dout = make(ql, heads=2, seed=2, extra=(77, 140))
    c = cu(ql)
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device="cuda")
    lse = torch.full(q.shape[:2], 7.0, device="cuda")
    ops.attention_packed(q, k, v, c, c, out=out, lse=lse)
    assert (out[52:] == 7).all() and (lse[52:] == 7).all() and (out[:52] != 7).any()
    dq, dk, dv = (torch.full(t.shape, 7.0, dtype=torch.bfloat16, device="cuda") for t in (q, k, v))
    ops.attention_packed_backward(dout, q, k, v, out, lse, c, c, dq=dq, dk=dk, dv=dv)
    for t in (dq, dk, dv):
        assert (t[52:] == 7).all() and not (t[:52] == 7).all()
    fresh, flse = ops.attention_packed(q, k, v, c, c)
    assert torch.equal(fresh[:52], out[:52]) and not fresh[52:].any() and (flse[52:] == -INF).all()


def test_split_keys_leave_the_tail_too():
    ops = _ops()
    q, k, v, _ = make([1], [2000], heads=4, kv=1, seed=2, extra=(3, 0))
    args = (q, k, v, cu([1]), cu([2000]))
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device="cuda")
    lse = torch.full(q.shape[:2], 7.0, device="cuda")
    ops.attention_packed(*args, out=out, lse=lse)
    fresh, flse = ops.attention_packed(*args)
    assert (out[1:] == 7).all() and (lse[1:] == 7).all()
    assert not fresh[1:].any() and (flse[1:] == -INF).all() and torch.equal(fresh[0], out[0])


def test_no_keys_or_no_queries_at_all():
    ops = _ops()
    q, k, v, dout = make([3, 2], [0, 0], heads=2, seed=2)
    c, z = cu([3, 2]), cu([0, 0])
    out, lse = ops.attention_packed(q, k, v, c, z)
    assert not out.any() and (lse == -INF).all()
    dq, dk, dv = ops.attention_packed_backward(dout, q, k, v, out, lse, c, z)
    assert not dq.any() and dk.shape == k.shape
    q, k, v, dout = make([0, 0], [3, 70], heads=2, seed=2)
    out, lse = ops.attention_packed(q, k, v, z, cu([3, 70]))
    dq, dk, dv = ops.attention_packed_backward(dout, q, k, v, out, lse, z, cu([3, 70]))
    assert out.shape == q.shape and not dk.any() and not dv.any()


@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("rows", [1, 70])
def test_scores_of_minus_infinity(rows, causal):
    """Keys whose visible scores are -inf have probability 0, also where they are a row's first ones and every other score
    is far below zero; with a NaN behind the mask too, where the row is done again."""
    ops = _ops()
    n = 300
    q, k, v, _ = make([rows], [n], heads=2, seed=4)
    q, k = q.abs() + 0.5, -k.abs() * 16 - 8                   # scores of some hundreds below zero
    k[:70, :, 0] = -INF
    c = (cu([rows]), cu([n]))
    ref = reference(q[:, :], k[70:], v[70:], [rows], [n - 70], causal, 0.125)
    out, lse = ops.attention_packed(q, k, v, *c, causal=causal)
    inside(out, ref["out"], ref["out_b"], "out")
    inside(lse, ref["lse"], ref["lse_b"], "lse")
    if causal and rows > 1:
        k[n - 1], v[n - 1] = float("nan"), float("nan")       # the last query's own
        out, lse = ops.attention_packed(q, k, v, *c, causal=True)
        inside(out[:-1], ref["out"][:-1], ref["out_b"][:-1], "out")
        inside(lse[:-1], ref["lse"][:-1], ref["lse_b"][:-1], "lse")


# ------------------------------------------------------------------ how it is called
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("batch", [16, 17, 64, 65, 200])
def test_numbers_of_sequences(batch, causal):
    """Either side of the sizes at which the lookup of a tile changes, with rows behind the last sequence."""
    gen = torch.Generator().manual_seed(batch)
    ql = torch.randint(0, 40, (batch,), generator=gen).tolist()
    kl = torch.randint(0, 60, (batch,), generator=gen).tolist()
    ql[0], kl[1], ql[-1], kl[-1] = 0, 0, 141, 150
    q, k, v, dout, out, lse = check(ql, kl, heads=2, kv=1, causal=causal, seed=batch, extra=(150, 270))
    assert not out[sum(ql):].any() and (lse[sum(ql):] == -INF).all()


def test_runs_are_alike_and_streams():
    ops = _ops()
    q, k, v, dout, out, lse = check([300, 64, 1, 150], heads=6, kv=2, causal=True, seed=31)
    c = cu([300, 64, 1, 150])
    first = ops.attention_packed_backward(dout, q, k, v, out, lse, c, causal=True)
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s in sides:                                          # two calls at once, each with its own workspace
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            o, l = ops.attention_packed(q, k, v, c, causal=True)
            got.append((o, l) + ops.attention_packed_backward(dout, q, k, v, o, l, c, causal=True))
    for s in sides:
        torch.cuda.current_stream().wait_stream(s)
    for g in got:
        for a, b in zip((out, lse) + first, g):
            assert torch.equal(a, b)


def test_captured_graph_follows_the_lengths():
    """A graph captured with one set of lengths and replayed with others: what cu and k_lens say at the replay counts."""
    ops = _ops()
    B, slab, heads, kv = 4, 600, 4, 2
    q, k, v, _ = make([1] * B, [slab] * B, heads, kv, seed=3)
    cq, ck = cu([1] * B), cu([slab] * B)
    lens = torch.tensor([5, 600, 0, 77], dtype=torch.int32).cuda()
    pq, pk, pv, pd = make([200, 100], heads=heads, kv=kv, seed=4)
    pc = cu([200, 100])

    def both():
        one = ops.attention_packed(q, k, v, cq, ck, k_lens=lens, causal=True)
        out, lse = ops.attention_packed(pq, pk, pv, pc, causal=True)
        return one + (out, lse) + ops.attention_packed_backward(pd, pq, pk, pv, out, lse, pc, causal=True)
    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for new, cut in (([6, 599, 1, 78], 200), ([600, 0, 320, 3], 1), ([1, 1, 1, 1], 299), ([64, 128, 256, 512], 150)):
        lens.copy_(torch.tensor(new, dtype=torch.int32))
        pc.copy_(cu([cut, 300 - cut]))
        q.copy_(torch.randn(q.shape, device="cuda"))
        graph.replay()
        want = both()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_gradient_against_differences():
    """<gradient, direction> against the central difference of the 64-bit forward pass."""
    ops = _ops()
    ql = [20, 33]
    q, k, v, dout = make(ql, heads=4, kv=2, seed=7)
    c = cu(ql)
    out, lse = ops.attention_packed(q, k, v, c, causal=True)
    grads = ops.attention_packed_backward(dout, q, k, v, out, lse, c, causal=True)
    ref = reference(q, k, v, ql, ql, True, 0.125, dout)
    base = [t.double().cpu() for t in (q, k, v)]
    gen = torch.Generator().manual_seed(1)
    for i, name in enumerate(("dq", "dk", "dv")):
        d = torch.randn(base[i].shape, generator=gen, dtype=torch.float64)
        h = 1e-5
        ends = []
        for sign in (1, -1):
            x = list(base)
            x[i] = x[i] + sign * h * d
            ends.append((reference(*x, ql, ql, True, 0.125)["out"] * dout.double().cpu()).sum())
        slope = (ends[0] - ends[1]) / (2 * h)
        got = (grads[i].double().cpu() * d).sum()
        # the difference itself: second order in h, 1e-16 / h of the loss's terms
        own = 1e-8 * float((dout.double().cpu().abs() * ref["out"].abs()).sum()) + 1e-7 * float((ref[name] * d).abs().sum())
        assert abs(float(got - slope)) <= float((ref[name + "_b"] * d.abs()).sum()) + own


def test_a_block_of_an_encoder_trains():
    """LayerNorm, QKV, packed attention, projection, LayerNorm, GELU and their backward passes, as one training step of
    an encoder block over images of different sizes runs them: against the same block in 64 bits by autograd, where the
    roundings of the bf16 operands in between leave some per cent."""
    ops = _ops()
    gen = torch.Generator().manual_seed(11)
    lens, dim, heads, hid = [50, 17, 82], 128, 2, 256
    T = sum(lens)
    x = torch.randn(T, dim, generator=gen).cuda()
    w = {n: (torch.randn(*s, generator=gen) / s[1] ** 0.5).to(torch.bfloat16).cuda()
         for n, s in (("qkv", (3 * dim, dim)), ("o", (dim, dim)), ("fc1", (hid, dim)), ("fc2", (dim, hid)))}
    g1, b1, g2, b2 = (torch.randn(dim, generator=gen).cuda() * 0.1 + o for o in (1, 0, 1, 0))
    dy = torch.randn(T, dim, generator=gen).cuda()
    c = cu(lens)
    t = lambda m: m.t().contiguous()                                              # noqa: E731
    # forward: the residual stream in fp32, operands in bf16
    h1, s1 = ops.layernorm_train(x, g1, b1, 1e-6)
    qkv = ops.linear(h1, w["qkv"]).view(T, 3, heads, 64)
    o, lse = ops.attention_packed(qkv[:, 0], qkv[:, 1], qkv[:, 2], c)
    x1 = ops.linear(o.view(T, dim), w["o"], res=x, out_f32=True)
    h2, s2 = ops.layernorm_train(x1, g2, b2, 1e-6)
    u = ops.linear(h2, w["fc1"])
    a, kept = ops.gelu_fp8(u)
    y = ops.linear(a, w["fc2"], res=x1, out_f32=True)
    # backward: dx1 takes the residual's gradient inside layernorm_backward
    da = ops.linear(ops.f32_to_bf16(dy), t(w["fc2"]))
    du, again = ops.gelu_fp8_backward(da, kept, recompute=True)
    dh2 = ops.linear(du, t(w["fc1"]))
    dx1, dg2, db2 = ops.layernorm_backward(dh2, x1, s2, g2, add=dy)
    do = ops.linear(ops.f32_to_bf16(dx1), t(w["o"])).view(T, heads, 64)
    dqkv = torch.empty_like(qkv)
    ops.attention_packed_backward(do, qkv[:, 0], qkv[:, 1], qkv[:, 2], o, lse, c, dq=dqkv[:, 0], dk=dqkv[:, 1], dv=dqkv[:, 2])
    dh1 = ops.linear(dqkv.view(T, 3 * dim), t(w["qkv"]))
    dx, dg1, db1 = ops.layernorm_backward(dh1, x, s1, g1, add=dx1)

    def leaf(v):
        return v.double().cpu().requires_grad_(True)
    X, G1, B1, G2, B2 = (leaf(v) for v in (x, g1, b1, g2, b2))
    W = {n: v.double().cpu() for n, v in w.items()}
    norm = torch.nn.functional.layer_norm
    QKV = (norm(X, (dim,), G1, B1, 1e-6) @ W["qkv"].T).view(T, 3, heads, 64)
    parts, at = [], 0
    for n in lens:
        Q, K, V = (QKV[at:at + n, i].transpose(0, 1) for i in range(3))
        parts.append((torch.softmax(Q @ K.transpose(1, 2) / 8, -1) @ V).transpose(0, 1).reshape(n, dim))
        at += n
    X1 = X + torch.cat(parts) @ W["o"].T
    Y = X1 + torch.nn.functional.gelu(norm(X1, (dim,), G2, B2, 1e-6) @ W["fc1"].T) @ W["fc2"].T
    (Y * dy.double().cpu()).sum().backward()
    # each of ~10 chained bf16 operands adds 2^-9 (rms) of its size, the 8-bit kept values 2^-5 of GELU's slope's change
    for name, got, want, tol in (("y", y, Y.detach(), 0.02), ("dx", dx, X.grad, 0.04), ("dg1", dg1, G1.grad, 0.06),
                                 ("db1", db1, B1.grad, 0.06), ("dg2", dg2, G2.grad, 0.06), ("db2", db2, B2.grad, 0.06)):
        rel = float((got.double().cpu() - want).norm() / want.norm())
        assert rel <= tol, f"{name}: {rel:.3e}"
    # the recomputed activation is that of the kept values
    assert float((again.float() - a.float()).norm() / a.float().norm()) <= 2.0 ** -4


def test_profiled_calls_are_listed(monkeypatch):
    """With a profile list every call leaves its label, bytes and two events, and computes the same."""
    ops = _ops()
    q, k, v, dout = make([40, 30], heads=2, seed=1)
    c, x, g = cu([40, 30]), torch.randn(9, 96, device="cuda"), torch.ones(96, device="cuda")
    want = ops.attention_packed(q, k, v, c)
    seen = []
    monkeypatch.setattr(ops, "profile", seen)
    out, lse = ops.attention_packed(q, k, v, c)
    ops.attention_packed_backward(dout, q, k, v, out, lse, c)
    y, stats = ops.layernorm_train(x, g, g, 1e-6)
    ops.layernorm_backward(y, x, stats, g)
    ops.gelu_fp8_backward(y, ops.gelu_fp8(y)[1])
    torch.cuda.synchronize()
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    assert [s[0] for s in seen] == ["k_attnp_fwd", "k_attnp_bwd", "k_lnt_fwd", "k_lnt_bwd", "k_gelu_keep", "k_gelu_back"]
    assert all(s[2] > 0 and s[3].elapsed_time(s[4]) >= 0 for s in seen)


@pytest.mark.parametrize("pitch", [0, 8, 3, 1 << 24])
def test_one_row_has_no_pitch(pitch):
    """The stride from row to row of an operand of one row is never taken."""
    ops = _ops()
    H = 4
    q, k, v, dout = make([1], heads=H, seed=6)
    q70, k70, v70, d70 = make([70], heads=H, seed=7)

    def one(t):
        return t.reshape(H, 64).as_strided((1, H, 64), (pitch, 64, 1))
    c1, c70 = cu([1]), cu([70])
    for qs, ks, c, ck in (((q, dout), (k70, v70), c1, c70), ((q70, d70), (k, v), c70, c1), ((q, dout), (k, v), c1, c1)):
        a, b = [t.clone() for t in qs + ks], [one(t.clone()) if t.shape[0] == 1 else t for t in qs + ks]
        out, lse = ops.attention_packed(a[0], a[2], a[3], c, ck)
        o2 = torch.empty_like(out) if out.shape[0] > 1 else one(torch.empty_like(out))
        l2 = torch.empty_like(lse)
        ops.attention_packed(b[0], b[2], b[3], c, ck, out=o2, lse=l2)
        assert torch.equal(out, o2) and torch.equal(lse, l2)
        want = ops.attention_packed_backward(a[1], a[0], a[2], a[3], out, lse, c, ck)
        got = [one(torch.empty_like(t)) if t.shape[0] == 1 else torch.empty_like(t) for t in want]
        ops.attention_packed_backward(b[1], b[0], b[2], b[3], o2, l2, c, ck, dq=got[0], dk=got[1], dv=got[2])
        for x, y in zip(want, got):
            assert torch.equal(x, y)


def test_one_head_has_no_pitch():
    ops = _ops()
    q, k, v, dout = make([70], heads=1, seed=6)
    out, lse = ops.attention_packed(q, k, v, cu([70]))
    odd = [t.as_strided((70, 1, 64), (64, 3, 1)) for t in (q, k, v, out, dout)]
    o2, l2 = ops.attention_packed(*odd[:3], cu([70]))
    assert torch.equal(out, o2) and torch.equal(lse, l2)
    for a, b in zip(ops.attention_packed_backward(dout, q, k, v, out, lse, cu([70])),
                    ops.attention_packed_backward(odd[4], *odd[:3], odd[3], lse, cu([70]))):
        assert torch.equal(a, b)


def test_a_half_without_a_probability_beside_a_masked_nan():
    """Two waves share a row's keys.  The rows from 32 on see 49 to 80 keys; the first 32 have scores of -inf, so that one wave
    has no probability for the rows up to 64 keys, and a NaN that the mask hides has it done again."""
    ops = _ops()
    q, k, v, _ = make([100], [116], heads=2, seed=4)
    q, k = q.abs() + 0.5, -k.abs() * 16 - 8                   # scores of some hundreds below zero
    k[:32, :, 0] = -INF
    v[90] = float("nan")
    out, lse = ops.attention_packed(q, k, v, cu([100]), cu([116]), causal=True)
    v2 = v.clone()
    v2[90] = 0
    ref = reference(q[16:], k[32:], v2[32:], [84], [84], True, 0.125)
    inside(out[16:74], ref["out"][:58], ref["out_b"][:58], "out")
    inside(lse[16:], ref["lse"], ref["lse_b"], "lse")
    assert out[74:].isnan().all()


@pytest.mark.parametrize("prompt", [700, 1500])
def test_prompts_and_single_tokens_in_one_pack(prompt):
    """Single tokens over slabs beside a prompt: a short one leaves their keys in shares, a long one fills the chip and does not."""
    ops = _ops()
    B, slab = 40, 3000
    ql, lens = [1] * B + [prompt], [1 + i * 2654435761 % 2999 for i in range(B)] + [prompt + 100]
    q, k, v, _ = make(ql, [slab] * (B + 1), 16, 4, seed=prompt)
    for b, n in enumerate(lens):
        k[b * slab + n:(b + 1) * slab] = float("nan")
        v[b * slab + n:(b + 1) * slab] = float("inf")
    out, lse = ops.attention_packed(q, k, v, cu(ql), cu([slab] * (B + 1)), k_lens=torch.tensor(lens, dtype=torch.int32).cuda(), causal=True)
    ref = reference(q, k, v, ql, lens, True, 0.125, starts=[b * slab for b in range(B + 1)])
    inside(out, ref["out"], ref["out_b"], "out")
    inside(lse, ref["lse"], ref["lse_b"], "lse")

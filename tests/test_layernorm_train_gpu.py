"""LayerNorm's training step against the formulas in 64 bits.

Tolerances count roundings: an output is off by half a step of its type (2^-8 of the value in bf16, 2^-24 in fp32) for
its own rounding, and by the fp32 arithmetic before it: a row's sums are trees of at most 16 sequential terms and nine
joins, so `U` = 40 units of 2^-24 of the summed magnitudes bound each, and what follows adds a few."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = 40 * 2.0 ** -24
BF = 2.0 ** -8
EPS = 1e-6


def _ops():
    from image_to_pointcloud_amd import ops
    return ops


def reference(x, gamma, beta, dy, add=None):
    x, gamma, beta, dy = (t.double() for t in (x, gamma, beta, dy))
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((x - mean).square().mean(1, keepdim=True) + EPS)
    h = (x - mean) * rstd
    g = dy * gamma
    a, b = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    dx = rstd * (g - a - h * b)
    if add is not None:
        dx = dx + add.double()
    return {"y": h * gamma + beta, "mean": mean, "rstd": rstd, "h": h, "g": g, "a": a, "b": b, "dx": dx,
            "dgamma": (dy * h).sum(0), "dbeta": dy.sum(0), "dgamma_abs": (dy * h).abs().sum(0), "dbeta_abs": dy.abs().sum(0)}


def case(rows, dim, dtype, seed, pitch=None, offset=0.5):
    """Inputs on the device; pitch: columns of the buffer that x, dy (and the gradients) are slices of."""
    gen = torch.Generator().manual_seed(seed)
    pitch = pitch or dim

    def wide(dt):
        t = torch.randn(rows, pitch, generator=gen)
        return t

    x = (wide(dtype) * (0.5 + torch.rand(pitch, generator=gen)) + offset).to(dtype).cuda()[:, :dim]
    dy = wide(dtype).to(torch.bfloat16).cuda()[:, :dim]
    add = wide(dtype).to(dtype).cuda()[:, :dim]
    gamma = (1 + 0.2 * torch.randn(dim, generator=gen)).cuda()
    beta = (0.1 * torch.randn(dim, generator=gen)).cuda()
    return x, gamma, beta, dy, add


def inside(got, want, bound, what):
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} values off, worst {(off - bound).max():.3e} over its bound"


def check(x, gamma, beta, dy, add, out=None, dx=None):
    ops = _ops()
    ref = reference(x, gamma, beta, dy, add)
    y, stats = ops.layernorm_train(x, gamma, beta, EPS, out=out)
    got_dx, dgamma, dbeta = ops.layernorm_backward(dy, x, stats, gamma, add=add, dx=dx)
    rows = x.shape[0]
    size = x.double().abs().amax(1, keepdim=True)
    # the normalised value: the mean's error and the subtraction's, over the deviation; the deviation's error
    eh = 2 * U * (size * ref["rstd"] + ref["h"].abs() + 1)
    inside(stats[:, :1], ref["mean"], U * size, "mean")
    inside(stats[:, 1:], ref["rstd"], ref["rstd"] * 2 * U * (size * ref["rstd"] + 1), "rstd")
    g = gamma.double().abs()
    inside(y, ref["y"], BF * ref["y"].abs() + 1.01 * (eh * g + U * ref["y"].abs()), "y")
    ga = ref["g"].abs()
    ea = U * ga.mean(1, keepdim=True)
    eb = U * (ref["g"] * ref["h"]).abs().mean(1, keepdim=True) + (ga * eh).mean(1, keepdim=True)
    inner = U * ga + ea + eh * ref["b"].abs() + ref["h"].abs() * eb
    edx = ref["rstd"] * inner + 2 * U * (size * ref["rstd"] + 1) * (ref["dx"].abs() + (add.double().abs() if add is not None else 0))
    step = BF if x.dtype == torch.bfloat16 else 2.0 ** -24
    inside(got_dx, ref["dx"], step * ref["dx"].abs() + 1.01 * edx, "dx")
    # a column's sum: at most rows / 4096 sequential terms a wave, then 8 + 16 + 512 / 16 joins
    n = rows / 4096 + 64
    edh = (dy.double().abs() * eh).sum(0)
    inside(dgamma, ref["dgamma"], 2.0 ** -24 * n * ref["dgamma_abs"] + edh, "dgamma")
    inside(dbeta, ref["dbeta"], 2.0 ** -24 * n * ref["dbeta_abs"], "dbeta")
    return y, stats, got_dx, dgamma, dbeta


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("rows,dim", [(1, 1), (1, 2), (3, 7), (2, 63), (9, 64), (5, 65), (4, 127), (17, 128), (6, 200), (8, 256),
                                      (5, 257), (3, 384), (7, 500), (577, 768), (2, 1001), (33, 1024), (4, 1025), (3, 1111),
                                      (5, 2048), (3, 2050), (2, 4096), (2, 4099), (3, 8192)])
def test_widths(rows, dim, dtype):
    x, gamma, beta, dy, add = case(rows, dim, dtype, rows * 10007 + dim)
    check(x, gamma, beta, dy, add)


@pytest.mark.parametrize("rows,dim", [(4099, 384), (9001, 64), (5003, 1030)])
def test_more_rows_than_one_round(rows, dim):
    check(*case(rows, dim, torch.float32, 3))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("dim,pitch,shift", [(384, 385, 0), (1111, 1203, 1), (64, 72, 3), (2050, 2051, 1), (33, 34, 1)])
def test_pitches_and_alignment(dim, pitch, shift, dtype):
    """Rows of any pitch that start at any element, the columns beside them untouched."""
    x, gamma, beta, dy, add = case(11, dim - shift, dtype, 5, pitch=pitch)
    n = dim - shift
    wide_y = torch.full((11, pitch), 7.0, dtype=torch.bfloat16, device="cuda")
    wide_dx = torch.full((11, pitch), 7.0, dtype=dtype, device="cuda")
    xs, dys, adds = (torch.cat([t.new_zeros(11, shift), t, t.new_zeros(11, pitch - dim)], 1)[:, shift:shift + n] for t in (x, dy, add))
    check(xs, gamma, beta, dys, adds, out=wide_y[:, shift:shift + n], dx=wide_dx[:, shift:shift + n])
    for w in (wide_y, wide_dx):
        assert (w[:, :shift] == 7).all() and (w[:, shift + n:] == 7).all()


def test_large_offset():
    """A row far from zero: two passes keep the variance."""
    check(*case(6, 1000, torch.float32, 9, offset=3000.0))


def test_add_in_place_and_without():
    ops = _ops()
    x, gamma, beta, dy, add = case(19, 517, torch.float32, 21)
    y, stats = ops.layernorm_train(x, gamma, beta, EPS)
    plain = ops.layernorm_backward(dy, x, stats, gamma)
    added = ops.layernorm_backward(dy, x, stats, gamma, add=add)
    check(x, gamma, beta, dy, None)
    inplace = add.clone()
    got = ops.layernorm_backward(dy, x, stats, gamma, add=inplace, dx=inplace)
    assert got[0] is inplace and torch.equal(inplace, added[0])
    assert torch.equal(got[1], plain[1]) and torch.equal(got[2], plain[2])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [513, 515, 1025, 1111, 2049, 4097, 8191])
def test_add_in_place_where_columns_repeat(dim, dtype):
    """Widths whose last load starts before another wave's columns end."""
    ops = _ops()
    x, gamma, beta, dy, add = case(1500, dim, dtype, 22)
    _, stats = ops.layernorm_train(x, gamma, beta, EPS)
    want = ops.layernorm_backward(dy, x, stats, gamma, add=add)
    got = add.clone()
    ops.layernorm_backward(dy, x, stats, gamma, add=got, dx=got)
    assert torch.equal(got, want[0])


def test_no_rows():
    ops = _ops()
    x = torch.zeros(0, 96, device="cuda")
    g = torch.ones(96, device="cuda")
    y, stats = ops.layernorm_train(x, g, g, EPS)
    assert y.shape == (0, 96) and stats.shape == (0, 2)
    dg = torch.full((96,), 5.0, device="cuda")
    dx, dgamma, dbeta = ops.layernorm_backward(y, x, stats, g, dgamma=dg)
    assert dx.shape == (0, 96) and dgamma is dg and not dgamma.any() and not dbeta.any()


def test_nonfinite_rows_stay_rows():
    """A NaN or an infinity spoils its own row and the column sums, no other row."""
    ops = _ops()
    x, gamma, beta, dy, add = case(12, 300, torch.float32, 4)
    clean = check(x, gamma, beta, dy, add)
    x2 = x.clone()
    x2[3, 17] = float("nan")
    x2[8, 0] = float("inf")
    y, stats = ops.layernorm_train(x2, gamma, beta, EPS)
    dx, _, _ = ops.layernorm_backward(dy, x2, stats, gamma, add=add)
    keep = [i for i in range(12) if i not in (3, 8)]
    assert torch.equal(y[keep], clean[0][keep]) and torch.equal(dx[keep], clean[2][keep])
    assert y[3].isnan().all() and dx[3].isnan().all()


def test_runs_are_alike_and_streams():
    ops = _ops()
    x, gamma, beta, dy, add = case(3001, 768, torch.bfloat16, 31)
    y, stats = ops.layernorm_train(x, gamma, beta, EPS)
    first = ops.layernorm_backward(dy, x, stats, gamma, add=add)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = ops.layernorm_backward(dy, x, stats, gamma, add=add)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, again):
        assert torch.equal(a, b)


def test_captured_and_replayed():
    ops = _ops()
    x, gamma, beta, dy, add = case(513, 384, torch.float32, 41)
    y, stats = ops.layernorm_train(x, gamma, beta, EPS)                     # warm
    ops.layernorm_backward(dy, x, stats, gamma, add=add)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gy, gs = ops.layernorm_train(x, gamma, beta, EPS)
        gout = ops.layernorm_backward(dy, x, gs, gamma, add=add)
    for seed in range(4):
        nx, _, _, ndy, nadd = case(513, 384, torch.float32, 100 + seed)
        x.copy_(nx), dy.copy_(ndy), add.copy_(nadd)
        graph.replay()
        ey, es = ops.layernorm_train(x, gamma, beta, EPS)
        eout = ops.layernorm_backward(dy, x, es, gamma, add=add)
        torch.cuda.synchronize()
        assert torch.equal(gy, ey) and torch.equal(gs, es)
        for a, b in zip(gout, eout):
            assert torch.equal(a, b)


def test_gradient_against_differences():
    """<gradient, direction> against the central difference of the 64-bit forward pass."""
    ops = _ops()
    x, gamma, beta, dy, _ = case(7, 96, torch.float32, 51)
    y, stats = ops.layernorm_train(x, gamma, beta, EPS)
    dx, dgamma, dbeta = ops.layernorm_backward(dy, x, stats, gamma)
    gen = torch.Generator().manual_seed(1)

    def loss(xx, gg, bb):
        m = xx.mean(1, keepdim=True)
        h = (xx - m) / torch.sqrt((xx - m).square().mean(1, keepdim=True) + EPS)
        return ((h * gg + bb) * dy.double()).sum()
    base = [x.double(), gamma.double(), beta.double()]
    for i, grad in enumerate((dx, dgamma, dbeta)):
        v = torch.randn(base[i].shape, generator=gen, dtype=torch.float64).cuda()
        step = 1e-5
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + step * v, base[i] - step * v
        slope = (loss(*up) - loss(*down)) / (2 * step)
        # the difference's own error is of order step^2 and 1e-16 / step: 1e-9 of the sum of magnitudes
        size = (grad.double().abs() * v.abs()).sum() + dy.double().abs().sum()
        assert abs(float((grad.double() * v).sum() - slope)) <= 1e-5 * float(size)


def test_offsets_beyond_32_bits():
    """Rows that lie 2^22 values apart in one buffer of more than 4 GiB, and the same rows packed."""
    ops = _ops()
    rows, dim, pitch = 600, 384, 1 << 22
    x, gamma, beta, dy, add = case(rows, dim, torch.bfloat16, 61)
    buf = torch.empty(rows * pitch, dtype=torch.bfloat16, device="cuda")              # only the rows are written
    far = [buf.as_strided((rows, dim), (pitch, 1), at * 1024) for at in range(5)]
    for to, t in zip(far, (x, dy, add)):
        to.copy_(t)
    y, stats = ops.layernorm_train(far[0], gamma, beta, EPS, out=far[3])
    y2, stats2 = ops.layernorm_train(x, gamma, beta, EPS)
    assert torch.equal(y, y2) and torch.equal(stats, stats2)
    got = ops.layernorm_backward(far[1], far[0], stats, gamma, add=far[2], dx=far[4])
    for a, b in zip(got, ops.layernorm_backward(dy, x, stats, gamma, add=add)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("pitch", [400, 3, 0])
def test_one_row_has_no_pitch(pitch):
    ops = _ops()
    x, gamma, beta, dy, add = case(1, 384, torch.float32, 71)
    y, stats = ops.layernorm_train(x, gamma, beta, EPS)
    want = ops.layernorm_backward(dy, x, stats, gamma, add=add)

    def odd(t):
        return t.reshape(-1).as_strided((1, 384), (pitch, 1))
    y2, s2 = ops.layernorm_train(odd(x.clone()), gamma, beta, EPS, out=odd(torch.zeros_like(y)))
    assert torch.equal(y, y2) and torch.equal(stats, s2)
    got = ops.layernorm_backward(odd(dy.clone()), odd(x.clone()), s2, gamma, add=odd(add.clone()), dx=odd(torch.zeros_like(x)))
    for a, b in zip(got, want):
        assert torch.equal(a, b)

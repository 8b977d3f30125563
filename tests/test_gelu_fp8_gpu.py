"""GELU with its input kept in 8 bits, against 64 bits.

Phi by the kernel's formula is within 0.75e-7 and five fp32 roundings of the true one; an output's own rounding to bf16 is
2^-8 of the value (2^-134 where it is subnormal).  What is kept is exact: the bytes of quant_fp8 and quantize_mx."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BF, TINY, PHI = 2.0 ** -8, 2.0 ** -133, 0.75e-7 + 5 * 2.0 ** -24


def _ops():
    from image_to_pointcloud_amd import ops
    return ops


def cdf(x):
    return 0.5 * torch.special.erfc(-x / math.sqrt(2.0))


def slope(x):
    return cdf(x) + x * torch.exp(-x.square() / 2) / math.sqrt(2 * math.pi)


def kept_values(kept):
    """What the bytes stand for, in 64 bits: the largest bf16 values round up to 2^128, which fp32 cannot hold."""
    v = kept.data.view(torch.float8_e4m3fn).double()
    return v * torch.pow(2.0, kept.scale.double() - 127).repeat_interleave(32, dim=-1)


def inside(got, want, bound, what):
    # from (2 - 2^-8) 2^127 on, half a step above the largest bf16 value, infinity is the nearest
    over = (want.abs() >= (2 - 2.0 ** -8) * 2.0 ** 127) & (got.double() == torch.sign(want) * math.inf)
    off = torch.where(over, torch.zeros_like(want), (got.double() - want).abs())
    assert (off <= bound).all(), f"{what}: {(off - bound).max():.3e} over its bound"


def check(x, dy, **kw):
    ops = _ops()
    y, kept = ops.gelu_fp8(x)
    x64, d64 = x.double(), dy.double()
    want = x64 * cdf(x64)
    inside(y, want, BF * want.abs() + PHI * x64.abs() + TINY, "y")
    q = ops.quantize_mx(x.float().contiguous())
    assert torch.equal(kept.data, q.data) and torch.equal(kept.scale, q.scale)
    k64 = kept_values(kept)
    dx, again = ops.gelu_fp8_backward(dy, kept, recompute=True)
    want = d64 * slope(k64)
    inside(dx, want, BF * want.abs() + d64.abs() * 3 * PHI + TINY, "dx")
    want = k64 * cdf(k64)
    inside(again, want, BF * want.abs() + PHI * k64.abs() + TINY, "again")
    only = ops.gelu_fp8_backward(dy, kept)
    assert torch.equal(only, dx)
    return y, kept, dx, again


def inputs(rows, dim, seed, pitch=None):
    gen = torch.Generator().manual_seed(seed)
    pitch = pitch or dim
    x = (2.0 * torch.randn(rows, pitch, generator=gen) * torch.exp(torch.randn(rows, 1, generator=gen))).to(torch.bfloat16).cuda()
    dy = torch.randn(rows, pitch, generator=gen).to(torch.bfloat16).cuda()
    return x[:, :dim], dy[:, :dim]


@pytest.mark.parametrize("rows,dim", [(1, 32), (1, 64), (3, 96), (7, 1536), (577, 160), (2, 8192), (1000, 4096)])
def test_sizes(rows, dim):
    check(*inputs(rows, dim, rows + dim))


def test_pitches():
    ops = _ops()
    x, dy = inputs(9, 96, 3, pitch=104)
    y0, k0, dx0, a0 = check(x.contiguous(), dy.contiguous())
    y, kept = ops.gelu_fp8(x, out=torch.zeros(9, 120, dtype=torch.bfloat16, device="cuda")[:, 8:104])
    assert torch.equal(y, y0) and torch.equal(kept.data, k0.data) and torch.equal(kept.scale, k0.scale)
    wide = torch.full((9, 112), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.gelu_fp8_backward(dy, kept, dx=wide[:, 8:104])
    assert torch.equal(wide[:, 8:104], dx0) and (wide[:, :8] == 7).all() and (wide[:, 104:] == 7).all()


def test_every_bf16_value():
    """All finite bf16 values, 32 neighbours a block (each block's scale is that of its own size)."""
    bits = torch.arange(65536, dtype=torch.int32)
    v = bits.to(torch.int16).view(torch.bfloat16)
    v = v[torch.isfinite(v.float())]
    v = v[:v.numel() // 32 * 32].reshape(-1, 32).cuda()
    check(v, torch.ones_like(v))


def test_nonfinite_and_zero_blocks():
    ops = _ops()
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")
    x[1, 3], x[1, 40], x[2, 5], x[3, 63] = float("nan"), 2.0, float("inf"), float("-inf")
    y, kept = ops.gelu_fp8(x)
    dy = torch.ones_like(x)
    dx, again = ops.gelu_fp8_backward(dy, kept, recompute=True)
    assert (y[0] == 0).all() and (dx[0] == 0.5).all() and (again[0] == 0).all()
    for t in (y, dx, again):
        assert t[1, 3].isnan() and t[1].isnan().sum() == 1
    assert y[2, 5] == math.inf and again[2, 5] == math.inf and dx[2, 5] == 1
    assert y[3, 63] == 0 and again[3, 63] == 0 and dx[3, 63] == 0
    assert torch.isfinite(y[2, :5].float()).all() and torch.isfinite(dx[3, :63].float()).all()


def test_no_rows():
    ops = _ops()
    x = torch.zeros(0, 64, dtype=torch.bfloat16, device="cuda")
    y, kept = ops.gelu_fp8(x)
    assert y.shape == (0, 64) and ops.gelu_fp8_backward(x, kept).shape == (0, 64)


def test_captured_and_replayed():
    ops = _ops()
    x, dy = inputs(100, 256, 1)
    ops.gelu_fp8_backward(dy, ops.gelu_fp8(x)[1], recompute=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, kept = ops.gelu_fp8(x)
        dx, again = ops.gelu_fp8_backward(dy, kept, recompute=True)
    for seed in range(3):
        nx, ndy = inputs(100, 256, 10 + seed)
        x.copy_(nx), dy.copy_(ndy)
        graph.replay()
        ey, ek = ops.gelu_fp8(x)
        edx, ea = ops.gelu_fp8_backward(dy, ek, recompute=True)
        torch.cuda.synchronize()
        assert torch.equal(y, ey) and torch.equal(kept.data, ek.data) and torch.equal(dx, edx) and torch.equal(again, ea)


def test_gradient_against_differences():
    ops = _ops()
    x, dy = inputs(5, 64, 8)
    _, kept = ops.gelu_fp8(x)
    dx = ops.gelu_fp8_backward(dy, kept)
    k = kept_values(kept)
    h = 1e-5
    want = dy.double() * ((k + h) * cdf(k + h) - (k - h) * cdf(k - h)) / (2 * h)
    # the difference is of second order in h (1e-10) and of 1e-16 |x| / h
    inside(dx, want, BF * want.abs() + dy.double().abs() * (3 * PHI + 1e-9 + 1e-11 * k.abs()) + TINY, "dx")


def test_in_place():
    ops = _ops()
    gen = torch.Generator().manual_seed(6)
    x, dy = (torch.randn(70, 96, generator=gen).to(torch.bfloat16).cuda() for _ in range(2))
    y, kept = ops.gelu_fp8(x)
    dx, again = ops.gelu_fp8_backward(dy, kept, recompute=True)
    x2, dy2 = x.clone(), dy.clone()
    got, kept2 = ops.gelu_fp8(x2, out=x2)
    assert got is x2 and torch.equal(x2, y) and torch.equal(kept2.data, kept.data) and torch.equal(kept2.scale, kept.scale)
    ops.gelu_fp8_backward(dy2, kept, dx=dy2, recompute=True)
    assert torch.equal(dy2, dx)


def test_offsets_beyond_32_bits():
    ops = _ops()
    rows, dim, pitch = 600, 96, 1 << 22
    x, dy = (torch.randn(rows, dim, generator=torch.Generator().manual_seed(i)).to(torch.bfloat16).cuda() for i in (1, 2))
    buf = torch.empty(rows * pitch, dtype=torch.bfloat16, device="cuda")              # only the rows are written
    far = [buf.as_strided((rows, dim), (pitch, 1), at * 128) for at in range(5)]
    far[0].copy_(x), far[1].copy_(dy)
    y, kept = ops.gelu_fp8(far[0], out=far[2])
    y2, kept2 = ops.gelu_fp8(x)
    assert torch.equal(y, y2) and torch.equal(kept.data, kept2.data) and torch.equal(kept.scale, kept2.scale)
    dx, again = ops.gelu_fp8_backward(far[1], kept, dx=far[3], again=far[4])
    dx2, again2 = ops.gelu_fp8_backward(dy, kept, recompute=True)
    assert torch.equal(dx, dx2) and torch.equal(again, again2)


def test_the_negative_tail():
    """Far below zero the value and the slope keep their own rounding, not the error of a number next to 1: every bf16 x in
    [-12.9, -4], a block to each.  Phi(-|x|) is within 2^-13.07 of its value by its polynomial and 2^-16.5 by the exponent of
    up to 122, which two fp32 roundings leave 122 * 2^-23 * ln 2 off; with ten roundings more, 2^-12.9 in all."""
    ops = _ops()
    rel = 2.0 ** -12.9
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    x = bits[(bits >= -12.9) & (bits <= -4)]
    x = x[:, None].expand(-1, 32).contiguous().cuda()
    dy = torch.ones_like(x)
    y, kept = ops.gelu_fp8(x)
    want = x.double() * cdf(x.double())
    inside(y, want, (BF + rel) * want.abs(), "y")
    dx, again = ops.gelu_fp8_backward(dy, kept, recompute=True)
    k = kept_values(kept)
    assert (k < -3.7).all()
    want = k * cdf(k)
    inside(again, want, (BF + rel) * want.abs(), "again")
    want = slope(k)
    terms = cdf(k) + k.abs() * torch.exp(-k.square() / 2) / math.sqrt(2 * math.pi)
    inside(dx, want, BF * want.abs() + rel * 1.02 * terms, "dx")


@pytest.mark.parametrize("pitch", [100, 3, 0])
def test_one_row_has_no_pitch(pitch):
    ops = _ops()
    x, dy = inputs(1, 96, 2)
    want = ops.gelu_fp8(x)
    wdx, wagain = ops.gelu_fp8_backward(dy, want[1], recompute=True)

    def odd(t):
        return t.reshape(-1).as_strided((1, 96), (pitch, 1))
    y, kept = ops.gelu_fp8(odd(x.clone()), out=odd(torch.zeros_like(x)))
    dx, again = ops.gelu_fp8_backward(odd(dy.clone()), kept, dx=odd(torch.zeros_like(x)), again=odd(torch.zeros_like(x)))
    for a, b in ((y, want[0]), (kept.data, want[1].data), (kept.scale, want[1].scale), (dx, wdx), (again, wagain)):
        assert torch.equal(a, b)

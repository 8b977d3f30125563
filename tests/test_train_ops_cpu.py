"""Refusals of the training operators and of packed attention: no device work (CPU tensors, or descriptors that the C side
turns down before it launches anything)."""
import ctypes
import os

import pytest

torch = pytest.importorskip("torch")

from image_to_pointcloud_amd import _lib, ops  # noqa: E402


def _built():
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("libi2pc.so not built")


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 64)
    b = x.to(torch.bfloat16)
    g = torch.ones(64)
    with pytest.raises(_lib.I2PCError):
        ops.layernorm_train(x, g, g, 1e-6)
    with pytest.raises(_lib.I2PCError):
        ops.layernorm_backward(b, x, torch.zeros(4, 2), g)
    with pytest.raises(_lib.I2PCError):
        ops.gelu_fp8(b)
    with pytest.raises(_lib.I2PCError):
        ops.gelu_fp8_backward(b, ops.Fp8(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)))
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(_lib.I2PCError):
        ops.attention_packed(q, q, q, cu)
    with pytest.raises(_lib.I2PCError):
        ops.attention_packed_backward(q, q, q, q, q, torch.zeros(4, 2), cu)


class _Device:
    """A CPU tensor that says it is on the device: what Python checks before any call into the library."""

    def __init__(self, t):
        self._t = t

    def get_device(self):
        return 0

    def __getattr__(self, n):
        return getattr(self._t, n)


def test_shapes_types_and_strides():
    bf = torch.bfloat16
    op = ops._operand
    op(_Device(torch.zeros(3, 4)), "t", (3, 4), torch.float32, None)
    with pytest.raises(_lib.I2PCError):
        op(torch.zeros(3, 4), "t", (3, 4), torch.float32, None)
    with pytest.raises(TypeError):
        op(_Device(torch.zeros(3, 4)), "t", (3, 4), bf, None)
    with pytest.raises(ValueError):
        op(_Device(torch.zeros(3, 5)), "t", (3, 4), torch.float32, None)
    with pytest.raises(ValueError):
        op(_Device(torch.zeros(4, 3).t()), "t", (3, 4), torch.float32, None)
    rows = ops._rows_dim
    assert rows(_Device(torch.zeros(3, 4)), "x", (torch.float32, bf)) == (3, 4, 4)
    assert rows(_Device(torch.zeros(3, 9)[:, 2:6]), "x", (torch.float32,)) == (3, 4, 9)
    assert rows(_Device(torch.zeros(1, 4).expand(1, 4)), "x", (torch.float32,)) == (1, 4, 4)
    for bad, error in ((torch.zeros(2, 3, 4), ValueError), (torch.zeros(4, 3).t(), ValueError), (torch.zeros(3, 4).half(), TypeError)):
        with pytest.raises(error):
            rows(_Device(bad), "x", (torch.float32, bf))
    with pytest.raises(TypeError):
        ops._kept_operand(torch.zeros(2, 32), 2, 32, 0)
    with pytest.raises(ValueError):
        ops._kept_operand(ops.Fp8(None, None), 2, 33, 0)
    dev = lambda *shape, dtype=bf: _Device(torch.zeros(*shape, dtype=dtype))              # noqa: E731
    q, lse, cu = dev(4, 2, 64), dev(4, 2, dtype=torch.float32), dev(2, dtype=torch.int32)
    desc = lambda q=q, k=q, v=q, out=q, lse=lse, cu_q=cu, cu_k=None, k_lens=None: ops._attn_packed_desc(               # noqa: E731
        q, k, v, out, lse, cu_q, cu_k, k_lens, None, True, False)
    d = desc()
    assert (d.batch, d.total_q, d.heads, d.causal, d.scale, d.q_t, d.o_h) == (1, 4, 2, 1, 0.125, 128, 64)
    for kw in ({"q": dev(4, 128)}, {"k": dev(4, 2, 32)}, {"v": dev(5, 2, 64)}, {"out": dev(3, 2, 64)}, {"lse": dev(2, 4, dtype=torch.float32)},
               {"cu_q": dev(1, dtype=torch.int32)}, {"cu_q": dev(2, 2, dtype=torch.int32)}, {"cu_k": dev(3, dtype=torch.int32)},
               {"k": dev(5, 2, 64), "v": dev(5, 2, 64)}, {"k_lens": dev(2, dtype=torch.int32)},
               {"lse": _Device(torch.zeros(2, 4).t())}):
        with pytest.raises(ValueError):
            desc(**kw)
    for kw in ({"q": dev(4, 2, 64, dtype=torch.float16)}, {"cu_q": dev(2, dtype=torch.int64)}, {"k_lens": dev(1, dtype=torch.int64)}):
        with pytest.raises(TypeError):
            desc(**kw)
    with pytest.raises(ValueError):
        ops.attention_packed(q, q, q, cu, out=q)
    with pytest.raises(ValueError):
        ops.attention_packed_backward(q, q, q, q, q, lse, cu, dq=q)


def _rc(name, *args):
    lib = _lib.load()
    rc = getattr(lib, name)(*args)
    return rc, lib.i2pc_last_error().decode()


def test_layernorm_refusals():
    _built()
    train = lambda rows, dim, x=16, ldx=None: _rc("i2pc_layernorm_train", x, 1, ldx or dim, 16, 16, 1e-6, rows, dim, 16, dim,  # noqa: E731
                                                  16, None)
    assert train(0, 64) == (0, "")
    for rows, dim, kw in ((-1, 64, {}), (4, 0, {}), (4, 8193, {}), (4, 64, {"x": None}), (4, 64, {"ldx": 63})):
        rc, msg = train(rows, dim, **kw)
        assert rc == -1 and msg, (rows, dim, kw)
    lib = _lib.load()
    need = lib.i2pc_layernorm_backward_workspace_bytes(100, 384)
    assert need > 0 and lib.i2pc_layernorm_backward_workspace_bytes(100, 9000) == 0
    assert lib.i2pc_layernorm_backward_workspace_bytes(8, 384) == 0            # one workgroup: no partial rows

    def backward(rows=100, dim=384, lda=384, ws=16, nb=need, dx=16):
        return _rc("i2pc_layernorm_backward", 16, dim, 16, 1, dim, 16, 16, 16, lda, rows, dim, dx, dim, 16, 16, ws, nb, None)
    assert backward(nb=need - 1)[0] == -2
    assert backward(ws=None)[0] == -2
    for kw in ({"rows": -1}, {"dim": 9000}, {"lda": 100}, {"dx": None}):
        assert backward(**kw)[0] == -1, kw


def test_gelu_refusals():
    _built()
    for rows, dim, ld, p in ((4, 33, 64, 16), (4, 0, 64, 16), (-1, 64, 64, 16), (4, 64, 60, 16), (4, 64, 68, 16), (4, 64, 64, 18),
                             (4, 64, 64, None)):
        assert _rc("i2pc_gelu_fp8", p, ld, rows, dim, 16, 64, 16, 16, None)[0] == -1, (rows, dim, ld, p)
        assert _rc("i2pc_gelu_fp8_backward", p, ld, 16, 16, rows, dim, 16, 64, None, 0, None)[0] == -1, (rows, dim, ld, p)
    assert _rc("i2pc_gelu_fp8", 16, 64, 1 << 40, 64, 16, 64, 16, 16, None)[0] == -4
    assert _rc("i2pc_gelu_fp8", None, 64, 0, 64, None, 64, None, None, None) == (0, "")


def _desc(**kw):
    d = ops.AttnPackedDesc()
    for n in ("q", "k", "v", "out", "lse", "cu_q", "cu_k"):
        setattr(d, n, 16)
    for n in ("q", "k", "v", "o"):
        setattr(d, n + "_t", 256)
        setattr(d, n + "_h", 64)
    d.batch, d.total_q, d.total_k, d.heads, d.kv_heads, d.head_dim, d.scale = 2, 100, 100, 4, 4, 64, 0.125
    for n, x in kw.items():
        setattr(d, n, x)
    return d


BAD = [({"head_dim": 128}, -4), ({"kv_heads": 3}, -1), ({"heads": 0}, -1), ({"total_q": -1}, -1), ({"batch": -1}, -1),
       ({"scale": 0.0}, -1), ({"scale": -1.0}, -1), ({"scale": float("nan")}, -1), ({"scale": float("inf")}, -1),
       ({"scale": 1e-30}, -1), ({"o_t": 64, "o_h": 64}, -1), ({"o_t": 128, "o_h": 64 * 100}, -1),
       ({"q": 24}, -1), ({"k_t": 252}, -1), ({"v_h": 60}, -1), ({"k_t": 0}, -1), ({"o_h": 0}, -1), ({"q_t": 1 << 23}, -1),
       ({"cu_q": None}, -1), ({"cu_k": None}, -1), ({"lse": None}, -1), ({"q": None}, -1), ({"total_q": 1 << 30}, -4),
       ({"total_k": (1 << 31) - 1, "kv_heads": 4}, -4)]


@pytest.mark.parametrize("kw,code", BAD, ids=[",".join(k) for k, _ in BAD])
def test_attention_refusals(kw, code):
    _built()
    d = _desc(**kw)
    rc, msg = _rc("i2pc_attention_packed", ctypes.byref(d), 16, 1 << 40, None)
    assert rc == code and msg
    g = ops.AttnPackedGradDesc()
    g.f = d
    for n in ("dout", "dq", "dk", "dv"):
        setattr(g, n, 16)
    for n in ("d", "dq", "dk", "dv"):
        setattr(g, n + "_t", 256)
        setattr(g, n + "_h", 64)
    assert _rc("i2pc_attention_packed_backward", ctypes.byref(g), 16, 1 << 40, None)[0] == code
    assert _lib.load().i2pc_attention_packed_workspace_bytes(ctypes.byref(d)) == 0


def test_attention_workspaces_and_the_backward_pass_own_refusals():
    _built()
    lib = _lib.load()
    d = _desc(batch=1, total_q=1, total_k=100000, q_t=256)
    need = lib.i2pc_attention_packed_workspace_bytes(ctypes.byref(d))
    assert need > 0                                                      # one token over many keys: they are split
    assert _rc("i2pc_attention_packed", ctypes.byref(d), 16, need - 1, None)[0] == -2
    assert _rc("i2pc_attention_packed", ctypes.byref(d), None, need, None)[0] == -2
    # the split takes the workspace from the totals alone, and no more shares than 256 keys each allow
    assert lib.i2pc_attention_packed_workspace_bytes(ctypes.byref(_desc(batch=1, total_q=1, total_k=256))) == 0
    assert lib.i2pc_attention_packed_workspace_bytes(ctypes.byref(_desc(batch=8, total_q=70000, total_k=70000))) == 0
    g = ops.AttnPackedGradDesc()
    g.f = _desc()
    for n in ("dout", "dq", "dk", "dv"):
        setattr(g, n, 16)
    for n in ("d", "dq", "dk", "dv"):
        setattr(g, n + "_t", 256)
        setattr(g, n + "_h", 64)
    need = lib.i2pc_attention_packed_backward_workspace_bytes(ctypes.byref(g))
    assert need > 0 and _rc("i2pc_attention_packed_backward", ctypes.byref(g), 16, need - 1, None)[0] == -2
    g.f.k_lens = 16
    assert _rc("i2pc_attention_packed_backward", ctypes.byref(g), 16, need, None)[0] == -1
    g.f.k_lens = None
    g.dk_h = 0
    assert _rc("i2pc_attention_packed_backward", ctypes.byref(g), 16, need, None)[0] == -1
    assert _rc("i2pc_attention_packed", ctypes.byref(_desc(total_q=0)), None, 0, None) == (0, "")


def test_outputs_that_overlap_themselves_are_refused():
    _built()
    lib = _lib.load()
    # [heads, rows, 64] underneath, heads next to each other, one row, one head
    for kw in ({"o_t": 64, "o_h": 6400}, {"o_t": 256, "o_h": 64}, {"total_q": 1, "o_t": 0, "o_h": 64},
               {"heads": 1, "kv_heads": 1, "o_t": 64, "o_h": 0}):
        g = _grad(**kw)
        assert lib.i2pc_attention_packed_backward_workspace_bytes(ctypes.byref(g)) > 0, kw
    for n in ("dq", "dk", "dv"):
        g = _grad()
        setattr(g, n + "_t", 128)
        assert lib.i2pc_attention_packed_backward_workspace_bytes(ctypes.byref(g)) == 0, n


def _grad(**kw):
    g = ops.AttnPackedGradDesc()
    g.f = _desc(**kw)
    for n in ("dout", "dq", "dk", "dv"):
        setattr(g, n, 16)
    for n in ("d", "dq", "dk", "dv"):
        setattr(g, n + "_t", 256)
        setattr(g, n + "_h", 64)
    return g


def test_sizes_above_31_bits_are_refused():
    """Not cut to their low 32 bits on the way to the library."""
    bf = torch.bfloat16
    many = _Device(torch.zeros(1, 64, dtype=bf).expand((1 << 32) + 4, 64))
    with pytest.raises(ValueError):
        ops._rows_dim(many, "x", (bf,))
    q = _Device(torch.zeros(4, 1, 64, dtype=bf))
    k = _Device(torch.zeros(1, 1, 64, dtype=bf).expand((1 << 32) + 4, 1, 64))
    cu = _Device(torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        ops._attn_packed_desc(q, k, k, q, None, cu, cu, None, None, False, True)


def test_one_row_has_no_pitch():
    """Its stride is never taken: not that of the buffer that it is a slice of, whatever that is."""
    bf = torch.bfloat16
    buf = torch.zeros(5, 100, dtype=bf)
    for t in (buf[:1, :96], buf.as_strided((1, 96), (3, 1)), buf.as_strided((1, 96), (0, 1)), buf.as_strided((0, 96), (5, 1))):
        assert ops._rows_dim(_Device(t), "x", (bf,))[1:] == (96, 96) and ops._pitch(t) == 96
    assert ops._rows_dim(_Device(buf[:2, :96]), "x", (bf,)) == (2, 96, 100) and ops._pitch(buf[:2, :96]) == 100


def test_strides_of_one_row_or_head_do_not_matter():
    _built()
    lib = _lib.load()
    for kw in ({"total_q": 1, "q_t": 3, "o_t": 1 << 40}, {"total_k": 1, "k_t": -5, "v_t": 0},
               {"heads": 1, "kv_heads": 1, "q_h": 3, "k_h": -1, "v_h": 1 << 50, "o_h": 1}):
        assert lib.i2pc_attention_packed_backward_workspace_bytes(ctypes.byref(_grad(**kw))) > 0, kw
    for kw in ({"total_q": 2, "q_t": 3}, {"heads": 2, "kv_heads": 2, "q_h": 3}, {"total_k": 1, "k": 24}):
        assert lib.i2pc_attention_packed_backward_workspace_bytes(ctypes.byref(_grad(**kw))) == 0, kw

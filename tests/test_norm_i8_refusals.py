"""Refusals of the norm's and the int8 calls on the CPU: the C entries' checks, which come
before any device is touched (the pointers are placeholders), and the Python layer's."""
import ctypes

import pytest
import torch

from hanuman_amd import _lib, kernels as K

P = ctypes.c_void_p(16)
ODD = ctypes.c_void_p(20)       # neither 16- nor 8-byte aligned
S = None
OK, INVALID, UNSUPPORTED, WORKSPACE = _lib.OK, _lib.ERR_INVALID, _lib.ERR_UNSUPPORTED, _lib.ERR_WORKSPACE
F32, BF16, E4M3, I8 = _lib.F32, _lib.BF16, _lib.FP8_E4M3, _lib.I8


def expect(code, needle, name, *args):
    rc = getattr(_lib.lib(), name)(*args)
    msg = _lib.lib().hmoe_last_error().decode()
    assert rc == code, f"{name}{args}: rc {rc}, expected {code} ({msg})"
    if needle:
        assert needle in msg, f"{name}: '{needle}' not in '{msg}'"


def test_norm():
    name = "hmoe_add_rms_norm"

    def args(x=P, xd=BF16, r=P, rd=BF16, w=P, wd=F32, eps=1e-6, rows=4, cols=64, s=P, y=P, yd=BF16, rstd=P, q=P, qt=I8,
             scale=P):
        return x, xd, r, rd, w, wd, eps, rows, cols, s, y, yd, rstd, q, qt, scale, S

    expect(INVALID, "rows", name, *args(rows=-1))
    for cols in (0, 12, 32776, -8):
        expect(UNSUPPORTED, "cols", name, *args(cols=cols))
    expect(INVALID, "dtypes", name, *args(xd=E4M3))
    expect(INVALID, "dtypes", name, *args(yd=7))
    expect(INVALID, "dtypes", name, *args(wd=I8))
    expect(INVALID, "residual dtype", name, *args(rd=E4M3))
    expect(INVALID, "q type", name, *args(qt=BF16))
    expect(INVALID, "eps", name, *args(eps=-1.0))
    expect(INVALID, "eps", name, *args(eps=float("nan")))
    for missing in ("x", "w", "y", "s", "r", "q", "scale"):
        expect(INVALID, "null", name, *args(**{missing: None}))
    for odd in ("x", "r", "w", "s", "y", "q"):
        expect(INVALID, "aligned", name, *args(**{odd: ODD}))
    expect(OK, None, name, *args(x=None, r=None, w=None, s=None, y=None, q=None, scale=None, rows=0))


def test_norm_bwd():
    name = "hmoe_add_rms_norm_bwd"
    need = _lib.lib().hmoe_add_rms_norm_bwd_workspace_bytes(800, 64)
    assert need == 512 * 64 * 4
    for few in (0, 1, 768):
        assert _lib.lib().hmoe_add_rms_norm_bwd_workspace_bytes(few, 64) == 0

    def args(dy=P, dd=BF16, s=P, sd=BF16, w=P, wd=F32, rstd=P, ds=P, rows=800, cols=64, dx=P, dw=P, ws=P, size=need):
        return dy, dd, s, sd, w, wd, rstd, ds, rows, cols, dx, dw, ws, size, S

    expect(INVALID, "rows", name, *args(rows=-1))
    expect(UNSUPPORTED, "cols", name, *args(cols=68))
    expect(INVALID, "dtypes", name, *args(dd=E4M3))
    expect(INVALID, "dtypes", name, *args(sd=I8))
    for missing in ("dy", "s", "w", "rstd", "dx"):
        expect(INVALID, "null", name, *args(**{missing: None}))
    for odd in ("dy", "s", "w", "ds", "dx", "dw", "ws"):
        expect(INVALID, "aligned", name, *args(**{odd: ODD}))
    expect(WORKSPACE, "workspace", name, *args(size=need - 1))
    expect(WORKSPACE, "workspace", name, *args(ws=None))
    expect(OK, None, name, *args(dy=None, s=None, w=None, rstd=None, ds=None, dx=None, dw=None, ws=None, size=0, rows=0))


PRODUCTS = [
    ("hmoe_grouped_gate_up_i8", lambda n, r, d, f, p: (p, p, p, n, r, d, f, p, p, p, S)),
    ("hmoe_grouped_gate_up_i8_gather", lambda n, r, d, f, p: (p, p, 64, 2, p, p, n, r, d, f, p, p, p, S)),
    ("hmoe_grouped_down_i8", lambda n, r, d, f, p: (p, p, p, n, r, f, d, p, p, p, S)),
]


@pytest.mark.parametrize("name,args", PRODUCTS, ids=[p[0] for p in PRODUCTS])
def test_products(name, args):
    expect(INVALID, "n_experts", name, *args(0, 10, 256, 128, P))
    expect(INVALID, "n_experts", name, *args(1025, 10, 256, 128, P))
    for bad in (192, 0, -128, 32896):
        expect(UNSUPPORTED, "d_model", name, *args(4, 10, bad, 128, P))
        expect(UNSUPPORTED, "d_ff", name, *args(4, 10, 256, bad, P))
    expect(INVALID, "rows_cap", name, *args(4, -1, 256, 128, P))
    expect(INVALID, "rows_cap", name, *args(4, (1 << 30) + 1, 256, 128, P))
    expect(INVALID, "too many tiles", name, *args(1, 1 << 30, 32768, 32768, P))
    expect(INVALID, "null", name, *args(4, 10, 256, 128, None))
    expect(INVALID, "aligned", name, *args(4, 10, 256, 128, ODD))
    expect(OK, None, name, *args(4, 0, 256, 128, None))


def test_gather():
    name = "hmoe_grouped_gate_up_i8_gather"
    tail = (P, P, 4, 10, 256, 128, P, P, P, S)
    expect(INVALID, "tokens", name, P, P, -1, 2, *tail)
    expect(INVALID, "tokens", name, P, P, 0, 2, *tail)
    expect(INVALID, "top_k", name, P, P, 64, 0, *tail)
    expect(INVALID, "2 GiB", name, P, P, 1 << 23, 2, *tail)
    expect(INVALID, "null", name, P, P, 64, 2, None, P, 4, 10, 256, 128, P, P, P, S)


def test_rows():
    for name, args, last in (
            ("hmoe_quantize_rows_i8", lambda p, t, r, c: (p, t, r, c, None, 0, p, p, S), 32776),
            ("hmoe_dequantize_rows_i8", lambda p, t, r, c: (p, p, r, c, p, t, S), 12),
            ("hmoe_dequantize_rows_fp8", lambda p, t, r, c: (p, p, r, c, p, t, S), 12)):
        for cols in (0, 12, last):
            expect(UNSUPPORTED, "cols", name, *args(P, F32, 4, cols))
        expect(INVALID, "rows", name, *args(P, F32, -1, 64))
        expect(INVALID, "dtype", name, *args(P, E4M3, 4, 64))
        expect(INVALID, "null", name, *args(None, BF16, 4, 64))
        expect(INVALID, "aligned", name, *args(ODD, BF16, 4, 64))
        expect(OK, None, name, *args(None, BF16, 0, 64))
    expect(INVALID, "n_experts", "hmoe_quantize_rows_i8", P, F32, 4, 64, P, -1, P, P, S)


def test_packs():
    for name, args in (("hmoe_pack_i8_gate_up", lambda p, t, n, d, f: (p, p, t, n, d, f, p, p, S)),
                       ("hmoe_pack_i8_down", lambda p, t, n, d, f: (p, t, n, f, d, p, p, S))):
        expect(INVALID, "n_experts", name, *args(P, F32, 0, 256, 128))
        expect(UNSUPPORTED, "d_model", name, *args(P, F32, 2, 200, 128))
        expect(UNSUPPORTED, "d_ff", name, *args(P, F32, 2, 256, 96))
        expect(UNSUPPORTED, "d_ff", name, *args(P, F32, 2, 256, 32896))
        expect(INVALID, "dtype", name, *args(P, E4M3, 2, 256, 128))
        expect(INVALID, "null", name, *args(None, F32, 2, 256, 128))
        expect(INVALID, "aligned", name, *args(ODD, F32, 2, 256, 128))
    lib = _lib.lib()
    assert lib.hmoe_packed_i8_gate_up_bytes(3, 256, 128) == 3 * 256 * 256
    assert lib.hmoe_packed_i8_down_bytes(3, 128, 256) == 3 * 128 * 256
    assert lib.hmoe_packed_i8_gate_up_bytes(0, 256, 128) == 0


def test_form():
    form = _lib.lib().hmoe_grouped_i8_form
    assert form(8, 64, 2048, 2048, 256) == 1 and form(131072, 64, 2048, 2048, 256) == 3
    for bad in ((0, 64, 2048, 2048, 256), (8, 0, 2048, 2048, 256), (8, 2000, 2048, 2048, 256),
                (8, 64, 100, 2048, 256), (8, 64, 2048, 64, 256), (8, 64, 2048, 2048, 0),
                (8, 64, 32896, 128, 256), (8, 64, 128, 65664, 256), (1 << 30, 1, 128, 32768, 256)):
        assert form(*bad) == -1


def test_python_layer():
    """Tensors that are not on a GPU are refused before anything is looked at."""
    x = torch.zeros((4, 64))
    q, s = torch.zeros((4, 64), dtype=torch.int8), torch.zeros(4)
    w = torch.zeros((2, 128, 128))
    packed, scales = torch.zeros((2, 8, 4, 64, 16), dtype=torch.int8), torch.zeros((2, 256))
    for call in (lambda: K.add_rms_norm(x, s), lambda: K.add_rms_norm_bwd(x, x, s, s), lambda: K.quantize_rows_i8(x),
                 lambda: K.dequantize_rows_i8(q, s), lambda: K.dequantize_rows_fp8(q, s),
                 lambda: K.pack_i8_gate_up(w, w), lambda: K.pack_i8_down(w),
                 lambda: K.grouped_gate_up_i8(q, s, s, packed, scales),
                 lambda: K.grouped_gate_up_i8_gather(q, s, None, packed, scales),
                 lambda: K.grouped_down_i8(q, s, s, packed, scales)):
        with pytest.raises(ValueError, match="GPU"):
            call()
    with pytest.raises(TypeError):
        K.quantize_rows_i8([1.0])

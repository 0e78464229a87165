"""Refusals of the MXFP4 calls on the CPU: the C entries' checks, which come before any
device is touched (the pointers are placeholders), and the Python layer's."""
import ctypes

import pytest
import torch

from hanuman_amd import _lib, kernels as K

P = ctypes.c_void_p(16)
ODD = ctypes.c_void_p(24)       # not 16-byte aligned
S = None
OK, INVALID, UNSUPPORTED = _lib.OK, _lib.ERR_INVALID, _lib.ERR_UNSUPPORTED
F32, BF16, E4M3 = _lib.F32, _lib.BF16, _lib.FP8_E4M3


def expect(code, needle, name, *args):
    rc = getattr(_lib.lib(), name)(*args)
    msg = _lib.lib().hmoe_last_error().decode()
    assert rc == code, f"{name}{args}: rc {rc}, expected {code} ({msg})"
    if needle:
        assert needle in msg, f"{name}: '{needle}' not in '{msg}'"


PRODUCTS = [
    ("hmoe_grouped_gate_up_mxfp4", lambda n, r, d, f, p: (p, p, p, n, r, d, f, p, p, p, p, S)),
    ("hmoe_grouped_gate_up_mxfp4_gather", lambda n, r, d, f, p: (p, p, 64, 2, p, p, n, r, d, f, p, p, p, p, S)),
    ("hmoe_grouped_down_mxfp4", lambda n, r, d, f, p: (p, p, p, n, r, f, d, p, p, p, S)),
]


@pytest.mark.parametrize("name,args", PRODUCTS, ids=[p[0] for p in PRODUCTS])
def test_products(name, args):
    expect(INVALID, "n_experts", name, *args(0, 10, 256, 128, P))
    expect(INVALID, "n_experts", name, *args(1025, 10, 256, 128, P))
    expect(UNSUPPORTED, "d_model", name, *args(4, 10, 192, 128, P))
    expect(UNSUPPORTED, "d_model", name, *args(4, 10, 0, 128, P))
    expect(UNSUPPORTED, "d_ff", name, *args(4, 10, 256, 64, P))
    expect(UNSUPPORTED, "d_ff", name, *args(4, 10, 256, -128, P))
    expect(INVALID, "rows_cap", name, *args(4, -1, 256, 128, P))
    expect(INVALID, "rows_cap", name, *args(4, 1 << 31, 256, 128, P))
    expect(INVALID, "null", name, *args(4, 10, 256, 128, None))
    expect(INVALID, "aligned", name, *args(4, 10, 256, 128, ODD))
    expect(OK, None, name, *args(4, 0, 256, 128, None))


def test_gather():
    name = "hmoe_grouped_gate_up_mxfp4_gather"
    tail = (P, P, 4, 10, 256, 128, P, P, P, P, S)
    expect(INVALID, "tokens", name, P, P, -1, 2, *tail)
    expect(INVALID, "tokens", name, P, P, 0, 2, *tail)
    expect(INVALID, "top_k", name, P, P, 64, 0, *tail)
    expect(INVALID, "2 GiB", name, P, P, 1 << 24, 2, *tail)
    expect(INVALID, "null", name, P, P, 64, 2, None, P, 4, 10, 256, 128, P, P, P, P, S)


def test_rows():
    for name, args in (("hmoe_quantize_rows_mxfp4", lambda p, t, r, c: (p, t, r, c, p, p, S)),
                       ("hmoe_dequantize_rows_mxfp4", lambda p, t, r, c: (p, p, r, c, p, t, S))):
        expect(UNSUPPORTED, "cols", name, *args(P, F32, 4, 48))
        expect(UNSUPPORTED, "cols", name, *args(P, F32, 4, 0))
        expect(INVALID, "rows", name, *args(P, F32, -1, 64))
        expect(INVALID, "dtype", name, *args(P, E4M3, 4, 64))
        expect(INVALID, "null", name, *args(None, BF16, 4, 64))
        expect(INVALID, "aligned", name, *args(ODD, BF16, 4, 64))
        expect(OK, None, name, *args(None, BF16, 0, 64))


def test_packs():
    for name, args in (("hmoe_pack_mxfp4_gate_up", lambda p, t, n, d, f: (p, p, t, n, d, f, p, p, S)),
                       ("hmoe_pack_mxfp4_down", lambda p, t, n, d, f: (p, t, n, f, d, p, p, S))):
        expect(INVALID, "n_experts", name, *args(P, F32, 0, 256, 128))
        expect(UNSUPPORTED, "d_model", name, *args(P, F32, 2, 200, 128))
        expect(UNSUPPORTED, "d_ff", name, *args(P, F32, 2, 256, 96))
        expect(INVALID, "dtype", name, *args(P, E4M3, 2, 256, 128))
        expect(INVALID, "null", name, *args(None, F32, 2, 256, 128))
        expect(INVALID, "aligned", name, *args(ODD, F32, 2, 256, 128))
    name = "hmoe_unpack_mxfp4"
    expect(INVALID, "n_experts", name, P, P, 0, 256, 128, P, F32, S)
    expect(UNSUPPORTED, "rows", name, P, P, 2, 40, 128, P, F32, S)
    expect(UNSUPPORTED, "cols", name, P, P, 2, 64, 192, P, F32, S)
    expect(INVALID, "dtype", name, P, P, 2, 64, 128, P, E4M3, S)
    expect(INVALID, "null", name, P, P, 2, 64, 128, None, F32, S)
    expect(INVALID, "aligned", name, P, P, 2, 64, 128, ODD, F32, S)


def test_sizes():
    lib = _lib.lib()
    assert lib.hmoe_packed_mxfp4_gate_up_bytes(3, 256, 128) == 3 * 256 * 256 // 2
    assert lib.hmoe_packed_mxfp4_down_bytes(3, 128, 256) == 3 * 128 * 256 // 2
    assert lib.hmoe_packed_mxfp4_gate_up_bytes(0, 256, 128) == 0


def test_form():
    form = _lib.lib().hmoe_grouped_mxfp4_form
    assert form(8, 64, 2048, 2048, 256) == 1 and form(131072, 64, 2048, 2048, 256) == 3
    for bad in ((0, 64, 2048, 2048, 256), (8, 0, 2048, 2048, 256), (8, 2000, 2048, 2048, 256),
                (8, 64, 100, 2048, 256), (8, 64, 2048, 64, 256), (8, 64, 2048, 2048, 0)):
        assert form(*bad) == -1


def test_python_layer():
    """Tensors that are not on a GPU are refused before anything is looked at."""
    x = torch.zeros((4, 64))
    u = torch.zeros((4, 32), dtype=torch.uint8)
    w = torch.zeros((2, 128, 128))
    packed, exps = torch.zeros((2, 8, 2, 64, 16), dtype=torch.uint8), torch.zeros((2, 1, 256, 4), dtype=torch.uint8)
    for call in (lambda: K.quantize_rows_mxfp4(x), lambda: K.dequantize_rows_mxfp4(u, u),
                 lambda: K.pack_mxfp4_gate_up(w, w), lambda: K.pack_mxfp4_down(w),
                 lambda: K.unpack_mxfp4(packed, exps),
                 lambda: K.grouped_gate_up_mxfp4(u, u, u, packed, exps),
                 lambda: K.grouped_gate_up_mxfp4_gather(u, u, None, packed, exps),
                 lambda: K.grouped_down_mxfp4(u, u, u, packed, exps)):
        with pytest.raises(ValueError, match="GPU"):
            call()
    with pytest.raises(TypeError):
        K.quantize_rows_mxfp4([1.0])


def test_module_arguments():
    from hanuman_amd import MoE
    with pytest.raises(ValueError, match="expert_dtype"):
        MoE(256, 128, 4, 2, 1, 0.02, 1.0, "bfloat16", rngs=0, expert_dtype="fp4", device="cpu")
    with pytest.raises(ValueError, match="bfloat16"):
        MoE(256, 128, 4, 2, 1, 0.02, 1.0, "float32", rngs=0, expert_dtype="mxfp4", device="cpu")
    for d, f in ((128, 128), (384, 128), (192, 128), (256, 64)):
        with pytest.raises(ValueError, match="128"):
            MoE(d, f, 4, 2, 1, 0.02, 1.0, "bfloat16", rngs=0, expert_dtype="mxfp4", device="cpu")


def test_limits():
    """Sizes whose rows, tiles or threads would not be counted in 32 bits."""
    for name, args in PRODUCTS:
        expect(INVALID, "rows_cap", name, *args(4, (1 << 30) + 1, 256, 128, P))
        expect(INVALID, "rows_cap", name, *args(1, (1 << 31) - 1, 128, 128, P))
        expect(UNSUPPORTED, "d_model", name, *args(4, 10, 1 << 21, 128, P))
        expect(UNSUPPORTED, "d_ff", name, *args(4, 10, 256, 1 << 21, P))
    for name, args in (("hmoe_pack_mxfp4_gate_up", lambda d, f: (P, P, F32, 1, d, f, P, P, S)),
                       ("hmoe_pack_mxfp4_down", lambda d, f: (P, F32, 1, f, d, P, P, S))):
        expect(UNSUPPORTED, "d_model", name, *args(1 << 21, 128))
        expect(UNSUPPORTED, "d_ff", name, *args(128, 1 << 30))
    expect(INVALID, "too large", "hmoe_unpack_mxfp4", P, P, 1024, 1 << 19, 128, P, BF16, S)
    assert _lib.lib().hmoe_grouped_mxfp4_form((1 << 30) + 1, 4, 256, 256, 256) == -1


def test_router_quant():
    name = "hmoe_router_quant_mxfp4"

    def args(p=P, xt=BF16, wt=F32, t=8, d=64, n=8, k=2, mode=_lib.ROUTE_SOFTMAX):
        return p, xt, p, wt, None, t, d, n, k, mode, 1.0, p, p, p, p, p, S
    expect(UNSUPPORTED, "d_model", name, *args(d=40))
    expect(UNSUPPORTED, "d_model", name, *args(d=0))
    expect(INVALID, "dtype", name, *args(xt=F32))
    expect(INVALID, "dtype", name, *args(wt=E4M3))
    expect(INVALID, "n_experts", name, *args(n=257))
    expect(INVALID, "top_k", name, *args(k=9))
    expect(INVALID, "mode", name, *args(mode=7))
    expect(INVALID, "tokens", name, *args(t=-1))
    expect(INVALID, "null", name, *args(p=None))
    expect(INVALID, "aligned", name, *args(p=ODD))
    expect(OK, None, name, *args(p=None, t=0))
    x = torch.zeros((8, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        K.router_quant_mxfp4(x, torch.zeros((64, 8)), None, 2)

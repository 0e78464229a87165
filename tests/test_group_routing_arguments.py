"""Refusals of routing by groups and of the module's arguments, on the CPU."""
import ctypes

import pytest
import torch

from hanuman_amd import MoE, RMSNorm, _lib, kernels as K

P = ctypes.c_void_p(16)
OK, INVALID = _lib.OK, _lib.ERR_INVALID


def expect(code, needle, name, *args):
    rc = getattr(_lib.lib(), name)(*args)
    msg = _lib.lib().hmoe_last_error().decode()
    assert rc == code, f"{name}{args}: rc {rc}, expected {code} ({msg})"
    if needle:
        assert needle in msg, f"{name}: '{needle}' not in '{msg}'"


CALLS = [
    ("hmoe_router_grouped", lambda t, n, k, mode, g, top, p: (p, _lib.BF16, p, _lib.F32, None, t, 64, n, k, mode, 1.0, g,
                                                              top, p, p, p, None)),
    ("hmoe_router_grouped_from_logits", lambda t, n, k, mode, g, top, p: (p, None, t, n, k, mode, 1.0, g, top, p, p,
                                                                          None)),
]


@pytest.mark.parametrize("name,args", CALLS, ids=[c[0] for c in CALLS])
def test_groups(name, args):
    expect(INVALID, "tokens", name, *args(-1, 64, 8, 0, 8, 4, P))
    expect(INVALID, "2^26", name, *args(1 << 26, 64, 8, 0, 8, 4, P))
    expect(INVALID, "n_experts", name, *args(4, 257, 8, 0, 1, 1, P))
    expect(INVALID, "top_k", name, *args(4, 64, 33, 0, 8, 8, P))
    expect(INVALID, "mode", name, *args(4, 64, 8, 2, 8, 4, P))
    for groups in (0, -8, 7, 65, 128):
        expect(INVALID, "n_groups", name, *args(4, 64, 8, 0, groups, 1, P))
    for top in (0, -1, 9):
        expect(INVALID, "top_groups", name, *args(4, 64, 8, 0, 8, top, P))
    expect(INVALID, "top_k 9", name, *args(4, 64, 9, 0, 8, 1, P))
    expect(INVALID, "two experts", name, *args(4, 64, 8, 0, 64, 8, P))
    expect(INVALID, "null", name, *args(4, 64, 8, 1, 64, 8, None))
    expect(INVALID, "null", name, *args(4, 64, 8, 0, 8, 4, None))
    expect(INVALID, "null", name, *args(4, 64, 8, 0, 8, 8, None))
    expect(OK, None, name, *args(0, 64, 8, 0, 8, 4, None))


def test_python_layer():
    x, w = torch.zeros((4, 64)), torch.zeros((64, 8))
    with pytest.raises(ValueError, match="GPU"):
        K.router(x, w, None, 2, 0, 1.0, 4, 2)
    with pytest.raises(ValueError, match="GPU"):
        K.router_from_logits(torch.zeros((4, 8)), None, 2, 0, 1.0, 4, 2)
    for groups in (3, 0, -2):
        with pytest.raises(ValueError, match="n_groups"):
            K.router(x, w, None, 2, 0, 1.0, groups)


def test_module_arguments():
    def layer(n=12, active=3, routing="sigmoid", dtype="bfloat16", d=256, f=128, **kw):
        return MoE(d, f, n, active, 1, 0.02, 1.0, dtype, rngs=0, device="cpu", routing=routing, **kw)

    assert layer(n_groups=4, top_groups=2).top_groups == 2
    assert layer(n_groups=4).top_groups == 4 and layer().n_groups == 1
    for groups, top in ((5, 2), (0, None), (4, 0), (4, 5), (-1, None)):
        with pytest.raises(ValueError, match="n_groups"):
            layer(n_groups=groups, top_groups=top)
    with pytest.raises(ValueError, match="hold fewer"):
        layer(n_groups=6, top_groups=1)
    with pytest.raises(ValueError, match="two"):
        layer(n_groups=12, top_groups=4)
    assert layer(n_groups=12, top_groups=4, routing="softmax").n_groups == 12
    assert layer(expert_dtype="int8").expert_dtype == "int8"
    with pytest.raises(ValueError, match="bfloat16"):
        layer(expert_dtype="int8", dtype="float32")
    for d, f in ((128, 128), (384, 128), (192, 128), (256, 64)):
        with pytest.raises(ValueError, match="128"):
            layer(expert_dtype="int8", d=d, f=f)
    with pytest.raises(ValueError, match="expert_dtype"):
        layer(expert_dtype="int4")


def test_norm_on_the_cpu():
    norm = RMSNorm(64, device="cpu")
    with pytest.raises(ValueError, match="GPU"):
        norm(torch.zeros((2, 64)))
    with pytest.raises(ValueError, match="shape"):
        norm.with_sum(torch.zeros((2, 64)), torch.zeros((3, 64)))


@pytest.mark.parametrize("name,args", CALLS, ids=[c[0] for c in CALLS])
def test_the_most_tokens(name, args):
    """A launch has fewer than 2^32 threads: 64 for each token with 33 groups and more (four
    tokens a workgroup), and in the router's own launch with more than 240 experts (sixteen)."""
    most = (1 << 26) - 16
    for experts, k in ((66, 2), (256, 8), (256, 12)):
        groups = 33 if experts == 66 else 64
        expect(INVALID, "2^26", name, *args(most + 1, experts, k, 0, groups, 8, P))
        expect(INVALID, "2^26", name, *args((1 << 26) - 3, experts, k, 0, groups, 8, P))
        expect(INVALID, "null", name, *args(most, experts, k, 0, groups, 8, None))
    for per_block, threads in ((4, 256), (16, 1024)):
        assert -(-most // per_block) * threads < 1 << 32


def test_operands_are_checked_in_their_order():
    """Without groups a call is checked as it was before it took any: x first, then the weight."""
    x = torch.zeros((4, 64))
    for w in (None, [1.0], torch.zeros(())):
        with pytest.raises(ValueError, match="x must be on a GPU"):
            K.router(x, w, None, 2)

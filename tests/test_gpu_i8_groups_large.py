"""int8 products and routing by groups on operands and results past 2^31 and 2^32 bytes."""
import pytest
import torch

from hanuman_amd import _lib, kernels as K

pytestmark = pytest.mark.gpu


def _codes(gpu, shape, seed):
    return torch.randint(-127, 128, shape, generator=torch.Generator(device=gpu).manual_seed(seed), device=gpu,
                         dtype=torch.int8)


def _weights(packed):
    """float64 [rows, K] of one expert's packed codes."""
    r, k = packed.shape[:2]
    return packed.reshape(r, k, 2, 32, 16).permute(0, 3, 1, 2, 4).reshape(r * 32, k * 32).double()


def _product(a, a_scale, packed, w_scale):
    """float32 operations on the exact sums, as the products are defined."""
    return (a.double() @ _weights(packed).t()).float() * w_scale * a_scale.unsqueeze(1)


@pytest.mark.parametrize("rows,k,n", [(70000, 128, 32768), (70000, 32768, 128)])
def test_rows_past_32_bits(gpu, rows, k, n):
    """Results of 4.6 GB; rows of 2.3 GB."""
    a, w = _codes(gpu, (rows, k), 1), _codes(gpu, (2, n // 32, k // 32, 64, 16), 2)
    a_s = torch.rand(rows, device=gpu) * 1e-3 + 1e-4
    w_s = torch.rand((2, n), device=gpu) * 1e-3 + 1e-4
    cut = 40000
    off = torch.tensor([0, cut, rows], dtype=torch.int32, device=gpu)
    ys = K.grouped_down_i8(a, a_s, off, w, w_s)
    for lo, hi, e in ((0, 40, 0), (cut - 33, cut, 0), (cut, cut + 20, 1), (rows - 50, rows, 1)):
        assert torch.equal(ys[lo:hi], _product(a[lo:hi], a_s[lo:hi], w[e], w_s[e]).bfloat16()), (lo, hi)


@pytest.mark.parametrize("rows", [9, 2500])
def test_weights_past_32_bits(gpu, rows):
    """An operand of 5.4 GB (few rows straight from memory, many through tiles)."""
    n_experts, k, n = 40, 32768, 4096
    w = _codes(gpu, (n_experts, n // 32, k // 32, 64, 16), 3)
    w_s = torch.rand((n_experts, n), device=gpu) * 1e-3 + 1e-4
    a, a_s = _codes(gpu, (rows, k), 4), torch.rand(rows, device=gpu) * 1e-3 + 1e-4
    off = torch.zeros(n_experts + 1, dtype=torch.int32, device=gpu)
    off[17:] = rows // 3
    off[40:] = rows
    ys = K.grouped_down_i8(a, a_s, off, w, w_s)
    assert torch.equal(ys[:3], _product(a[:3], a_s[:3], w[16], w_s[16]).bfloat16())
    assert torch.equal(ys[-5:], _product(a[-5:], a_s[-5:], w[39], w_s[39]).bfloat16())


def test_gathered_tokens_up_to_the_limit(gpu):
    """Tokens of just under 2 GB, of which the last are gathered."""
    d, f, tokens = 32768, 128, 65535
    x, x_s = _codes(gpu, (tokens, d), 5), torch.rand(tokens, device=gpu) * 1e-3 + 1e-5
    w = _codes(gpu, (1, 2 * f // 32, d // 32, 64, 16), 6)
    w_s = torch.rand((1, 2 * f), device=gpu) * 1e-4 + 1e-5
    for rows in (12, 3000):
        src = torch.arange(tokens - rows, tokens, device=gpu, dtype=torch.int32)
        off = torch.tensor([0, rows], dtype=torch.int32, device=gpu)
        slots = torch.full((tokens,), -1, dtype=torch.int32, device=gpu)
        plan = K.Plan(off[1:].clone(), off, slots, src, slots.bool(), rows, rows, 1, 1)
        h = K.grouped_gate_up_i8_gather(x, x_s, plan, w, w_s)
        straight = K.grouped_gate_up_i8(x[-rows:].contiguous(), x_s[-rows:].contiguous(), off, w, w_s)
        assert torch.equal(h, straight)
        y = _product(x[-3:], x_s[-3:], w[0], w_s[0]).double().reshape(3, -1, 2, 32)
        g, u = y[:, :, 0].reshape(3, f), y[:, :, 1].reshape(3, f)
        want = g * torch.sigmoid(g) * u
        off_by = want.abs() * (2.0**-8 + (1.25 * g.abs() + 8) * 2.0**-24)
        assert ((h[-3:].double() - want).abs() <= off_by + 1e-30).all()


def test_logits_past_32_bits(gpu):
    """8.6 GB of logits: every token's experts are those it has alone."""
    tokens, n = (1 << 23) + 5, 256
    logits = torch.randn((tokens, n), generator=torch.Generator(device=gpu).manual_seed(7), device=gpu)
    bias = torch.randn(n, device=gpu) * 0.05
    idx, gates = K.router_from_logits(logits, bias, 8, _lib.ROUTE_SIGMOID_BIAS, 2.5, 8, 3)
    for lo in (0, (1 << 22) - 2, (1 << 23) - 3, tokens - 7):
        part = K.router_from_logits(logits[lo:lo + 7].clone(), bias, 8, _lib.ROUTE_SIGMOID_BIAS, 2.5, 8, 3)
        assert torch.equal(part[0], idx[lo:lo + 7]) and torch.equal(part[1], gates[lo:lo + 7])

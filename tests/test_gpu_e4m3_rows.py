"""e4m3 rows that are not ordinary on the GPU: NaN, infinities, and rows so small that 448 over
their largest value passes float32's range, in every call that quantises rows by that rule."""
import numpy as np
import pytest
import torch

import oracle as O
from hanuman_amd import kernels as K

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
BAD = {1: [(0, np.nan)], 2: [(-1, -np.nan)], 3: [(5, np.inf)], 4: [(-3, -np.inf)],
       5: [(0, np.inf), (9, -np.inf), (-1, np.nan)]}
SMALL = {7: 2.0**-119, 8: 1e-36, 9: 2.0**-126, 10: 3e-39, 11: 2.0**-133}


def _rows(gpu, cols, dtype, n=13):
    g = torch.Generator().manual_seed(cols)
    a = torch.randn((n, cols), generator=g).to(BF16).float()
    for row, places in BAD.items():
        for at, value in places:
            a[row, at] = value
    a[6] = 0.0
    for row, most in SMALL.items():
        a[row] = (a[row].double() / a[row].abs().max() * most).float()
    return a.to(dtype).to(gpu)


def _same(q, scale, a):
    """Codes and scales are the rule's; rows that are not finite read back as NaN, no others."""
    want_q, want_s = O.quantize_rows_e4m3(a.float().cpu().numpy())
    assert np.array_equal(scale.cpu().numpy(), want_s, equal_nan=True)
    assert np.array_equal(q.cpu().numpy(), want_q)
    back = K.dequantize_rows_fp8(q, scale, F32)
    finite = torch.isfinite(a).all(1)
    assert torch.isnan(back[~finite]).all() and torch.isfinite(back[finite]).all()
    # half a step of a code, four float32 roundings, and the scale's own where it is subnormal
    v, b, s = a[finite].double(), back[finite].double(), scale[finite].double().unsqueeze(1)
    bound = torch.maximum(v.abs() * 2.0**-4, 2.0**-10 * s) * (1 + 2.0**-20) + v.abs() * 4 * 2.0**-24 + 449 * 2.0**-150
    assert ((b - v).abs() <= bound).all()


# rows in registers and rows that are read twice
@pytest.mark.parametrize("cols", [16, 264, 4096, 4104])
def test_quantize_rows(gpu, cols):
    a = _rows(gpu, cols, BF16)
    _same(*K.quantize_rows_fp8(a), a)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("cols", [264, 4104])
def test_permuted_rows(gpu, cols, dtype):
    a = _rows(gpu, cols, dtype)
    idx = torch.tensor([[t % 4] for t in range(a.shape[0])], dtype=torch.int32, device=gpu)
    plan = K.dispatch_plan(idx, 4, a.shape[0])
    q, scale = K.permute_rows_fp8(a, plan)
    pos = plan.slot_pos.long()
    _same(q[pos].contiguous(), scale[pos].contiguous(), a)


@pytest.mark.parametrize("cols", [256, 4352])
def test_in_the_routers_launch(gpu, cols):
    a = _rows(gpu, cols, BF16)
    w = 0.02 * torch.randn((cols, 16), generator=torch.Generator(device=gpu).manual_seed(1), device=gpu)
    *_, q, scale = K.router_quant_fp8(a, w, None, 2)
    _same(q, scale, a)


# a row by a wave, by a workgroup of 256 and of 1024
@pytest.mark.parametrize("rows,cols", [(13, 264), (13, 8208), (2053, 264), (2053, 2048)])
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_of_the_norm(gpu, rows, cols, dtype):
    a = _rows(gpu, cols, dtype, max(13, rows))
    out = K.add_rms_norm(a, torch.ones(cols, device=gpu), None, 1e-6, quant="e4m3")
    bad = sorted(BAD)
    assert torch.isnan(out.scale[bad]).all() and torch.isfinite(out.scale).sum() == rows - len(bad)
    assert torch.isnan(K.dequantize_rows_fp8(out.q, out.scale, F32)[bad]).all()
    _same(out.q, out.scale, out.y)
    # a weight that leaves every row that small (its bf16 would be rounded to 8 bits, which is all that it has)
    for most in (1e-36, 2.0**-126, 3e-39):
        w = torch.full((cols,), most / 16, device=gpu)
        out = K.add_rms_norm(a, w, None, 1e-6, quant="e4m3")
        _same(out.q, out.scale, out.y)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_columns_of_the_masters(gpu, dtype):
    """Output columns that are not ordinary, of the gate, the up and the down master."""
    k, cols, n = 96, 64, 2
    bad, tiny = [1, 33, 40], {2: 1e-36, 34: 2.0**-126, 5: 3e-39}

    def master(seed):
        w = 0.02 * torch.randn((n, k, cols), generator=torch.Generator().manual_seed(seed))
        w[0, 3, 1], w[0, k - 1, 33], w[0, 0, 40] = float("nan"), float("inf"), -float("inf")
        w[1, :, 0] = 0.0
        for col, most in tiny.items():
            w[1, :, col] = (w[1, :, col].double() / w[1, :, col].abs().max() * most).float()
        return w.to(dtype).to(gpu)

    def rule(w):
        q, s = O.quantize_cols_e4m3(w.float().cpu().numpy())
        assert np.array_equal(np.isnan(s[0]), np.isin(np.arange(cols), bad)) and not np.isnan(s[1]).any()
        return np.swapaxes(q, 1, 2), s

    wg, wu = master(1), master(2)
    packed, scale = (t.cpu().numpy() for t in K.pack_fp8_gate_up(wg, wu))
    for up, w in enumerate((wg, wu)):
        at = [(c // 32) * 64 + 32 * up + c % 32 for c in range(cols)]
        q, s = rule(w)
        assert np.array_equal(scale[:, at], s, equal_nan=True) and np.array_equal(packed[:, at], q)
    packed, scale = (t.cpu().numpy() for t in K.pack_fp8_down(wg))
    q, s = rule(wg)
    assert np.array_equal(scale, s, equal_nan=True) and np.array_equal(packed, q)


# few rows an expert, and tiles of 256
@pytest.mark.parametrize("tokens,n,top_k", [(24, 16, 2), (3000, 4, 2)], ids=["few", "tiles"])
def test_block_scaled_h(gpu, tokens, n, top_k):
    """Tokens that are not finite, and ones whose h overflows in some columns, through the
    products: exponents 255 where h is not finite, NaN in those tokens' results only."""
    d, f = 256, 256
    g = torch.Generator(device=gpu).manual_seed(tokens)
    x = torch.randn((tokens, d), generator=g, device=gpu).to(BF16)
    clean = x.clone()
    x[2, 7], x[11, 0], x[19, 255] = float("nan"), float("inf"), -float("inf")
    x[5] = x[5] * 2.0**65               # g and u about 0.3 * 2^65: one h in 30 passes 2^128
    wg, wu, wd = (0.02 * torch.randn(s, generator=g, device=gpu) for s in ((n, d, f), (n, d, f), (n, f, d)))
    gu, gu_s = K.pack_fp8_gate_up(wg, wu)
    dn, dn_s = K.pack_fp8_down(wd)
    idx = torch.stack([torch.randperm(n, generator=torch.Generator().manual_seed(t))[:top_k] for t in range(tokens)])
    plan = K.dispatch_plan(idx.to(torch.int32).to(gpu), n, tokens * top_k)
    token = plan.perm_src.long() // top_k

    def run(t):
        t_q, t_s = K.quantize_rows_fp8(t)
        h = K.grouped_gate_up_fp8_gather(t_q, t_s, plan, gu, gu_s)
        h_q, h_exp = K.grouped_gate_up_fp8_gather_qh(t_q, t_s, plan, gu, gu_s)
        return h, h_exp, K.grouped_down_fp8_mx(h_q, h_exp, plan.offsets, dn, dn_s)

    h, h_exp, ys = run(x)
    lost = ~torch.isfinite(h).view(-1, f // 32, 32).all(2)
    assert torch.equal(h_exp == 255, lost)
    assert lost[(token == 2) | (token == 11) | (token == 19)].all()
    over = lost[token == 5]
    assert over.any() and not over.all()
    assert torch.equal(torch.isnan(ys).all(1), lost.any(1)) and torch.equal(torch.isnan(ys).any(1), lost.any(1))
    same = ~((token == 2) | (token == 11) | (token == 19) | (token == 5))
    _, _, want = run(clean)
    assert torch.equal(ys[same], want[same])

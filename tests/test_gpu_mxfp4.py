"""MXFP4 rows, operands and products on the GPU against float64."""
import numpy as np
import pytest
import torch

import mxfp4_reference as R
from hanuman_amd import _lib, kernels as K

pytestmark = pytest.mark.gpu


def _to(a, dev):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


def _bf16(v):
    return torch.from_numpy(np.ascontiguousarray(v, dtype=np.float32)).bfloat16()


# ------------------------------------------------------------ rows and back --

def _rows(kind, rng):
    """float32 rows where quantising can go wrong."""
    if kind == "normal":
        return rng.standard_normal((37, 96)).astype(np.float32)
    if kind == "one":
        return rng.standard_normal((1, 32)).astype(np.float32)
    if kind == "wide":      # every block at a size of its own, over float32's range
        return (rng.standard_normal((64, 1056)) * np.exp2(rng.integers(-126, 125, (64, 33))).repeat(32, 1)).astype(np.float32)
    if kind == "ties":      # multiples of a quarter of a unit, at 60 scales: borders among them
        return (rng.integers(-28, 29, (120, 64)) * 0.25 * np.exp2(rng.integers(-60, 60, (120, 1)))).astype(np.float32)
    if kind == "small":     # blocks of subnormals and zeros of both signs
        v = (rng.integers(-9, 10, (40, 64)) * 2.0**-149 * np.exp2(rng.integers(0, 26, (40, 1)))).astype(np.float32)
        v[3] = 0.0
        v[4] = -0.0
        return v
    if kind == "edges":     # largest values of a block around 7 units, at the range's ends
        v = np.zeros((16, 32), dtype=np.float32)
        for i, a in enumerate((7.0, 6.999999, 7.000001, 6.5, 3.5, 3.4999998)):
            v[i, 5] = -a
            v[i, 6] = a / 3
        v[6, 0] = np.finfo(np.float32).max
        v[7, 0] = 1.7 * 2.0**127
        v[8, 0] = 2.0**-149
        v[9, 0] = 2.0**-126
        return v
    v = rng.standard_normal((12, 96)).astype(np.float32)   # "special"
    v[0, 3] = np.inf
    v[1, 40] = -np.inf
    v[2, 95] = np.nan
    v[3, 31] = np.nan
    v[3, 0] = np.inf
    return v


KINDS = ("normal", "one", "wide", "ties", "small", "edges", "special")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_quantised_rows(gpu, kind, dtype):
    v = torch.from_numpy(_rows(kind, np.random.default_rng(5))).to(dtype)
    q, e = K.quantize_rows_mxfp4(v.to(gpu))
    want_q, want_e = R.quantise(v.float().numpy())
    assert np.array_equal(e.cpu().numpy(), want_e)
    assert np.array_equal(q.cpu().numpy(), want_q)
    for out in (torch.float32, torch.bfloat16):
        back = K.dequantize_rows_mxfp4(q, e, out).cpu()
        with np.errstate(over="ignore"):
            want = torch.from_numpy(R.values(want_q, want_e).astype(np.float32)).to(out)
        assert torch.equal(torch.nan_to_num(back, 7e30), torch.nan_to_num(want, 7e30))
        assert torch.equal(torch.isnan(back), torch.isnan(want))


def test_every_bf16_value(gpu):
    """Every bf16 number, each in a block with a larger one eight octaves up at most."""
    rng = np.random.default_rng(9)
    bits = np.arange(0x0000, 0x7F80, dtype=np.uint32)
    v = (bits << 16).view(np.float32).repeat(2)
    v[1::2] *= -1
    v = np.concatenate([v, np.zeros(-len(v) % 31, dtype=np.float32)]).reshape(-1, 31)
    with np.errstate(over="ignore"):
        top = np.abs(v).max(1, keepdims=True) * np.exp2(rng.integers(0, 9, (len(v), 1)))
    top = np.minimum(top, 3e38).astype(np.float32)
    t = _bf16(np.concatenate([v, top], 1))
    q, e = K.quantize_rows_mxfp4(t.to(gpu))
    want_q, want_e = R.quantise(t.float().numpy())
    assert np.array_equal(e.cpu().numpy(), want_e)
    assert np.array_equal(q.cpu().numpy(), want_q)


def test_rows_larger_than_the_grid(gpu):
    """More chunks than one pass of the grid covers, checked where the passes meet."""
    rows, cols = 4200, 32768
    g = torch.Generator(device=gpu).manual_seed(3)
    x = torch.randn((rows, cols), generator=g, device=gpu, dtype=torch.bfloat16)
    q, e = K.quantize_rows_mxfp4(x)
    back = K.dequantize_rows_mxfp4(q, e)
    for r in (0, 1, 4095, 4096, rows - 1):
        want_q, want_e = R.quantise(x[r:r + 1].float().cpu().numpy())
        assert np.array_equal(q[r:r + 1].cpu().numpy(), want_q)
        assert np.array_equal(e[r:r + 1].cpu().numpy(), want_e)
        assert np.array_equal(back[r:r + 1].float().cpu().numpy(), R.values(want_q, want_e))


# ----------------------------------------------------------------- operands --

@pytest.mark.parametrize("N,D,F", [(1, 128, 128), (3, 384, 128), (2, 128, 640), (5, 640, 256)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_packed_operands(gpu, N, D, F, dtype):
    rng = np.random.default_rng(N * D + F)
    wg, wu, wd = (torch.from_numpy((rng.standard_normal(s) * np.exp2(rng.integers(-9, 9, s))).astype(np.float32)).to(dtype)
                  for s in ((N, D, F), (N, D, F), (N, F, D)))
    wd[0, 3, 1] = float("inf")
    gu, gu_e = K.pack_mxfp4_gate_up(wg.to(gpu), wu.to(gpu))
    dn, dn_e = K.pack_mxfp4_down(wd.to(gpu))
    gu_v, dn_v = K.unpack_mxfp4(gu, gu_e), K.unpack_mxfp4(dn, dn_e, torch.float32)
    for n in range(N):
        rows = np.empty((2 * F, D), dtype=np.float32)
        for p in range(2 * F):
            which, c = R.gate_up_column(p, F)
            rows[p] = (wu if which else wg)[n, :, c].float().numpy()
        for rows, codes, exps, vals in ((rows, gu[n], gu_e[n], gu_v[n]),
                                        (wd[n].float().numpy().T, dn[n], dn_e[n], dn_v[n])):
            want_q, want_e = R.quantise(rows)
            q, e = R.operand_rows(codes.cpu().numpy(), exps.cpu().numpy())
            assert np.array_equal(e, want_e) and np.array_equal(q, want_q)
            assert np.array_equal(vals.float().cpu().numpy(), R.values(want_q, want_e).astype(np.float32),
                                  equal_nan=True)


# ----------------------------------------------------------------- products --

def _case(tokens, experts, active, d_model, d_ff, seed, gpu, skew=0.0, capacity=None):
    """A quantised layer: tokens, operands (host and GPU) and the library's plan."""
    rng = np.random.default_rng(seed)
    x = _bf16(rng.standard_normal((tokens, d_model)) * np.exp(rng.standard_normal((tokens, 1))))
    logits = rng.standard_normal((tokens, experts)) - skew * np.arange(experts)
    top = np.argsort(-logits, axis=1)[:, :active].astype(np.int32)
    cap = tokens * active if capacity is None else capacity
    plan = K.dispatch_plan(_to(top, gpu), experts, cap)
    host = []
    for rows, k in ((2 * d_ff, d_model), (d_model, d_ff)):
        host.append([R.quantise(rng.standard_normal((rows, k)) * 0.05) for _ in range(experts)])
    ops = []
    for side in host:
        packed = [R.packed_operand(q, e) for q, e in side]
        ops.append((_to(np.stack([p for p, _ in packed]), gpu), _to(np.stack([e for _, e in packed]), gpu)))
    return x, plan, host, ops


def _check_gate_up(h_q, h_exp, x_vals, plan, weights, d_ff, top_k):
    off = plan.offsets.cpu().numpy()
    src = plan.perm_src.cpu().numpy()
    h_q, h_exp = h_q.cpu().numpy(), h_exp.cpu().numpy()
    gate = np.array([p for p in range(2 * d_ff) if R.gate_up_column(p, d_ff)[0] == 0])
    for e, (wq, we) in enumerate(weights):
        lo, hi = off[e], off[e + 1]
        if lo == hi:
            continue
        w, a = R.values(wq, we), x_vals[src[lo:hi] // top_k]
        gu, bound = a @ w.T, R.product_bound(a, w, w.shape[1])
        h, d = R.swiglu_with_bound(gu[:, gate], gu[:, gate + 32], bound[:, gate], bound[:, gate + 32])
        R.check_quantised(h_q[lo:hi], h_exp[lo:hi], h, d, f"expert {e}")


def _check_down(ys, h_vals, off, weights):
    ys = ys.double().cpu().numpy()
    for e, (wq, we) in enumerate(weights):
        lo, hi = off[e], off[e + 1]
        if lo == hi:
            continue
        w, a = R.values(wq, we), h_vals[lo:hi]
        want = a @ w.T
        # one rounding to bf16 (half a step: 2^-8 of the value) of a float32 sum
        allowed = np.abs(want) * 2.0**-8 + R.product_bound(a, w, w.shape[1]) * (1 + 2.0**-8) + 1e-38
        off_by = np.abs(ys[lo:hi] - want) - allowed
        assert (off_by <= 0).all(), f"expert {e}: {int((off_by > 0).sum())} values, worst {off_by.max()}"


SHAPES = [
    # tokens, experts, active, d_model, d_ff
    (1, 4, 2, 128, 128),        # one token
    (1, 1, 1, 384, 256),
    (5, 8, 2, 256, 128),
    (31, 3, 1, 640, 384),       # odd multiples of 128 both ways
    (33, 2, 2, 128, 640),       # a row more than a tile of 32
    (64, 40, 3, 256, 256),      # experts without rows
    (100, 64, 8, 384, 128),
    (200, 70, 5, 128, 128),     # more experts than a wave has lanes
    (257, 2, 1, 512, 384),      # a row more than a tile of 256, halved
    (700, 2, 2, 384, 640),
    (1300, 3, 2, 256, 128),
]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_products(gpu, shape):
    tokens, experts, active, d_model, d_ff = shape
    x, plan, (gu_w, dn_w), (gu, dn) = _case(*shape, seed=sum(shape), gpu=gpu)
    x_q, x_e = K.quantize_rows_mxfp4(x.to(gpu))
    h_q, h_e = K.grouped_gate_up_mxfp4_gather(x_q, x_e, plan, *gu)
    x_vals = R.values(x_q.cpu().numpy(), x_e.cpu().numpy())
    _check_gate_up(h_q, h_e, x_vals, plan, gu_w, d_ff, active)
    # the same rows in the experts' order: the same bits
    src = plan.perm_src.long() // active
    g_q, g_e = K.grouped_gate_up_mxfp4(x_q[src].contiguous(), x_e[src].contiguous(), plan.offsets, *gu)
    assert torch.equal(g_q, h_q) and torch.equal(g_e, h_e)
    ys = K.grouped_down_mxfp4(h_q, h_e, plan.offsets, *dn)
    _check_down(ys, R.values(h_q.cpu().numpy(), h_e.cpu().numpy()), plan.offsets.cpu().numpy(), dn_w)
    # and once more, into other buffers: the same bits
    assert torch.equal(K.grouped_down_mxfp4(h_q, h_e, plan.offsets, *dn), ys)


FORMS = [
    # the shape, and the form that its gate/up and down products take; tiles go in steps
    # of 256 values
    ((9000, 3, 1, 128, 256), 2, 0),     # half a step a tile
    ((6000, 3, 1, 128, 1280), 2, 1),
    ((8000, 2, 1, 256, 384), 2, 0),     # one step
    ((3000, 4, 2, 640, 384), 2, 0),     # two and a half
    ((2600, 2, 2, 512, 1152), 2, 2),    # two; four and a half, a last column tile of 128
    ((1500, 20, 2, 640, 1152), 2, 0),   # segments that end inside tiles
    ((7000, 1, 1, 1152, 1152), 3, 2),
    ((10000, 1, 1, 1152, 640), 3, 3),   # a last column tile of 128
    ((50000, 1, 1, 128, 1152), 3, 0),   # half a step a tile of 128 rows
]


@pytest.mark.parametrize("shape,gate_up,down", FORMS, ids=lambda s: "x".join(map(str, s)) if isinstance(s, tuple) else str(s))
def test_forms(gpu, shape, gate_up, down):
    tokens, experts, active, d_model, d_ff = shape
    cus = torch.cuda.get_device_properties(gpu).multi_processor_count // 8 * 8
    form = _lib.lib().hmoe_grouped_mxfp4_form
    if cus == 256:
        assert form(tokens * active, experts, d_model, 2 * d_ff, cus) == gate_up
        assert form(tokens * active, experts, d_ff, d_model, cus) == down
    test_products(gpu, shape)


def test_forms_agree(gpu):
    """The first expert's rows alone, in registers, and among many, through LDS: the same
    sums in the same order."""
    D, F, rows = 384, 640, 6000
    rng = np.random.default_rng(12)
    x_q, x_e = K.quantize_rows_mxfp4(torch.randn((rows, D), device=gpu))
    gu = [_to(np.stack(t), gpu) for t in zip(*(R.packed_operand(*R.quantise(rng.standard_normal((2 * F, D)))) for _ in range(2)))]
    off = torch.tensor([0, 70, rows], dtype=torch.int32, device=gpu)
    form = _lib.lib().hmoe_grouped_mxfp4_form
    assert form(rows, 2, D, 2 * F, 256) >= 2 and form(70, 2, D, 2 * F, 256) == 0
    many = K.grouped_gate_up_mxfp4(x_q, x_e, off, *gu)
    few = K.grouped_gate_up_mxfp4(x_q[:70].contiguous(), x_e[:70].contiguous(), off.clamp(max=70), *gu)
    assert torch.equal(many[0][:70], few[0]) and torch.equal(many[1][:70], few[1])


@pytest.mark.parametrize("shape,skew", [((300, 6, 1, 256, 128), 3.0), ((90, 20, 2, 128, 256), 1.0)])
def test_skewed_products(gpu, shape, skew):
    """Nearly all rows on the first experts, the last ones empty."""
    x, plan, (gu_w, dn_w), (gu, dn) = _case(*shape, seed=11, gpu=gpu, skew=skew)
    assert (plan.counts == 0).any()
    x_q, x_e = K.quantize_rows_mxfp4(x.to(gpu))
    h_q, h_e = K.grouped_gate_up_mxfp4_gather(x_q, x_e, plan, *gu)
    _check_gate_up(h_q, h_e, R.values(x_q.cpu().numpy(), x_e.cpu().numpy()), plan, gu_w, shape[4], shape[2])
    ys = K.grouped_down_mxfp4(h_q, h_e, plan.offsets, *dn)
    _check_down(ys, R.values(h_q.cpu().numpy(), h_e.cpu().numpy()), plan.offsets.cpu().numpy(), dn_w)


@pytest.mark.parametrize("rows_cap", [40, 700])
def test_rows_past_the_segments_stay(gpu, rows_cap):
    """Buffers with more rows than the segments have: the others are left as they were."""
    N, D, F = 3, 256, 128
    off = torch.tensor([0, 7, 7, 33], dtype=torch.int32, device=gpu)
    rng = np.random.default_rng(2)
    x_q, x_e = K.quantize_rows_mxfp4(torch.randn((rows_cap, D), device=gpu))
    gu = [_to(np.stack(t), gpu) for t in zip(*(R.packed_operand(*R.quantise(rng.standard_normal((2 * F, D)))) for _ in range(N)))]
    dn = [_to(np.stack(t), gpu) for t in zip(*(R.packed_operand(*R.quantise(rng.standard_normal((D, F)))) for _ in range(N)))]
    h_q = torch.full((rows_cap, F // 2), 0xA5, dtype=torch.uint8, device=gpu)
    h_e = torch.full((rows_cap, F // 32), 0xA5, dtype=torch.uint8, device=gpu)
    ys = torch.full((rows_cap, D), 7.0, dtype=torch.bfloat16, device=gpu)
    s = torch.cuda.current_stream().cuda_stream
    _lib.call("hmoe_grouped_gate_up_mxfp4", x_q.data_ptr(), x_e.data_ptr(), off.data_ptr(), N, rows_cap, D, F,
              gu[0].data_ptr(), gu[1].data_ptr(), h_q.data_ptr(), h_e.data_ptr(), s)
    _lib.call("hmoe_grouped_down_mxfp4", h_q.data_ptr(), h_e.data_ptr(), off.data_ptr(), N, rows_cap, F, D,
              dn[0].data_ptr(), dn[1].data_ptr(), ys.data_ptr(), s)
    assert (h_q[33:] == 0xA5).all() and (h_e[33:] == 0xA5).all() and (ys[33:] == 7.0).all()
    want_q, want_e = K.grouped_gate_up_mxfp4(x_q[:33].contiguous(), x_e[:33].contiguous(), off, *gu)
    assert torch.equal(h_q[:33], want_q) and torch.equal(h_e[:33], want_e)


def test_rows_inside_a_buffer(gpu):
    """Operands that start at a later row of their buffers: exponents then lie on words only."""
    D, F = 384, 128
    rng = np.random.default_rng(14)
    x_q, x_e = K.quantize_rows_mxfp4(torch.randn((2003, D), device=gpu))
    gu = [_to(t[None], gpu) for t in R.packed_operand(*R.quantise(rng.standard_normal((2 * F, D))))]
    dn = [_to(t[None], gpu) for t in R.packed_operand(*R.quantise(rng.standard_normal((D, F))))]
    for start, rows in ((1, 33), (3, 2000)):
        off = torch.tensor([0, rows], dtype=torch.int32, device=gpu)
        a_q, a_e = x_q[start:start + rows], x_e[start:start + rows]
        assert a_e.data_ptr() % 16 != 0
        h = K.grouped_gate_up_mxfp4(a_q, a_e, off, *gu)
        want = K.grouped_gate_up_mxfp4(a_q.clone(), a_e.clone(), off, *gu)
        assert torch.equal(h[0], want[0]) and torch.equal(h[1], want[1])
        h_q, h_e = (torch.cat((t[:1], t)) for t in h)
        assert torch.equal(K.grouped_down_mxfp4(h_q[1:], h_e[1:], off, *dn), K.grouped_down_mxfp4(*h, off, *dn))
    assert torch.equal(K.dequantize_rows_mxfp4(x_q[1:], x_e[1:]), K.dequantize_rows_mxfp4(x_q, x_e)[1:])


def test_dropped_slots(gpu):
    """A capacity that drops slots: the kept rows are right, and combine leaves out the others."""
    shape = (64, 4, 2, 256, 128)
    x, plan, (gu_w, dn_w), (gu, dn) = _case(*shape, seed=4, gpu=gpu, skew=1.0, capacity=20)
    assert int(plan.offsets[-1]) < 128
    x_q, x_e = K.quantize_rows_mxfp4(x.to(gpu))
    h_q, h_e = K.grouped_gate_up_mxfp4_gather(x_q, x_e, plan, *gu)
    _check_gate_up(h_q, h_e, R.values(x_q.cpu().numpy(), x_e.cpu().numpy()), plan, gu_w, 128, 2)
    ys = K.grouped_down_mxfp4(h_q, h_e, plan.offsets, *dn)
    _check_down(ys, R.values(h_q.cpu().numpy(), h_e.cpu().numpy()), plan.offsets.cpu().numpy(), dn_w)


def test_nan_blocks(gpu):
    """A token with a value that is not finite gives NaN in its rows alone."""
    shape = (40, 4, 2, 256, 128)
    x, plan, _, (gu, dn) = _case(*shape, seed=8, gpu=gpu)
    x[3, 100] = float("nan")
    x[17, 0] = float("inf")
    x_q, x_e = K.quantize_rows_mxfp4(x.to(gpu))
    h_q, h_e = K.grouped_gate_up_mxfp4_gather(x_q, x_e, plan, *gu)
    token = plan.perm_src.long() // 2
    bad = (token == 3) | (token == 17)
    assert (h_e[bad] == 255).all() and (h_e[~bad] < 255).all()
    ys = K.grouped_down_mxfp4(h_q, h_e, plan.offsets, *dn)
    assert torch.isnan(ys[bad]).all() and torch.isfinite(ys[~bad]).all()


def test_scale_extremes(gpu):
    """Operands at the ends of the exponents' range: sums that stay in float32."""
    N, D, F = 1, 128, 128
    rng = np.random.default_rng(6)
    off = torch.tensor([0, 9], dtype=torch.int32, device=gpu)
    for hi, lo in ((250, 20), (1, 200), (127, 127)):
        h_q = rng.integers(0, 256, (9, F // 2), dtype=np.uint8)
        h_e = np.full((9, F // 32), hi, dtype=np.uint8) - rng.integers(0, 2, (9, F // 32), dtype=np.uint8)
        w_q, w_e = rng.integers(0, 256, (D, F // 2), dtype=np.uint8), np.full((D, F // 32), lo, dtype=np.uint8)
        packed, exps = R.packed_operand(w_q, w_e)
        ys = K.grouped_down_mxfp4(_to(h_q, gpu), _to(h_e, gpu), off, _to(packed[None], gpu), _to(exps[None], gpu))
        _check_down(ys, R.values(h_q, h_e), [0, 9], [(w_q, w_e)])


def test_against_the_bf16_products(gpu):
    """The bf16 down product on the same values widened to bf16: two float32 sums of the
    same exact products, each rounded once."""
    shape = (150, 5, 2, 512, 256)
    x, plan, _, (gu, dn) = _case(*shape, seed=21, gpu=gpu)
    x_q, x_e = K.quantize_rows_mxfp4(x.to(gpu))
    h_q, h_e = K.grouped_gate_up_mxfp4_gather(x_q, x_e, plan, *gu)
    a = K.grouped_down_mxfp4(h_q, h_e, plan.offsets, *dn).float()
    h = K.dequantize_rows_mxfp4(h_q, h_e)
    w = K.unpack_mxfp4(*dn)
    b = K.grouped_down(h, plan.offsets, w).float()
    off = plan.offsets.cpu().numpy()
    for e in range(5):
        lo, hi = off[e], off[e + 1]
        size = h[lo:hi].float().abs() @ w[e].float().abs().t()
        # two roundings of half a bf16 step each, two float32 sums
        allowed = 2 * 2.0**-8 * b[lo:hi].abs() + 2 * 256 * 2.0**-23 * size + 1e-30
        assert ((a[lo:hi] - b[lo:hi]).abs() <= allowed).all()


def test_captured_and_replayed(gpu):
    """The whole run in a graph, replayed on new tokens with eager work between."""
    shape = (48, 8, 2, 256, 256)
    x, plan, _, (gu, dn) = _case(*shape, seed=31, gpu=gpu)
    gates = torch.rand((48, 2), device=gpu)
    static = x.to(gpu)

    def step(t):
        x_q, x_e = K.quantize_rows_mxfp4(t)
        h_q, h_e = K.grouped_gate_up_mxfp4_gather(x_q, x_e, plan, *gu)
        return K.combine(K.grouped_down_mxfp4(h_q, h_e, plan.offsets, *dn), plan, gates)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for i in range(4):
        new = torch.randn((48, 256), device=gpu, generator=torch.Generator(device=gpu).manual_seed(i)).bfloat16()
        static.copy_(new)
        graph.replay()
        got = out.clone()
        want = step(new)
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_two_streams_at_once(gpu):
    """Calls on two streams: no scratch is shared between them."""
    shape = (200, 8, 2, 512, 256)
    x, plan, _, (gu, dn) = _case(*shape, seed=41, gpu=gpu)
    tokens = [x.to(gpu), (x * 0.5).to(gpu)]

    def run(t):
        h_q, h_e = K.grouped_gate_up_mxfp4_gather(*K.quantize_rows_mxfp4(t), plan, *gu)
        return K.grouped_down_mxfp4(h_q, h_e, plan.offsets, *dn)

    want = [run(t) for t in tokens]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in tokens]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(tokens[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for y in got[i]:
            assert torch.equal(y, want[i])


def test_zero_rows(gpu):
    q, e = K.quantize_rows_mxfp4(torch.empty((0, 256), device=gpu))
    assert q.shape == (0, 128) and e.shape == (0, 8)
    assert K.dequantize_rows_mxfp4(q, e).shape == (0, 256)
    rng = np.random.default_rng(0)
    gu = [_to(t[None], gpu) for t in R.packed_operand(*R.quantise(rng.standard_normal((256, 256))))]
    off = torch.zeros(2, dtype=torch.int32, device=gpu)
    h_q, h_e = K.grouped_gate_up_mxfp4(q, e, off, *gu)
    assert h_q.shape == (0, 64) and h_e.shape == (0, 4)
    dn = [_to(t[None], gpu) for t in R.packed_operand(*R.quantise(rng.standard_normal((256, 128))))]
    assert K.grouped_down_mxfp4(h_q, h_e, off, *dn).shape == (0, 256)


def test_rows_past_32_bits(gpu):
    """Rows whose codes (2.2 GB) and results (9 GB) lie past 2^31 and 2^32 bytes: the last
    ones as in a call of their own."""
    rows, D, F, tail = 2_200_003, 2048, 128, 20_001
    form = _lib.lib().hmoe_grouped_mxfp4_form
    assert min(form(rows, 2, D, 2 * F, 256), form(tail, 1, D, 2 * F, 256), form(rows, 2, F, D, 256),
               form(tail, 1, F, D, 256)) >= 2
    g = torch.Generator(device=gpu).manual_seed(3)
    x_q = torch.randint(0, 256, (rows, D // 2), dtype=torch.uint8, device=gpu, generator=g)
    x_e = torch.randint(120, 128, (rows, D // 32), dtype=torch.uint8, device=gpu, generator=g)
    gu = K.pack_mxfp4_gate_up(*(torch.randn((2, D, F), device=gpu, generator=g) * 0.05 for _ in range(2)))
    dn = K.pack_mxfp4_down(torch.randn((2, F, D), device=gpu, generator=g))
    off = torch.tensor([0, rows - tail, rows], dtype=torch.int32, device=gpu)
    one = torch.tensor([0, tail], dtype=torch.int32, device=gpu)
    h_q, h_e = K.grouped_gate_up_mxfp4(x_q, x_e, off, *gu)
    last = [t[1:].contiguous() for t in gu]
    w_q, w_e = K.grouped_gate_up_mxfp4(x_q[-tail:].contiguous(), x_e[-tail:].contiguous(), one, *last)
    assert torch.equal(h_q[-tail:], w_q) and torch.equal(h_e[-tail:], w_e)
    ys = K.grouped_down_mxfp4(h_q, h_e, off, *dn)
    want = K.grouped_down_mxfp4(w_q, w_e, one, *(t[1:].contiguous() for t in dn))
    assert torch.equal(ys[-tail:], want) and bool(want.isfinite().all()) and float(want.float().abs().max()) > 0
    del ys
    # and read back, 9 GB
    back = K.dequantize_rows_mxfp4(x_q, x_e)[-3:]
    assert torch.equal(back, K.dequantize_rows_mxfp4(x_q[-3:].contiguous(), x_e[-3:].contiguous()))


def test_weights_past_32_bits(gpu):
    """An operand of 4.3 GB: the last experts as in calls of their own."""
    N, D, F, rows = 1024, 4096, 1024, 40
    form = _lib.lib().hmoe_grouped_mxfp4_form
    assert form(rows, N, D, 2 * F, 256) == form(3, 1, D, 2 * F, 256)
    g = torch.Generator(device=gpu).manual_seed(4)
    w_q = torch.randint(0, 256, (N, 2 * F // 32, D // 64, 64, 16), dtype=torch.uint8, device=gpu, generator=g)
    w_e = torch.randint(115, 124, (N, D // 128, 2 * F, 4), dtype=torch.uint8, device=gpu, generator=g)
    x_q, x_e = K.quantize_rows_mxfp4(torch.randn((rows, D), device=gpu, generator=g))
    counts = torch.zeros(N, dtype=torch.int64)
    counts[5], counts[600], counts[1022], counts[1023] = 20, 10, 7, 3
    off = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)]).to(gpu, torch.int32)
    h_q, h_e = K.grouped_gate_up_mxfp4(x_q, x_e, off, w_q, w_e)
    for e in (600, 1022, 1023):
        lo, hi = int(off[e]), int(off[e + 1])
        one = torch.tensor([0, hi - lo], dtype=torch.int32, device=gpu)
        q, x = K.grouped_gate_up_mxfp4(x_q[lo:hi].contiguous(), x_e[lo:hi].contiguous(), one, w_q[e:e + 1], w_e[e:e + 1])
        assert torch.equal(h_q[lo:hi], q) and torch.equal(h_e[lo:hi], x), e
    back = K.unpack_mxfp4(w_q, w_e)
    assert torch.equal(back[-1], K.unpack_mxfp4(w_q[-1:], w_e[-1:])[0])

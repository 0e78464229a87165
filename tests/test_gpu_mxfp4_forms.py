"""The MXFP4 products in the forms that carry large calls: each test says which form its
sizes take, and asserts it.  Forms 0 (32 rows a wave, from memory), 2 and 3 (tiles of 64 and
128 rows through LDS) sum in the same order, so that pieces of a few rows give the tiles'
bits; form 1 adds four parts and is held to float64."""
import numpy as np
import pytest
import torch

import mxfp4_reference as R
from hanuman_amd import _lib, kernels as K
from test_gpu_mxfp4 import _case, _check_down, _check_gate_up

pytestmark = pytest.mark.gpu

TILES = [2, 3]
PIECE = 96


def _form(gpu, rows, experts, kdim, ncols):
    cus = torch.cuda.get_device_properties(gpu).multi_processor_count // 8 * 8
    return _lib.lib().hmoe_grouped_mxfp4_form(rows, experts, kdim, ncols, cus)


def _randn(gpu, seed, *shape):
    return torch.randn(shape, generator=torch.Generator(device=gpu).manual_seed(seed), device=gpu)


def _gate_up_operand(gpu, experts, d_model, d_ff):
    return K.pack_mxfp4_gate_up(*(_randn(gpu, 70 + i, experts, d_model, d_ff) * 0.05 for i in range(2)))


def _down_operand(gpu, experts, d_ff, d_model):
    return K.pack_mxfp4_down(_randn(gpu, 80, experts, d_ff, d_model) * 0.05)


def _in_pieces(gpu, product, q, exps, offsets, packed, packed_exp):
    """The product of every segment, a few rows of one expert a call, on form 0."""
    off = offsets.tolist()
    kdim, ncols = q.shape[1] * 2, packed.shape[1] * 32
    assert _form(gpu, PIECE, 1, kdim, ncols) == 0
    outs = []
    for e, (lo, hi) in enumerate(zip(off, off[1:])):
        for r in range(lo, hi, PIECE):
            n = min(PIECE, hi - r)
            one = torch.tensor([0, n], dtype=torch.int32, device=gpu)
            out = product(q[r:r + n].clone(), exps[r:r + n].clone(), one, packed[e:e + 1], packed_exp[e:e + 1])
            outs.append(out if isinstance(out, tuple) else (out,))
    return [torch.cat(t) for t in zip(*outs)]


def _raw_gate_up(x_q, x_e, offsets, gu, h_q, h_e):
    N, D, F = gu[0].shape[0], gu[0].shape[2] * 64, gu[0].shape[1] * 16
    _lib.call("hmoe_grouped_gate_up_mxfp4", x_q.data_ptr(), x_e.data_ptr(), offsets.data_ptr(), N, h_q.shape[0], D, F,
              gu[0].data_ptr(), gu[1].data_ptr(), h_q.data_ptr(), h_e.data_ptr(),
              torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("rows,experts,d_model,d_ff,gate_up,down", [
    (12000, 3, 256, 1152, 2, 2),      # gate/up: one step of 256 a tile
    (12000, 3, 128, 1152, 2, 2),      # half a step
    (60000, 3, 256, 1152, 3, 3),
    (60000, 3, 128, 1152, 3, 3),
    (12000, 3, 2048, 256, 3, 2),      # down: one step
    (60000, 3, 2048, 256, 3, 3),
    (60000, 3, 2048, 128, 3, 3),      # half a step
], ids=lambda v: str(v))
def test_tiles_back_to_back(gpu, rows, experts, d_model, d_ff, gate_up, down):
    """Tiles of a step or less, many a workgroup: what a tile puts into LDS for its rows'
    ends follows the last tile's at once.  Against pieces of few rows, bit for bit."""
    assert _form(gpu, rows, experts, d_model, 2 * d_ff) == gate_up
    assert _form(gpu, rows, experts, d_ff, d_model) == down
    off = torch.tensor([0, rows // 3 + 5, rows // 3 + 5 + rows // 2, rows], dtype=torch.int32, device=gpu)
    if d_model <= 256:
        x_q, x_e = K.quantize_rows_mxfp4(_randn(gpu, 1, rows, d_model))
        gu = _gate_up_operand(gpu, experts, d_model, d_ff)
        want = _in_pieces(gpu, K.grouped_gate_up_mxfp4, x_q, x_e, off, *gu)
        for _ in range(3):
            got = K.grouped_gate_up_mxfp4(x_q, x_e, off, *gu)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    else:
        h_q, h_e = K.quantize_rows_mxfp4(_randn(gpu, 2, rows, d_ff))
        dn = _down_operand(gpu, experts, d_ff, d_model)
        want, = _in_pieces(gpu, K.grouped_down_mxfp4, h_q, h_e, off, *dn)
        for _ in range(3):
            assert torch.equal(K.grouped_down_mxfp4(h_q, h_e, off, *dn), want)


# ------------------------------------------------------- against float64 --

def _float64(gpu, shape, seed, **kw):
    """A layer's gathered gate/up and down products against float64, the gathered rows
    against rows in the experts' order, and the plan."""
    tokens, experts, active, d_model, d_ff = shape
    x, plan, (gu_w, dn_w), (gu, dn) = _case(*shape, seed=seed, gpu=gpu, **kw)
    x_q, x_e = K.quantize_rows_mxfp4(x.to(gpu))
    h_q, h_e = K.grouped_gate_up_mxfp4_gather(x_q, x_e, plan, *gu)
    _check_gate_up(h_q, h_e, R.values(x_q.cpu().numpy(), x_e.cpu().numpy()), plan, gu_w, d_ff, active)
    kept = int(plan.offsets[-1])
    src = (plan.perm_src.long() // active).clamp(min=0)
    g_q, g_e = K.grouped_gate_up_mxfp4(x_q[src], x_e[src], plan.offsets, *gu)
    assert torch.equal(g_q[:kept], h_q[:kept]) and torch.equal(g_e[:kept], h_e[:kept])
    ys = K.grouped_down_mxfp4(h_q, h_e, plan.offsets, *dn)
    _check_down(ys, R.values(h_q[:kept].cpu().numpy(), h_e[:kept].cpu().numpy()), plan.offsets.cpu().numpy(), dn_w)
    return plan


@pytest.mark.parametrize("shape,gate_up,down", [
    ((12000, 3, 2, 640, 640), 3, 2),        # gathered, several experts, 128 rows a tile
    ((14000, 12, 2, 640, 640), 2, 3),
    ((3000, 70, 4, 384, 640), 2, 2),        # more experts than a wave has lanes
    ((20000, 70, 2, 640, 640), 3, 2),
    ((6000, 70, 2, 640, 256), 2, 2),
    ((40, 4, 2, 2048, 2048), 1, 1),         # four groups of a wave's reduction at a time
    ((9, 3, 2, 2176, 4224), 1, 1),          # and five, and nine
], ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else str(v))
def test_many_experts(gpu, shape, gate_up, down):
    tokens, experts, active, d_model, d_ff = shape
    assert _form(gpu, tokens * active, experts, d_model, 2 * d_ff) == gate_up
    assert _form(gpu, tokens * active, experts, d_ff, d_model) == down
    _float64(gpu, shape, seed=sum(shape))


@pytest.mark.parametrize("shape,skew,gate_up,down", [
    ((9000, 9, 1, 640, 640), 4.0, 2, 2),
    ((12000, 6, 1, 640, 640), 4.0, 3, 2),
    ((20000, 6, 1, 640, 640), 4.0, 2, 3),
    ((12000, 12, 1, 640, 1152), 2.0, 2, 2),
], ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else str(v))
def test_skewed_experts(gpu, shape, skew, gate_up, down):
    """Nearly all rows on the first experts, the last ones empty, segments of a few rows
    between."""
    tokens, experts, active, d_model, d_ff = shape
    assert _form(gpu, tokens * active, experts, d_model, 2 * d_ff) == gate_up
    assert _form(gpu, tokens * active, experts, d_ff, d_model) == down
    plan = _float64(gpu, shape, seed=5, skew=skew)
    counts = plan.counts.tolist()
    assert 0 in counts and any(0 < c < 64 for c in counts)


@pytest.mark.parametrize("where", ["first", "middle", "last"])
@pytest.mark.parametrize("form", TILES)
def test_experts_without_rows(gpu, form, where):
    """66 experts, rows on three only, the others empty before, between and after them."""
    rows, D, F = {2: 9000, 3: 60000}[form], 256, 1152
    N = 66
    assert _form(gpu, rows, N, D, 2 * F) == form
    live = {"first": (0, 1, 2), "middle": (0, 63, 65), "last": (63, 64, 65)}[where]
    counts = torch.zeros(N, dtype=torch.int64)
    for e, c in zip(live, (rows - 3001, 3000, 1)):
        counts[e] = c
    off = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)]).to(gpu, torch.int32)
    x_q, x_e = K.quantize_rows_mxfp4(_randn(gpu, 1, rows, D))
    gu = _gate_up_operand(gpu, N, D, F)
    got = K.grouped_gate_up_mxfp4(x_q, x_e, off, *gu)
    want = _in_pieces(gpu, K.grouped_gate_up_mxfp4, x_q, x_e, off, *gu)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ---------------------------------------------------- what rows may be like --

ROWS = {2: 12000, 3: 30000}     # of 4 experts: reductions of 384, 1152 columns of h or ys


def _edge_sizes(gpu, form):
    """Rows, experts and the sizes (D, F) whose gate/up and (F, D) whose down take `form`."""
    rows, N, K_, cols = ROWS[form], 4, 384, 1152
    assert _form(gpu, rows, N, K_, 2 * cols) == form and _form(gpu, rows, N, K_, cols) == form
    return rows, N, K_, cols


@pytest.mark.parametrize("form", TILES)
def test_rows_past_the_segments_stay(gpu, form):
    """Buffers with more rows than the segments, which end inside tiles: the others are left
    as they were."""
    rows, N, K_, cols = _edge_sizes(gpu, form)
    kept = rows - 777
    off = torch.tensor([0, 1, 1, kept // 2 + 7, kept], dtype=torch.int32, device=gpu)
    q, e = K.quantize_rows_mxfp4(_randn(gpu, 1, rows, K_))
    gu, dn = _gate_up_operand(gpu, N, K_, cols), _down_operand(gpu, N, K_, cols)
    h_q = torch.full((rows, cols // 2), 0xA5, dtype=torch.uint8, device=gpu)
    h_e = torch.full((rows, cols // 32), 0xA5, dtype=torch.uint8, device=gpu)
    _raw_gate_up(q, e, off, gu, h_q, h_e)
    want = _in_pieces(gpu, K.grouped_gate_up_mxfp4, q, e, off, *gu)
    assert torch.equal(h_q[:kept], want[0]) and torch.equal(h_e[:kept], want[1])
    assert (h_q[kept:] == 0xA5).all() and (h_e[kept:] == 0xA5).all()
    ys = torch.full((rows, cols), 7.0, dtype=torch.bfloat16, device=gpu)
    _lib.call("hmoe_grouped_down_mxfp4", q.data_ptr(), e.data_ptr(), off.data_ptr(), N, rows, K_, cols,
              dn[0].data_ptr(), dn[1].data_ptr(), ys.data_ptr(), torch.cuda.current_stream().cuda_stream)
    want, = _in_pieces(gpu, K.grouped_down_mxfp4, q, e, off, *dn)
    assert torch.equal(ys[:kept], want) and (ys[kept:] == 7.0).all()


@pytest.mark.parametrize("start", [1, 3, 4])
@pytest.mark.parametrize("form", TILES)
def test_rows_inside_a_buffer(gpu, form, start):
    """Rows that start at a later row of their buffers: codes at 16 bytes, exponents at words
    only.  The rows before and behind hold NaN, which no result may show."""
    rows, N, K_, cols = _edge_sizes(gpu, form)
    off = torch.tensor([0, 5000, 5001, rows - 64, rows], dtype=torch.int32, device=gpu)
    q, e = K.quantize_rows_mxfp4(_randn(gpu, 3, rows + start + 2, K_))
    e[:start] = 255
    e[start + rows:] = 255
    a_q, a_e = q[start:start + rows], e[start:start + rows]
    assert a_e.data_ptr() % 16 == start * 12 % 16 and a_q.data_ptr() % 16 == 0
    gu, dn = _gate_up_operand(gpu, N, K_, cols), _down_operand(gpu, N, K_, cols)
    got = K.grouped_gate_up_mxfp4(a_q, a_e, off, *gu)
    want = _in_pieces(gpu, K.grouped_gate_up_mxfp4, a_q, a_e, off, *gu)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and (got[1] < 255).all()
    ys = K.grouped_down_mxfp4(a_q, a_e, off, *dn)
    assert torch.equal(ys, _in_pieces(gpu, K.grouped_down_mxfp4, a_q, a_e, off, *dn)[0]) and ys.isfinite().all()
    # gathered from tokens that start there
    src = torch.randperm(rows, generator=torch.Generator().manual_seed(1)).to(gpu, torch.int32)
    plan = K.Plan(off.diff(), off, src.clone(), src, torch.ones(rows, dtype=torch.uint8, device=gpu), rows, rows, N, 1)
    got = K.grouped_gate_up_mxfp4_gather(a_q, a_e, plan, *gu)
    want = K.grouped_gate_up_mxfp4(a_q[src.long()], a_e[src.long()], off, *gu)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("form", TILES)
def test_dropped_slots(gpu, form):
    """A capacity that drops slots, so that the segments end before the rows do."""
    rows, N, K_, cols = _edge_sizes(gpu, form)
    tokens = rows // 2
    gen = torch.Generator(device=gpu).manual_seed(6)
    logits = torch.randn((tokens, N), generator=gen, device=gpu) - 1.5 * torch.arange(N, device=gpu)
    top = logits.topk(2, dim=1).indices.int()
    plan = K.dispatch_plan(top, N, rows // 3)
    kept = int(plan.offsets[-1])
    assert kept < plan.rows_cap and _form(gpu, plan.rows_cap, N, K_, 2 * cols) == form
    x_q, x_e = K.quantize_rows_mxfp4(_randn(gpu, 4, tokens, K_))
    gu = _gate_up_operand(gpu, N, K_, cols)
    h_q = torch.full((plan.rows_cap, cols // 2), 0xA5, dtype=torch.uint8, device=gpu)
    h_e = torch.full((plan.rows_cap, cols // 32), 0xA5, dtype=torch.uint8, device=gpu)
    _lib.call("hmoe_grouped_gate_up_mxfp4_gather", x_q.data_ptr(), x_e.data_ptr(), tokens, 2, plan.perm_src.data_ptr(),
              plan.offsets.data_ptr(), N, plan.rows_cap, K_, cols, gu[0].data_ptr(), gu[1].data_ptr(), h_q.data_ptr(),
              h_e.data_ptr(), torch.cuda.current_stream().cuda_stream)
    src = plan.perm_src[:kept].long() // 2
    want = _in_pieces(gpu, K.grouped_gate_up_mxfp4, x_q[src], x_e[src], plan.offsets, *gu)
    assert torch.equal(h_q[:kept], want[0]) and torch.equal(h_e[:kept], want[1])
    assert (h_q[kept:] == 0xA5).all() and (h_e[kept:] == 0xA5).all()


@pytest.mark.parametrize("form", TILES)
def test_nan_tokens(gpu, form):
    """Tokens with a value that is not finite: their rows are NaN through both products, all
    others as if they had been zeros."""
    rows, N, K_, cols = _edge_sizes(gpu, form)
    tokens = rows // 2
    assert _form(gpu, rows, N, cols, K_) == form
    x = _randn(gpu, 7, tokens, K_)
    zeros = x.clone()
    for t, c, v in ((3, 100, float("nan")), (17, 0, float("inf")), (tokens // 2, 383, float("-inf")), (tokens - 1, 31, float("nan"))):
        x[t, c] = v
        zeros[t] = 0
    top = _randn(gpu, 8, tokens, N).topk(2, dim=1).indices.int()
    plan = K.dispatch_plan(top, N, rows)
    gu, dn = _gate_up_operand(gpu, N, K_, cols), _down_operand(gpu, N, cols, K_)

    def run(v):
        h = K.grouped_gate_up_mxfp4_gather(*K.quantize_rows_mxfp4(v), plan, *gu)
        return (*h, K.grouped_down_mxfp4(*h, plan.offsets, *dn))

    (h_q, h_e, ys), (z_q, z_e, zs) = run(x), run(zeros)
    bad = ~x.isfinite().all(1)[plan.perm_src.long() // 2]
    assert int(bad.sum()) == 8
    assert (h_e[bad] == 255).all() and (h_q[bad] == 0).all() and ys[bad].isnan().all()
    assert torch.equal(h_q[~bad], z_q[~bad]) and torch.equal(h_e[~bad], z_e[~bad]) and torch.equal(ys[~bad], zs[~bad])
    assert ys[~bad].isfinite().all()


def test_offsets_of_a_subclass(gpu):
    """Index arrays that a module holds as parameters."""
    off = torch.tensor([0, 5, 9], dtype=torch.int32, device=gpu)
    q, e = K.quantize_rows_mxfp4(_randn(gpu, 1, 9, 256))
    dn = _down_operand(gpu, 2, 256, 128)
    held = torch.nn.Parameter(off, requires_grad=False)
    assert torch.equal(K.grouped_down_mxfp4(q, e, held, *dn), K.grouped_down_mxfp4(q, e, off, *dn))
    with pytest.raises(ValueError, match=r"offsets must be int32 \[3\]"):
        K.grouped_down_mxfp4(q, e, torch.nn.Parameter(off[:2].clone(), requires_grad=False), *dn)


# ----------------------------------------------------- the ends of the SwiGLU --

def _ones(gpu, rows, d_model):
    """Rows of ones."""
    return (torch.full((rows, d_model // 2), 0x22, dtype=torch.uint8, device=gpu),
            torch.full((rows, d_model // 32), 127, dtype=torch.uint8, device=gpu))


def _sums_operand(gpu, gate, gate_exp, up, up_exp):
    """The operand of one expert with given codes [F, D] and exponents [F] of its columns."""
    F, D = gate.shape
    codes, exps = np.empty((2 * F, D), dtype=np.uint8), np.empty((2 * F, D // 32), dtype=np.uint8)
    for p in range(2 * F):
        which, c = R.gate_up_column(p, F)
        codes[p], exps[p] = ((up[c], up_exp[c]) if which else (gate[c], gate_exp[c]))
    return [torch.from_numpy(t[None]).to(gpu) for t in R.packed_operand(codes[:, 0::2] | (codes[:, 1::2] << 4), exps)]


@pytest.mark.parametrize("rows,form", [(40, 0), (9000, 2), (60000, 3)])
def test_far_negative_gates(gpu, rows, form):
    """Gates from -60 to -90 with large up values.  Both sums are exact (at most 1536 halves of
    a power of two), so that h is off by the SwiGLU's own roundings alone: the argument of the
    exponential by half a step of |g| log2(e) and by log2(e)'s rounding, 1.25 |g| 2^-24 of h;
    exponential and reciprocal by a step, the sum and two products by half a step, 7 of them,
    and one for the products of these errors.  Where 1 + e^-g passes 2^126 its reciprocal may
    be zero: |g u| 2^-126."""
    D, F = 128, 2048
    assert _form(gpu, rows, 1, D, 2 * F) == form
    rng = np.random.default_rng(3)
    t = np.concatenate([np.arange(60, 90.25, 0.5), [88.5, 87.0, 87.5]]).repeat(32)      # -g of each column
    gate = np.zeros((F, D), dtype=np.uint8)
    for c in range(F):
        ones = int(t[c])
        gate[c, :ones] = 0xA                                                            # -1
        gate[c, ones:ones + int(2 * (t[c] - ones))] = 0x9                               # -1 / 2
    up, up_exp = rng.integers(0, 16, (F, D), dtype=np.uint8), np.where(t < 87, 207, 227).astype(np.uint8)
    gu = _sums_operand(gpu, gate, np.full(F, 127, dtype=np.uint8), up, up_exp)
    h_q, h_e = K.grouped_gate_up_mxfp4(*_ones(gpu, rows, D), torch.tensor([0, rows], dtype=torch.int32, device=gpu), *gu)
    assert (h_q == h_q[:1]).all() and (h_e == h_e[:1]).all()
    u = np.where(up >= 8, -1.0, 1.0) * R.SIZES[up & 7] * np.ldexp(1.0, up_exp.astype(int) - 127)[:, None]
    g, u = -t[None], u.sum(1)[None]
    h = g / (1.0 + np.exp(-g)) * u
    bound = np.abs(h) * (1.25 * np.abs(g) + 8) * 2.0**-24 + np.where(t > 126 * np.log(2), np.abs(g * u) * 2.0**-126, 0.0)
    R.check_quantised(h_q[:1].cpu().numpy(), h_e[:1].cpu().numpy(), h, bound)
    assert (h_e[0, :54] > 0).all()      # (down to -86.5 h is not lost)


@pytest.mark.parametrize("rows,form", [(40, 0), (9000, 2), (60000, 3)])
def test_sums_past_float32(gpu, rows, form):
    """Gate sums of both signs and up sums past float32's range: NaN in their blocks alone."""
    D, F = 128, 2048
    assert _form(gpu, rows, 1, D, 2 * F) == form
    gate, up = np.full((F, D), 0x1, dtype=np.uint8), np.full((F, D), 0x2, dtype=np.uint8)
    gate_exp, up_exp = np.full(F, 123, dtype=np.uint8), np.full(F, 127, dtype=np.uint8)     # g = 4, u = 128
    gate[64 + 5], gate_exp[64 + 5] = 0x7, 254
    gate[992 + 31], gate_exp[992 + 31] = 0xF, 254
    up[2016], up_exp[2016] = 0x7, 254
    gu = _sums_operand(gpu, gate, gate_exp, up, up_exp)
    h_q, h_e = K.grouped_gate_up_mxfp4(*_ones(gpu, rows, D), torch.tensor([0, rows], dtype=torch.int32, device=gpu), *gu)
    nan = torch.zeros(F // 32, dtype=torch.bool, device=gpu)
    nan[[2, 31, 63]] = True
    assert (h_e[:, nan] == 255).all() and (h_q.reshape(rows, -1, 16)[:, nan] == 0).all()
    # 4 / (1 + e^-4) * 128 = 502.8: a scale of 2^7, of which it is 3.93, code 6 (4)
    assert (h_e[:, ~nan] == 127 + 7).all() and (h_q.reshape(rows, -1, 16)[:, ~nan] == 0x66).all()

"""int8 rows, operands and products on the GPU against exact integer sums."""
import numpy as np
import pytest
import torch

import i8_reference as R
from hanuman_amd import _lib, kernels as K

pytestmark = pytest.mark.gpu


def _to(a, dev):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


# ------------------------------------------------------------ rows and back --

def _rows(kind, rng):
    if kind == "normal":
        return rng.standard_normal((37, 96))
    if kind == "one":
        return rng.standard_normal((1, 8))
    if kind == "wide":      # rows over float32's range
        return rng.standard_normal((300, 1056)) * np.exp2(rng.integers(-140, 125, (300, 1)))
    if kind == "ties":      # halves of a code at power-of-two scales: 127 units the largest
        v = rng.integers(-253, 254, (120, 64)) * 0.5
        v[:, 7] = 127.0
        return v * np.exp2(rng.integers(-60, 60, (120, 1)))
    if kind == "small":     # subnormals, zeros of both signs
        v = rng.integers(-9, 10, (40, 64)) * 2.0**-149 * np.exp2(rng.integers(0, 26, (40, 1)))
        v[3] = 0.0
        v[4] = -0.0
        return v
    if kind == "long":
        return rng.standard_normal((3, 32768))
    v = rng.standard_normal((12, 96))   # "special"
    v[0, 3] = np.inf
    v[1, 40] = -np.inf
    v[2, 95] = np.nan
    v[3, 31] = np.nan
    v[3, 0] = np.inf
    v[5, 0] = np.finfo(np.float32).max
    return v


@pytest.mark.parametrize("kind", ["normal", "one", "wide", "ties", "small", "long", "special"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("repeat", [1, 300])
def test_quantised_rows(gpu, kind, dtype, repeat):
    """(`repeat`: rows enough for a wave to take one each.)"""
    if repeat > 1 and kind == "long":
        pytest.skip("the long rows are a workgroup's either way")
    with np.errstate(over="ignore"):
        v = torch.from_numpy(_rows(kind, np.random.default_rng(5)).astype(np.float32)).to(dtype).repeat(repeat, 1)
    q, s = K.quantize_rows_i8(v.to(gpu))
    want_q, want_s = R.quantise(v.float().numpy())
    assert np.array_equal(s.cpu().numpy(), want_s, equal_nan=True)
    assert np.array_equal(q.cpu().numpy(), want_q)
    for out in (torch.float32, torch.bfloat16):
        back = K.dequantize_rows_i8(q, s, out).cpu()
        with np.errstate(all="ignore"):
            want = torch.from_numpy(want_q.astype(np.float32) * want_s[:, None]).to(out)
        assert torch.equal(torch.nan_to_num(back, 7e30), torch.nan_to_num(want, 7e30))
        assert torch.equal(torch.isnan(back), torch.isnan(want))


def test_codes_of_bf16_rows_are_the_nearest(gpu):
    """Every bf16 mantissa against every largest mantissa, over ten octaves: the codes are the
    nearest to the exact quotient (where that is a half, as for half the largest value, both
    neighbours are)."""
    rows = []
    for b in range(128, 256):
        v = np.concatenate([np.arange(128, 256) * 2.0**-k for k in range(0, 10)])
        rows.append(np.concatenate([np.where(v <= b, v, 0.0), [b] * 8]))
    v = np.array(rows)
    q = K.quantize_rows_i8(torch.from_numpy(v).to(torch.bfloat16).to(gpu))[0].cpu().numpy().astype(np.float64)
    largest = v.max(1, keepdims=True)
    # |q - 127 v / largest| <= 1 / 2, in integers that 64 bits hold
    assert (np.abs(q * largest - 127 * v) * 2 <= largest).all()


def test_rows_past_the_segments(gpu):
    a = torch.randn((50, 64), device=gpu).bfloat16()
    off = torch.tensor([0, 11, 31], dtype=torch.int32, device=gpu)
    q, s = K.quantize_rows_i8(a, off)
    want_q, want_s = K.quantize_rows_i8(a)
    assert torch.equal(q[:31], want_q[:31]) and torch.equal(s[:31], want_s[:31]) and (s[31:] == 1.0).all()
    guard = torch.full((50, 64), 77, dtype=torch.int8, device=gpu)
    _lib.call("hmoe_quantize_rows_i8", a.data_ptr(), _lib.BF16, 50, 64, off.data_ptr(), 2, guard.data_ptr(), s.data_ptr(),
              torch.cuda.current_stream().cuda_stream)
    assert torch.equal(guard[:31], want_q[:31]) and (guard[31:] == 77).all()


def test_e4m3_rows_read_back(gpu):
    codes = torch.arange(256, dtype=torch.uint8).repeat(3, 1)
    scale = torch.tensor([1.0, 0.37, 2.0**-130])
    back = K.dequantize_rows_fp8(codes.to(gpu), scale.to(gpu), torch.float32).cpu()
    want = codes.view(torch.float8_e4m3fn).float() * scale.unsqueeze(1)
    assert torch.equal(torch.nan_to_num(back, 7e30), torch.nan_to_num(want, 7e30))
    assert torch.equal(torch.isnan(back), torch.isnan(want))


# ----------------------------------------------------------------- operands --

@pytest.mark.parametrize("N,D,F", [(1, 128, 128), (3, 384, 128), (2, 128, 640), (5, 640, 256)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_packed_operands(gpu, N, D, F, dtype):
    rng = np.random.default_rng(N * D + F)
    wg, wu, wd = (torch.from_numpy((rng.standard_normal(s) * np.exp2(rng.integers(-9, 9, s))).astype(np.float32)).to(dtype)
                  for s in ((N, D, F), (N, D, F), (N, F, D)))
    wd[0, 3, 1] = float("inf")
    wg[0, :, 5] = 0.0
    gu, gu_s = (t.cpu().numpy() for t in K.pack_i8_gate_up(wg.to(gpu), wu.to(gpu)))
    dn, dn_s = (t.cpu().numpy() for t in K.pack_i8_down(wd.to(gpu)))
    for n in range(N):
        g, u, d = (w[n].float().numpy().T for w in (wg, wu, wd))
        q, s = R.quantise(R.gate_up_rows(g, u))
        assert np.array_equal(gu[n], R.operand(q)) and np.array_equal(gu_s[n], s)
        q, s = R.quantise(d)
        assert np.array_equal(dn[n], R.operand(q)) and np.array_equal(dn_s[n], s)


# ----------------------------------------------------------------- products --

def _weights(rng, N, rows, k):
    q = rng.integers(-128, 128, (N, rows, k)).astype(np.int8)        # (a user's own codes may be -128)
    s = (rng.random((N, rows)) * 1e-3 + 1e-5).astype(np.float32)
    return q, s


def _segments(kind, N, rng):
    if kind == "one":
        return [1]
    if kind == "few":
        return [int(c) for c in rng.integers(0, 5, N)]
    if kind == "mid":
        return [int(c) for c in rng.integers(0, 130, N)]
    if kind == "many":
        return [int(c) for c in rng.integers(200, 700, N)]
    if kind == "crowd":     # (sums that the larger tiles are taken for)
        counts = rng.multinomial(9000, rng.dirichlet([2.0] * N))
        counts[0] = 0
        return [int(c) for c in counts]
    counts = [0] * N                # "skewed", "lopsided": most rows with one expert, several without any
    counts[N // 2], counts[-1] = 14001 if kind == "lopsided" else 1000, 3
    return counts


CASES = [("one", 1, 128, 128), ("one", 1, 2048, 256), ("few", 7, 256, 128), ("few", 9, 1152, 384), ("mid", 6, 384, 640),
         ("mid", 5, 1280, 256), ("many", 3, 256, 384), ("many", 4, 1152, 640), ("many", 8, 128, 128),
         ("skewed", 6, 512, 256), ("skewed", 70, 128, 128), ("mid", 130, 256, 128), ("one", 1, 4096, 4096),
         ("crowd", 8, 1280, 1152), ("crowd", 40, 1152, 640), ("lopsided", 4, 896, 896), ("lopsided", 6, 128, 640)]


@pytest.fixture(scope="module")
def forms_seen():
    return set()


@pytest.mark.parametrize("kind,N,D,F", CASES)
@pytest.mark.parametrize("gather", [False, True], ids=["rows", "gather"])
def test_products(gpu, kind, N, D, F, gather, forms_seen):
    rng = np.random.default_rng(N * 1000 + D + F)
    counts = _segments(kind, N, rng)
    kept = sum(counts)
    cap = kept + 5                                   # rows past the segments are left alone
    off = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    top_k = 3
    T = -(-cap // top_k)
    x_q = rng.integers(-127, 128, (T if gather else cap, D)).astype(np.int8)
    x_s = (rng.random(len(x_q)) * 0.1 + 1e-3).astype(np.float32)
    if kept > 2:
        x_s[1] = np.nan
    src = rng.permutation(T * top_k)[:cap].astype(np.int32)
    src[kept:] = -1
    gu, gu_s = _weights(rng, N, 2 * F, D)
    dn, dn_s = _weights(rng, N, D, F)
    pg = _to(np.stack([R.operand(gu[e]) for e in range(N)]), gpu), _to(gu_s, gpu)
    pd = _to(np.stack([R.operand(dn[e]) for e in range(N)]), gpu), _to(dn_s, gpu)
    offs = _to(off, gpu)
    cus = torch.cuda.get_device_properties(gpu).multi_processor_count
    for k, ncols in ((D, 2 * F), (F, D)):
        forms_seen.add(_lib.lib().hmoe_grouped_i8_form(cap, N, k, ncols, cus))
    h = torch.full((cap, F), 7.0, dtype=torch.bfloat16, device=gpu)
    xq, xs, perm = _to(x_q, gpu), _to(x_s, gpu), _to(src, gpu)
    st = torch.cuda.current_stream().cuda_stream
    if gather:
        _lib.call("hmoe_grouped_gate_up_i8_gather", xq.data_ptr(), xs.data_ptr(), T, top_k, perm.data_ptr(),
                  offs.data_ptr(), N, cap, D, F, pg[0].data_ptr(), pg[1].data_ptr(), h.data_ptr(), st)
    else:
        _lib.call("hmoe_grouped_gate_up_i8", xq.data_ptr(), xs.data_ptr(), offs.data_ptr(), N, cap, D, F,
                  pg[0].data_ptr(), pg[1].data_ptr(), h.data_ptr(), st)
    assert (h[kept:] == 7.0).all()
    got = h.float().cpu().numpy()
    row = src // top_k if gather else np.arange(cap)
    for e in range(N):
        lo, hi = off[e], off[e + 1]
        if lo == hi:
            continue
        y = R.product(x_q[row[lo:hi]], x_s[row[lo:hi]], gu[e], gu_s[e]).reshape(hi - lo, -1, 2, 32)
        want, bound = R.swiglu_with_bound(y[:, :, 0].reshape(hi - lo, F), y[:, :, 1].reshape(hi - lo, F))
        nan = np.isnan(want)
        assert np.array_equal(np.isnan(got[lo:hi]), nan)
        d = np.abs(got[lo:hi] - want)[~nan]
        assert (d <= (bound + (np.abs(want) + bound) * 2.0**-8 + 2.0**-134)[~nan]).all(), (e, d.max())
    # the down product, of h's codes: the same bits as float32 operations on the exact sums
    hq, hs = K.quantize_rows_i8(h, offs)
    ys = torch.full((cap, D), 7.0, dtype=torch.bfloat16, device=gpu)
    _lib.call("hmoe_grouped_down_i8", hq.data_ptr(), hs.data_ptr(), offs.data_ptr(), N, cap, F, D, pd[0].data_ptr(),
              pd[1].data_ptr(), ys.data_ptr(), st)
    assert (ys[kept:] == 7.0).all()
    got = ys.float().cpu().numpy()
    hq, hs = hq.cpu().numpy(), hs.cpu().numpy()
    for e in range(N):
        lo, hi = off[e], off[e + 1]
        if lo < hi:
            want = R.bf16(R.product(hq[lo:hi], hs[lo:hi], dn[e], dn_s[e]))
            assert np.array_equal(got[lo:hi], want, equal_nan=True), e


def test_every_form_is_tested(gpu, forms_seen):
    assert forms_seen == {0, 1, 2, 3}


def test_largest_sums(gpu):
    """Codes of -128 throughout the longest reduction: sums of 2^29."""
    k = 32768
    w = torch.full((1, 128 // 32, k // 32, 64, 16), -128, dtype=torch.int8, device=gpu)
    one = torch.ones((1, 128), device=gpu)
    for rows in (3, 700):
        a = torch.full((rows, k), -128, dtype=torch.int8, device=gpu)
        off = K.one_group_offsets(rows, gpu)
        ys = K.grouped_down_i8(a, torch.full((rows,), 2.0**-20, device=gpu), off, w, one)
        assert (ys == 512.0).all()

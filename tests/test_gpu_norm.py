"""The root-mean-square norm with the residual's addition, its 8-bit codes and its gradients
on the GPU against float64."""
import numpy as np
import pytest
import torch

from hanuman_amd import _lib, kernels as K

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
HALF_STEP = {F32: 2.0**-24, BF16: 2.0**-8}
EPS = 1e-5


def _rows(gpu, rows, cols, dtype, seed, scale=1.0):
    g = torch.Generator(device=gpu).manual_seed(seed)
    v = torch.randn((rows, cols), generator=g, device=gpu) * torch.exp(torch.randn((rows, 1), generator=g, device=gpu))
    return (v * scale).to(dtype)


def _terms(cols):
    """float32 roundings that a row's sum may add up: a thread's values one after another (32
    columns at most), the wave's six, the workgroup's sixteen, the quotient."""
    return 32 + 6 + 16 + 1


SIZES = [(1, 8), (3, 24), (5, 256), (2, 1032), (7, 2048), (4, 2056), (3, 4104), (2, 8200), (2, 32768), (2050, 40),
         (2049, 1024), (2048, 2048), (2055, 1056), (2053, 3000), (9000, 64)]


@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("x_type,r_type,y_type", [(BF16, BF16, BF16), (F32, F32, F32), (BF16, None, BF16),
                                                  (F32, None, BF16), (F32, BF16, BF16), (BF16, F32, F32)])
@pytest.mark.parametrize("quant", ["int8", "e4m3"])
def test_norm(gpu, rows, cols, x_type, r_type, y_type, quant):
    x = _rows(gpu, rows, cols, x_type, rows + cols)
    r = None if r_type is None else _rows(gpu, rows, cols, r_type, rows + cols + 1)
    w_type = F32 if cols % 16 else BF16
    w = (1.0 + 0.2 * torch.randn(cols, generator=torch.Generator(device=gpu).manual_seed(3), device=gpu)).to(w_type)
    out = K.add_rms_norm(x, w, r, EPS, out_dtype=y_type, quant=quant)
    if r is None:
        assert out.sum is x
    else:
        assert torch.equal(out.sum, (x.float() + r.float()).to(r_type))
    s = out.sum.double()
    rstd = (s.square().mean(1) + EPS).rsqrt()
    # the sum's roundings count half under the root; the mean, eps, root and reciprocal once
    off = (0.5 * (_terms(cols) + 2) + 2) * 2.0**-24
    assert ((out.rstd.double() - rstd).abs() <= off * rstd).all()
    y = s * rstd.unsqueeze(1) * w.double()
    assert out.y.dtype == y_type
    assert ((out.y.double() - y).abs() <= (off + 2 * 2.0**-24 + HALF_STEP[y_type] * 1.01) * y.abs() + 1e-40).all()
    # the codes are those of the rounded y
    if quant == "int8":
        q, scale = K.quantize_rows_i8(out.y)
        assert out.q.dtype == torch.int8
    elif y_type == BF16:
        q, scale = K.quantize_rows_fp8(out.y)
    else:
        amax = out.y.abs().amax(1)
        # (in 64 bits: torch divides by a number by multiplying with its reciprocal)
        scale = (amax.double() / 448.0).float()
        inv = (torch.full_like(amax, 448.0).double() / amax.double()).float()
        q = (out.y * inv.unsqueeze(1)).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    assert torch.equal(out.q, q) and torch.equal(out.scale, scale)
    plain = K.add_rms_norm(x, w, r, EPS, out_dtype=y_type)
    assert plain.q is None and plain.scale is None
    assert torch.equal(plain.y, out.y) and torch.equal(plain.sum, out.sum) and torch.equal(plain.rstd, out.rstd)


def test_rows_that_are_not_ordinary(gpu):
    """Rows of zeros, of one value, with infinities and NaN, and beside them rows that stay what
    they are alone."""
    x = _rows(gpu, 9, 200, F32, 4)
    alone = x.clone()
    x[1] = 0.0
    x[2] = 0.0
    x[2, 7] = -3.0
    x[3, 5] = float("nan")
    x[4, 0] = float("inf")
    x[6] = 1e-30
    w = torch.ones(200, device=gpu)
    for quant in ("int8", "e4m3"):
        out = K.add_rms_norm(x, w, None, EPS, quant=quant)
        assert (out.y[1] == 0).all() and (out.q[1] == 0).all() and out.scale[1] == 1.0
        assert abs(out.y[2, 7].item() + 3.0 / (9.0 / 200 + EPS)**0.5) < 1e-5 and (out.y[2, :7] == 0).all()
        assert torch.isnan(out.y[3]).all() and torch.isnan(out.y[4, 0])
        # 1e-30 squared is nothing: the root is eps's
        assert torch.allclose(out.y[6], torch.full((200,), 1e-30 * EPS**-0.5, device=gpu), rtol=1e-6)
        ref = K.add_rms_norm(alone, w, None, EPS, quant=quant)
        for i in (0, 5, 7, 8):
            assert torch.equal(out.y[i], ref.y[i]) and torch.equal(out.q[i], ref.q[i])
    bad = K.add_rms_norm(x, w, None, EPS, quant="int8")
    back = K.dequantize_rows_i8(bad.q, bad.scale, F32)
    assert torch.isnan(back[3]).all() and torch.isnan(back[4]).all()


def test_no_rows(gpu):
    x = torch.empty((0, 64), device=gpu)
    w = torch.ones(64, device=gpu)
    out = K.add_rms_norm(x, w, x, quant="int8")
    assert out.y.shape == (0, 64) and out.q.shape == (0, 64)
    dx, dw = K.add_rms_norm_bwd(x, x, w, out.rstd)
    assert dx.shape == (0, 64) and (dw == 0).all()


@pytest.mark.parametrize("rows,cols", [(1, 8), (3, 24), (40, 256), (5, 1032), (700, 2048), (33, 4104), (6, 8200),
                                       (3, 32768), (2050, 40), (5000, 1056), (2049, 2048), (9000, 64), (4001, 2056),
                                       (768, 264), (769, 264), (777, 8200), (780, 16392), (40, 16384)])
@pytest.mark.parametrize("g_type,s_type,more", [(BF16, BF16, True), (F32, F32, True), (BF16, F32, False),
                                                (F32, BF16, True), (BF16, BF16, False)])
def test_gradients(gpu, rows, cols, g_type, s_type, more):
    s = _rows(gpu, rows, cols, s_type, 2 * rows + cols)
    dy = _rows(gpu, rows, cols, g_type, 2 * rows + cols + 1, 1e-2)
    ds = _rows(gpu, rows, cols, s_type, 2 * rows + cols + 2, 1e-2) if more else None
    w = 1.0 + 0.2 * torch.randn(cols, generator=torch.Generator(device=gpu).manual_seed(3), device=gpu)
    if cols % 16 == 0:
        w = w.to(BF16)
    rstd = (s.double().square().mean(1) + EPS).rsqrt().float()
    dx, dw = K.add_rms_norm_bwd(dy, s, w, rstd, ds)
    assert dx.dtype == s_type and dw.dtype == F32
    u = 2.0**-24
    r = rstd.double().unsqueeze(1)
    n, dn = s.double() * r, dy.double() * w.double()
    mean = (dn * n).mean(1, keepdim=True)
    size = (dn * n).abs().mean(1, keepdim=True)
    want = r * (dn - n * mean) + (ds.double() if more else 0.0)
    # n, dn and their product are rounded, then the row's sum; the last line's operations
    bound = (_terms(cols) + 4) * u * r * n.abs() * size + 6 * u * (r * (dn.abs() + (n * mean).abs()) + want.abs())
    assert ((dx.double() - want).abs() <= bound + 1.01 * HALF_STEP[s_type] * (want.abs() + bound) + 1e-40).all()
    # a part's rows one after another, a run of parts, the 32 runs, the products and n
    parts = max(1, _lib.lib().hmoe_add_rms_norm_bwd_workspace_bytes(rows, cols) // (4 * cols))
    terms = -(-rows // parts) + 1 + -(-parts // 32) + 32 + 2
    assert ((dw.double() - (dy.double() * n).sum(0)).abs() <= terms * u * (dy.double() * n).abs().sum(0) + 1e-40).all()
    only, none = K.add_rms_norm_bwd(dy, s, w, rstd, ds, need_weight=False)
    assert none is None and torch.equal(only, dx)
    again = K.add_rms_norm_bwd(dy, s, w, rstd, ds)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


def test_gradients_against_differences(gpu):
    """Central differences of the float64 formula along random directions."""
    rows, cols, step = 5, 72, 1e-4
    g = torch.Generator().manual_seed(11)
    x, r, dy, ds = (torch.randn((rows, cols), generator=g, dtype=torch.float64) for _ in range(4))
    w = 1.0 + 0.3 * torch.randn(cols, generator=g, dtype=torch.float64)
    x, r, dy, ds, w = (t.float() for t in (x, r, dy, ds, w))
    out = K.add_rms_norm(x.to(gpu), w.to(gpu), r.to(gpu), EPS)
    dx, dw = K.add_rms_norm_bwd(dy.to(gpu), out.sum, w.to(gpu), out.rstd, ds.to(gpu))

    def value(total, weight):
        y = total / (total.square().mean(1, keepdim=True) + EPS).sqrt() * weight
        return (y * dy.double()).sum() + (total * ds.double()).sum()

    total = out.sum.cpu().double()
    for _ in range(4):
        d, e = torch.randn((rows, cols), generator=g, dtype=torch.float64), torch.randn(cols, generator=g, dtype=torch.float64)
        slope = (value(total + step * d, w.double()) - value(total - step * d, w.double())) / (2 * step)
        # float32 gradients: some 80 roundings of terms whose sizes add up to this; the
        # differences' own error is a third derivative times 1e-8
        size = (dx.cpu().double() * d).abs().sum() + (dy.double() * d).abs().sum()
        assert abs((dx.cpu().double() * d).sum() - slope) <= 80 * 2.0**-24 * size + 1e-6 * size
        slope = (value(total, w.double() + step * e) - value(total, w.double() - step * e)) / (2 * step)
        size = (dw.cpu().double() * e).abs().sum() + (dy.double() * total).abs().sum()
        assert abs((dw.cpu().double() * e).sum() - slope) <= 80 * 2.0**-24 * size + 1e-6 * size


def test_results_over_operands(gpu):
    """sum over x or the residual, y over x, dx over its operands, as the header allows."""
    rows, cols = 37, 520
    x, r = _rows(gpu, rows, cols, BF16, 1), _rows(gpu, rows, cols, BF16, 2)
    w = torch.ones(cols, device=gpu)
    want = K.add_rms_norm(x, w, r, EPS)

    def call(x, r, total, y):
        rstd = torch.empty(rows, device=gpu)
        _lib.call("hmoe_add_rms_norm", x.data_ptr(), _lib.BF16, r.data_ptr(), _lib.BF16, w.data_ptr(), _lib.F32, EPS,
                  rows, cols, total.data_ptr(), y.data_ptr(), _lib.BF16, rstd.data_ptr(), None, 0, None,
                  torch.cuda.current_stream().cuda_stream)
        return total, y

    for over in range(3):
        a, b, free = x.clone(), r.clone(), torch.empty_like(x)
        total, y = call(a, b, *((a, free), (b, free), (b, a))[over])
        assert torch.equal(total, want.sum) and torch.equal(y, want.y)
    dy, ds = _rows(gpu, rows, cols, BF16, 3), _rows(gpu, rows, cols, BF16, 4)
    dx, _ = K.add_rms_norm_bwd(dy, want.sum, w, want.rstd, ds, need_weight=False)
    for over in range(3):
        ops = [dy.clone(), want.sum.clone(), ds.clone()]
        _lib.call("hmoe_add_rms_norm_bwd", ops[0].data_ptr(), _lib.BF16, ops[1].data_ptr(), _lib.BF16, w.data_ptr(),
                  _lib.F32, want.rstd.data_ptr(), ops[2].data_ptr(), rows, cols, ops[over].data_ptr(), None, None, 0,
                  torch.cuda.current_stream().cuda_stream)
        assert torch.equal(ops[over], dx)


@pytest.mark.parametrize("rows,cols", [(1, 264), (37, 520), (768, 1032), (900, 520), (30, 8200), (3000, 256)])
def test_gradients_over_operands(gpu, rows, cols):
    """dx over its operands with the weight's gradient wanted, which reads two of them."""
    s, dy, ds = (_rows(gpu, rows, cols, BF16, i) for i in (2, 3, 4))
    w = torch.ones(cols, device=gpu)
    rstd = torch.rand(rows, device=gpu) + 0.5
    dx, dw = K.add_rms_norm_bwd(dy, s, w, rstd, ds)
    need = _lib.lib().hmoe_add_rms_norm_bwd_workspace_bytes(rows, cols)
    for over in range(3):
        ops = [dy.clone(), s.clone(), ds.clone()]
        got, ws = torch.empty_like(dw), torch.empty(need, dtype=torch.uint8, device=gpu)
        _lib.call("hmoe_add_rms_norm_bwd", ops[0].data_ptr(), _lib.BF16, ops[1].data_ptr(), _lib.BF16, w.data_ptr(),
                  _lib.F32, rstd.data_ptr(), ops[2].data_ptr(), rows, cols, ops[over].data_ptr(), got.data_ptr(),
                  ws.data_ptr() if need else None, need, torch.cuda.current_stream().cuda_stream)
        assert torch.equal(ops[over], dx) and torch.equal(got, dw)


def test_more_rows_than_a_grid(gpu):
    """Rows past 2^22 are taken in a second round of the workgroups; offsets pass 2^31 bytes."""
    rows, cols = (1 << 22) + 5, 264
    g = torch.Generator(device=gpu).manual_seed(2)
    x = torch.randn((rows, cols), generator=g, device=gpu, dtype=BF16)
    w = torch.ones(cols, device=gpu)
    out = K.add_rms_norm(x, w, None, EPS, quant="int8")
    q, scale = K.quantize_rows_i8(out.y)
    for lo in (0, (1 << 22) - 3):
        part = K.add_rms_norm(x[lo:lo + 8].clone(), w, None, EPS, quant="int8")
        hi = min(lo + 8, rows)
        n = hi - lo
        # (few rows are summed by a workgroup, many by a wave each: another order)
        assert ((part.rstd[:n] / out.rstd[lo:hi] - 1).abs() < 64 * 2.0**-24).all()
        assert torch.equal(out.q[lo:hi], q[lo:hi]) and torch.equal(out.scale[lo:hi], scale[lo:hi])
        again = K.quantize_rows_i8(out.y[lo:hi].clone())
        assert torch.equal(again[0], q[lo:hi]) and torch.equal(again[1], scale[lo:hi])
        back = K.dequantize_rows_i8(q, scale)[lo:hi]
        assert torch.equal(back, (q[lo:hi].float() * scale[lo:hi].unsqueeze(1)).to(BF16))

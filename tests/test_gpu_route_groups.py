"""Routing limited to groups on the GPU: which experts are taken, bit for bit."""
import numpy as np
import pytest
import torch

import oracle as O
from hanuman_amd import _lib, kernels as K
from oracle import moe_oracle as M

pytestmark = pytest.mark.gpu

SIGMOID, SOFTMAX = _lib.ROUTE_SIGMOID_BIAS, _lib.ROUTE_SOFTMAX
LOWEST = -2**31 + 1     # of the keys; NaN scores have it


def _select(logits, bias, k, mode, rsf, groups, top):
    """(indices, gates) from the definition: float32 keys in totalOrder, lower index first."""
    t, n = logits.shape
    value = M.sigmoid_det(logits) if mode == SIGMOID else logits
    key = value if mode == SOFTMAX or bias is None else (value + bias[None, :]).astype(np.float32)
    order = np.maximum(M.total_order_key(key), LOWEST).reshape(t, groups, n // groups)
    if mode == SIGMOID:
        best = np.sort(order, axis=2)[:, :, -2:]
        as_value = np.where(best < 0, best ^ 0x7FFFFFFF, best).astype(np.int32).view(np.float32)
        with np.errstate(invalid="ignore"):
            score = (as_value[:, :, 0] + as_value[:, :, 1]).astype(np.float32)
        score = np.where(np.isnan(score), LOWEST, np.maximum(M.total_order_key(score), LOWEST))
    else:
        score = order.max(2)
    first = np.argsort(-score, axis=1, kind="stable")[:, :top]
    kept = np.zeros((t, groups), dtype=bool)
    np.put_along_axis(kept, first, True, axis=1)
    order = np.where(kept[:, :, None], order, -2**40).reshape(t, n)
    idx = np.argsort(-order, axis=1, kind="stable")[:, :k]
    picked = np.take_along_axis(value, idx, axis=1)
    if mode == SOFTMAX:
        picked = M.exp_det((picked - picked[:, :1]).astype(np.float32))
    total = np.zeros(t, dtype=np.float32)
    for j in range(k):
        total = (total + picked[:, j]).astype(np.float32)
    if mode == SOFTMAX:
        return idx, (picked / total[:, None]).astype(np.float32)
    total = (total + np.float32(1e-9)).astype(np.float32)
    return idx, ((picked / total[:, None]).astype(np.float32) * np.float32(rsf)).astype(np.float32)


# experts, groups, groups taken, experts taken
SHAPES = [(64, 8, 4, 8), (256, 8, 4, 8), (256, 2, 1, 32), (80, 4, 2, 8), (256, 64, 3, 12), (6, 3, 2, 3), (8, 2, 1, 4),
          (255, 3, 2, 7), (130, 5, 1, 26), (16, 8, 1, 2), (160, 16, 4, 9), (4, 2, 1, 1), (128, 32, 31, 32), (96, 3, 2, 6),
          (250, 2, 1, 5), (34, 17, 16, 32), (256, 128 // 4, 2, 16),
          # lists of sixteen and of 32, on tokens of eight and sixteen lanes
          (128, 8, 2, 32), (120, 8, 3, 25), (112, 8, 7, 17), (120, 8, 1, 13), (60, 4, 3, 9), (256, 16, 2, 32), (252, 7, 6, 31)]


def _check(gpu, logits, bias, shape, mode, rsf=2.5):
    n, groups, top, k = shape
    b = None if bias is None else torch.from_numpy(bias).to(gpu)
    idx, gates = K.router_from_logits(torch.from_numpy(logits).to(gpu), b, k, mode, rsf, groups, top)
    want_idx, want_gates = _select(logits, bias, k, mode, rsf, groups, top)
    assert np.array_equal(idx.cpu().numpy(), want_idx)
    assert np.array_equal(gates.cpu().numpy(), want_gates, equal_nan=True)


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("mode", [SIGMOID, SOFTMAX], ids=["sigmoid", "softmax"])
@pytest.mark.parametrize("tokens", [1, 7, 33, 1000])
def test_from_logits(gpu, shape, mode, tokens):
    rng = np.random.default_rng(shape[0] * 7 + tokens)
    logits = rng.standard_normal((tokens, shape[0])).astype(np.float32)
    bias = (0.05 * rng.standard_normal(shape[0])).astype(np.float32)
    _check(gpu, logits, bias if mode == SIGMOID else None, shape, mode)
    if mode == SIGMOID:
        _check(gpu, logits, None, shape, mode)


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("mode", [SIGMOID, SOFTMAX], ids=["sigmoid", "softmax"])
def test_ties(gpu, shape, mode):
    """Few different logits and biases: equal keys and equal scores everywhere."""
    rng = np.random.default_rng(shape[0])
    logits = rng.integers(-1, 2, (400, shape[0])).astype(np.float32)
    logits[0] = 0.0
    bias = (0.1 * rng.integers(-1, 2, shape[0])).astype(np.float32)
    _check(gpu, logits, bias if mode == SIGMOID else None, shape, mode)


@pytest.mark.parametrize("mode", [SIGMOID, SOFTMAX], ids=["sigmoid", "softmax"])
def test_values_that_are_not_ordinary(gpu, mode):
    """Infinities, the lowest and the largest numbers, zeros of both signs; NaN in softmax
    (with sigmoid a NaN's sign is the arithmetic's)."""
    rng = np.random.default_rng(3)
    pool = np.array([np.inf, -np.inf, np.finfo(np.float32).max, np.finfo(np.float32).min, 0.0, -0.0, 88.0, -88.0,
                     -100.0, 1e-40, 1.0], dtype=np.float32)
    logits = rng.choice(pool, (300, 64)).astype(np.float32)
    logits[5] = -np.inf
    n, groups, top, k = 64, 8, 3, 8
    bias = np.where(rng.random(64) < 0.1, -np.inf, 0.1).astype(np.float32) if mode == SIGMOID else None
    b = None if bias is None else torch.from_numpy(bias).to(gpu)
    idx, _ = K.router_from_logits(torch.from_numpy(logits).to(gpu), b, k, mode, 1.0, groups, top)
    with np.errstate(all="ignore"):
        assert np.array_equal(idx.cpu().numpy(), _select(logits, bias, k, mode, 1.0, groups, top)[0])
        if mode == SOFTMAX:
            logits[7, 20] = np.nan
            logits[8, 3] = np.array([0xFFFFFFFF], dtype=np.uint32).view(np.float32)[0]
            idx, _ = K.router_from_logits(torch.from_numpy(logits).to(gpu), None, k, mode, 1.0, groups, top)
            assert np.array_equal(idx.cpu().numpy(), _select(logits, None, k, mode, 1.0, groups, top)[0])


@pytest.mark.parametrize("mode", [SIGMOID, SOFTMAX], ids=["sigmoid", "softmax"])
def test_all_groups_are_the_router(gpu, mode):
    g = torch.Generator(device=gpu).manual_seed(1)
    logits = torch.randn((100, 96), generator=g, device=gpu)
    bias = 0.1 * torch.randn(96, generator=g, device=gpu) if mode == SIGMOID else None
    want = K.router_from_logits(logits, bias, 6, mode, 2.0)
    for groups in (1, 4, 96):
        for got in (K.router_from_logits(logits, bias, 6, mode, 2.0, groups, groups),
                    K.router_from_logits(logits, bias, 6, mode, 2.0, groups)):
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # the same selection from inside the grouped kernel: groups that hold what is taken
    first = logits.clone()
    first[:, 48:] -= 50.0
    want = K.router_from_logits(first, bias, 6, mode, 2.0)
    if mode == SOFTMAX:
        got = K.router_from_logits(first, bias, 6, mode, 2.0, 2, 1)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("x_type,w_type", [(torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("tokens,d_model,shape", [(1, 2048, (64, 8, 4, 8)), (5, 264, (80, 4, 2, 8)), (300, 512, (256, 8, 4, 8)),
                                                  (3000, 256, (16, 4, 1, 2)), (2500, 128, (30, 3, 2, 6)), (70, 64, (8, 4, 3, 5))])
@pytest.mark.parametrize("mode", [SIGMOID, SOFTMAX], ids=["sigmoid", "softmax"])
def test_router(gpu, x_type, w_type, tokens, d_model, shape, mode):
    n, groups, top, k = shape
    g = torch.Generator(device=gpu).manual_seed(tokens)
    x = torch.randn((tokens, d_model), generator=g, device=gpu).to(x_type)
    w = (torch.randn((d_model, n), generator=g, device=gpu) * d_model**-0.5).to(w_type)
    bias = 0.05 * torch.randn(n, generator=g, device=gpu) if mode == SIGMOID else None
    plain_logits, _, _ = K.router(x, w, bias, k, mode, 2.5)
    logits, idx, gates = K.router(x, w, bias, k, mode, 2.5, groups, top)
    assert torch.equal(logits, plain_logits)
    want_idx, want_gates = _select(logits.cpu().numpy(), None if bias is None else bias.cpu().numpy(), k, mode, 2.5,
                                   groups, top)
    assert np.array_equal(idx.cpu().numpy(), want_idx) and np.array_equal(gates.cpu().numpy(), want_gates)


@pytest.mark.parametrize("shape", [(96, 6, 3, 9), (256, 8, 4, 32), (34, 17, 16, 32), (64, 4, 1, 16), (128, 8, 5, 32)],
                         ids=str)
@pytest.mark.parametrize("mode", [SIGMOID, SOFTMAX], ids=["sigmoid", "softmax"])
def test_router_with_more_experts_a_token(gpu, shape, mode):
    """More than eight experts: the selection in a launch behind the logits'."""
    n, groups, top, k = shape
    g = torch.Generator(device=gpu).manual_seed(n)
    x = torch.randn((130, 128), generator=g, device=gpu).bfloat16()
    w = torch.randn((128, n), generator=g, device=gpu).bfloat16() * 128**-0.5
    bias = 0.05 * torch.randn(n, generator=g, device=gpu) if mode == SIGMOID else None
    logits, idx, gates = K.router(x, w, bias, k, mode, 1.5, groups, top)
    assert torch.equal(logits, K.router(x, w, bias, 8, mode, 1.5)[0])
    want_idx, want_gates = _select(logits.cpu().numpy(), None if bias is None else bias.cpu().numpy(), k, mode, 1.5,
                                   groups, top)
    assert np.array_equal(idx.cpu().numpy(), want_idx) and np.array_equal(gates.cpu().numpy(), want_gates)


@pytest.mark.parametrize("shape", [(256, 8, 4, 8), (64, 8, 2, 12), (36, 3, 2, 7)], ids=str)
@pytest.mark.parametrize("logits_at,bias_at", [(1, 0), (0, 1), (2, 3), (3, 0)])
def test_logits_and_bias_inside_buffers(gpu, shape, logits_at, bias_at):
    """Operands that start anywhere: the results of the same values at 16 bytes."""
    n, groups, top, k = shape
    rng = np.random.default_rng(n + logits_at)
    logits = torch.from_numpy(rng.standard_normal((77, n)).astype(np.float32)).to(gpu)
    bias = torch.from_numpy((0.05 * rng.standard_normal(n)).astype(np.float32)).to(gpu)

    def inside(t, at):
        buffer = torch.full((t.numel() + 8,), float("nan"), device=gpu)
        buffer[at:at + t.numel()] = t.reshape(-1)
        return buffer[at:at + t.numel()].view(t.shape)

    want = K.router_from_logits(logits, bias, k, SIGMOID, 2.5, groups, top)
    got = K.router_from_logits(inside(logits, logits_at), inside(bias, bias_at), k, SIGMOID, 2.5, groups, top)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("shape", [(64, 8, 3, 8), (250, 5, 2, 7), (128, 4, 2, 20)], ids=str)
@pytest.mark.parametrize("mode", [SIGMOID, SOFTMAX], ids=["sigmoid", "softmax"])
def test_nan_takes_experts_that_exist(gpu, shape, mode):
    """Rows with NaN, alone or throughout, from logits and from tokens: every slot has another
    expert, from as many groups as are taken; rows without are not touched by them."""
    n, groups, top, k = shape
    g = torch.Generator(device=gpu).manual_seed(n)
    x = torch.randn((48, 64), generator=g, device=gpu)
    w = torch.randn((64, n), generator=g, device=gpu) / 8
    bias = 0.05 * torch.randn(n, generator=g, device=gpu) if mode == SIGMOID else None
    clean = K.router(x, w, bias, k, mode, 1.0, groups, top)
    bad = x.clone()
    bad[3] = float("nan")
    bad[17, 5] = float("inf")
    one = clean[0].clone()
    one[3] = float("nan")
    one[17, n // 2:n // 2 + 3] = float("nan")
    one[18, ::2] = -float("nan")
    ordinary = torch.ones(48, dtype=torch.bool, device=gpu)
    ordinary[[3, 17, 18]] = False
    for idx, gates in (K.router(bad, w, bias, k, mode, 1.0, groups, top)[1:],
                       K.router_from_logits(one, bias, k, mode, 1.0, groups, top)):
        assert int(idx.min()) >= 0 and int(idx.max()) < n
        for row in idx.cpu().tolist():
            assert len(set(row)) == k and len({i // (n // groups) for i in row}) <= top
        assert torch.equal(idx[ordinary], clean[1][ordinary]) and torch.equal(gates[ordinary], clean[2][ordinary])


def test_no_tokens(gpu):
    logits, idx, gates = K.router(torch.empty((0, 64), device=gpu), torch.zeros((64, 8), device=gpu), None, 2, SOFTMAX,
                                  1.0, 4, 2)
    assert logits.shape == (0, 8) and idx.shape == (0, 2) and gates.shape == (0, 2)


@pytest.mark.parametrize("mode", [SIGMOID, SOFTMAX], ids=["sigmoid", "softmax"])
def test_gradient(gpu, mode):
    """The gates' gradient with the selection held fixed: against the formula in float64 and
    against differences of the gates."""
    n, groups, top, k, rsf = 24, 4, 2, 5, 2.5 if mode == SIGMOID else 1.0
    g = torch.Generator().manual_seed(9)
    logits = torch.randn((40, n), generator=g)
    bias = 0.05 * torch.randn(n, generator=g) if mode == SIGMOID else None
    dg = torch.randn((40, k), generator=g)
    on = lambda t: None if t is None else t.to(gpu)
    idx, gates = K.router_from_logits(on(logits), on(bias), k, mode, rsf, groups, top)
    dl = K.router_bwd(on(logits), idx, gates, on(dg), n, mode, rsf).cpu().double()
    idx = idx.cpu().long()

    def value(l):
        picked = torch.gather(l, 1, idx)
        if mode == SOFTMAX:
            return torch.softmax(picked, 1)
        s = torch.sigmoid(picked)
        return s / (s.sum(1, keepdim=True) + 1e-9) * rsf

    l64 = logits.double().requires_grad_(True)
    (value(l64) * dg.double()).sum().backward()
    # some 40 roundings of terms of at most rsf |dg|, each step's error of size 2^-24
    assert (dl - l64.grad).abs().max() <= 40 * 2.0**-24 * rsf * float(dg.abs().sum(1).max())
    untouched = torch.ones((40, n), dtype=torch.bool).scatter_(1, idx, False)
    assert (dl[untouched] == 0).all()
    step = 1e-4
    for _ in range(3):
        d = torch.randn((40, n), generator=g, dtype=torch.float64)
        slope = ((value(logits.double() + step * d) - value(logits.double() - step * d)) * dg.double()).sum() / (2 * step)
        assert abs((dl * d).sum() - slope) <= 1e-5 * (dl * d).abs().sum() + 1e-5


def test_rows_beside_the_results_are_left(gpu):
    """Buffers longer than the results keep what is behind them."""
    t, n, k = 13, 64, 6
    logits = torch.randn((t, n), device=gpu)
    idx = torch.full((t + 4, k), 77, dtype=torch.int32, device=gpu)
    gates = torch.full((t + 4, k), 7.0, device=gpu)
    _lib.call("hmoe_router_grouped_from_logits", logits.data_ptr(), None, t, n, k, SOFTMAX, 1.0, 8, 2, idx.data_ptr(),
              gates.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert (idx[t:] == 77).all() and (gates[t:] == 7.0).all() and (idx[:t] < n).all()


def test_where_nan_is(gpu):
    """Softmax: a NaN's group comes first, one of NaNs with the sign set last; sigmoid: a group
    whose sum is NaN comes last."""
    logits = np.tile(np.linspace(0.0, 1.0, 16, dtype=np.float32), (4, 1))
    nan, minus = np.array([0x7FC00000, 0xFFFFFFFF], dtype=np.uint32).view(np.float32)
    logits[1, 2] = logits[2, 9] = nan
    logits[3, 12:] = minus
    dev = torch.from_numpy(logits).to(gpu)
    idx, gates = K.router_from_logits(dev, None, 4, SOFTMAX, 1.0, 4, 1)
    groups = (idx // 4).cpu().numpy()
    assert (groups == np.array([3, 0, 2, 2])[:, None]).all()
    assert idx[1, 0] == 2 and idx[2, 0] == 9
    assert torch.isnan(gates[1:3]).all() and torch.isfinite(gates[[0, 3]]).all()
    idx, _ = K.router_from_logits(dev, None, 12, SIGMOID, 1.0, 4, 3)
    left_out = [(set(range(4)) - set((idx[t] // 4).tolist())).pop() for t in range(4)]
    assert left_out[0] == 0 and left_out[3] == 3

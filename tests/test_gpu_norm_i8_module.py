"""The norm, routing by groups and int8 experts run together: the module, the measured layer,
autograd and capture."""
from dataclasses import replace

import numpy as np
import pytest
import torch

import i8_reference as R
from hanuman_amd import MoE, RMSNorm, kernels as K, workloads as W
from hanuman_amd._lib import HmoeError
from hanuman_amd.layer import DeviceLayer

pytestmark = pytest.mark.gpu

B, S, D, F, N, TOP = 2, 31, 256, 128, 12, 3


def _layer(gpu, **kw):
    return MoE(D, kw.pop("d_ff", F), N, TOP, kw.pop("shared", 1), 0.02, 2.5, kw.pop("dtype", "bfloat16"), rngs=3, device=gpu,
               d_ff_shared=256, **kw)


def _tokens(gpu, seed=1, dtype=torch.bfloat16):
    return torch.randn((B, S, D), generator=torch.Generator(device=gpu).manual_seed(seed), device=gpu).to(dtype)


def _int8_layer(layer, y, codes, shared):
    """The operators of a layer with int8 experts in a row, on tokens y [T, D]."""
    T = y.shape[0]
    bias = layer.bias.value if layer.routing == "sigmoid" else None
    logits, idx, gates = K.router(y, layer.router.value, bias, TOP, 0, 2.5, layer.n_groups, layer.top_groups)
    plan = K.dispatch_plan(idx, N, T * TOP)
    gu = K.pack_i8_gate_up(layer.expert_w_gate.value, layer.expert_w_up.value)
    dn = K.pack_i8_down(layer.expert_w_down.value)
    h = K.grouped_gate_up_i8_gather(*codes, plan, *gu)
    ys = K.grouped_down_i8(*K.quantize_rows_i8(h, plan.offsets), plan.offsets, *dn)
    return K.combine(ys, plan, gates, shared, torch.float32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("shared", [1, 2])
@pytest.mark.parametrize("groups", [(1, None), (4, 2)])
def test_module(gpu, dtype, shared, groups):
    """Against the operators in a row, and against the bf16 module on the same weights."""
    kw = dict(shared=shared, n_groups=groups[0], top_groups=groups[1])
    eight, full = _layer(gpu, expert_dtype="int8", **kw), _layer(gpu, **kw)
    x = _tokens(gpu, dtype=dtype)
    out, aux = eight(x)
    ref, ref_aux = full(x)
    assert out.shape == (B, S, D) and out.dtype == torch.float32
    for k in aux:
        assert torch.equal(aux[k], ref_aux[k])          # the router is the same
    y = x.reshape(B * S, D)
    part = eight._shared_ffn_promoted(y) if dtype == torch.float32 else eight._shared_ffn(y)
    assert torch.equal(out.reshape(B * S, D), _int8_layer(eight, y, K.quantize_rows_i8(y), part))
    # a code is off by half a 127th of its row's largest, about 3.5 root mean squares: 0.8 % of
    # a root mean square; tokens, two weights and h so rounded: under 4 %, over bf16's 0.1 %
    err = float((out - ref).norm() / ref.norm())
    assert 0.001 < err < 0.04, err


def test_module_follows_its_masters(gpu):
    layer = _layer(gpu, expert_dtype="int8")
    x = _tokens(gpu)
    a, _ = layer(x)
    assert torch.equal(a, layer(x)[0])
    with torch.no_grad():
        layer.expert_w_down.value.mul_(3.0)
    b, _ = layer(x)
    assert not torch.equal(a, b)
    layer.load_state(layer.state())
    assert torch.equal(layer(x)[0], b)


def test_int8_refuses_gradients(gpu):
    layer = _layer(gpu, expert_dtype="int8")
    x = _tokens(gpu).requires_grad_(True)
    with pytest.raises(NotImplementedError, match="int8"):
        layer(x)
    with pytest.raises(NotImplementedError, match="int8"):
        layer.behind_norm(RMSNorm(D, device=gpu), x)
    with torch.no_grad():
        layer(x)


@pytest.mark.parametrize("experts", [None, "int8", "mxfp4"])
@pytest.mark.parametrize("x_type,r_type", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32),
                                           (torch.float32, torch.bfloat16), (torch.bfloat16, None)])
def test_behind_norm(gpu, experts, x_type, r_type):
    """The block's half: addition, norm (with the tokens' codes), routing by groups, experts."""
    layer = _layer(gpu, expert_dtype=experts, n_groups=4, top_groups=2)
    norm = RMSNorm(D, 1e-5, device=gpu)
    norm.scale.value += 0.1 * torch.randn(D, generator=torch.Generator(device=gpu).manual_seed(5), device=gpu)
    x = _tokens(gpu, 1, x_type)
    r = None if r_type is None else _tokens(gpu, 2, r_type)
    out, total, aux = layer.behind_norm(norm, x, r)
    want = x if r is None else (x.float() + r.float()).to(r_type)
    assert torch.equal(total, want) and total.shape == (B, S, D)
    y = K.add_rms_norm(want.reshape(-1, D), norm.scale.value, None, 1e-5, out_dtype=torch.bfloat16).y
    ref, ref_aux = layer(y.view(B, S, D))
    assert torch.equal(out, ref)
    for k in aux:
        assert torch.equal(aux[k], ref_aux[k])
    if experts == "int8":
        assert torch.equal(out.reshape(-1, D), _int8_layer(layer, y, K.quantize_rows_i8(y), layer._shared_ffn(y)))


def test_behind_norm_float32(gpu):
    layer = _layer(gpu, dtype="float32", n_groups=3, top_groups=1)
    norm = RMSNorm(D, device=gpu)
    x, r = _tokens(gpu, 1, torch.float32), _tokens(gpu, 2, torch.float32)
    out, total, _ = layer.behind_norm(norm, x, r)
    y, total2 = norm.with_sum(x, r)
    assert torch.equal(total, total2) and torch.equal(out, layer(y)[0])


@pytest.mark.parametrize("compute", ["bfloat16", "float32"])
def test_training_behind_norm(gpu, compute):
    """Gradients through experts of the best groups, the norm and the addition: the layer's own
    gradient (tested elsewhere) carried on through the norm's formula in float64."""
    # (256: the bf16 gradients' products)
    layer = _layer(gpu, dtype=compute, d_ff=256, n_groups=4, top_groups=2)
    norm = RMSNorm(D, 1e-5, device=gpu)
    dt = layer.dtype
    x, r = _tokens(gpu, 1, dt).requires_grad_(True), _tokens(gpu, 2, torch.float32).requires_grad_(True)
    norm.scale.value.requires_grad_(True)
    params = [p.value.requires_grad_(True) for n, p in layer.named_params().items() if n != "bias"]
    out, total, aux = layer.behind_norm(norm, x, r)
    g = torch.Generator(device=gpu).manual_seed(7)
    dy, ds = torch.randn((B, S, D), generator=g, device=gpu), torch.randn((B, S, D), generator=g, device=gpu)
    grads = torch.autograd.grad((out, total, aux["router_z_loss"]), [x, r, norm.scale.value, *params],
                                (dy, ds, torch.ones((), device=gpu)), retain_graph=True)
    # the layer alone on the same normed tokens
    y, total2 = norm.with_sum(x.detach(), r.detach(), out_dtype=dt)
    assert torch.equal(total, total2)
    y = y.detach().requires_grad_(True)
    out2, aux2 = layer(y)
    assert torch.equal(out, out2)
    inner = torch.autograd.grad((out2, aux2["router_z_loss"]), [y, *params], (dy, torch.ones((), device=gpu)))
    for a, b in zip(grads[3:], inner[1:]):
        assert torch.equal(a, b)
    t64 = total.detach().double().requires_grad_(True)
    w64 = norm.scale.value.detach().double().requires_grad_(True)
    y64 = t64 / (t64.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w64
    want_t, want_w = torch.autograd.grad((y64, t64 * 1.0), (t64, w64), (inner[0].double(), ds.double()))
    # float32 sums of 256 terms and rstd's rounding: 80 steps of the terms' size
    size = want_t.abs() + inner[0].double().abs().amax(-1, keepdim=True) * 4
    assert ((grads[1].double() - want_t).abs() <= 80 * 2.0**-24 * size).all()
    assert grads[0].dtype == dt and torch.equal(grads[0], grads[1].to(dt))
    size = (inner[0].double() * y64.detach()).abs().sum((0, 1)) + 1e-6
    assert ((grads[2].double() - want_w).abs() <= 80 * 2.0**-24 * size).all()
    # a retained graph again
    again = torch.autograd.grad(total, [x, r], ds)
    assert torch.equal(again[1], ds) and torch.equal(again[0], ds.to(dt))


def test_norm_alone_under_autograd(gpu):
    norm = RMSNorm(D, device=gpu)
    x = _tokens(gpu, 1, torch.float32).requires_grad_(True)
    y = norm(x)
    assert torch.equal(y, norm(x.detach()))
    y.backward(torch.ones_like(y))
    rstd = (x.detach().double().square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    n = x.detach().double() * rstd
    want = rstd * (1 - n * n.mean(-1, keepdim=True))
    assert ((x.grad.double() - want).abs() <= 80 * 2.0**-24 * rstd * (1 + n.abs())).all()
    assert norm.scale.value.grad is None
    with pytest.raises(ValueError, match="shape"):
        norm.with_sum(x, x[:, :5])


def _inside(t, elements):
    buffer = torch.zeros(t.numel() + elements, dtype=t.dtype, device=t.device)
    buffer[elements:] = t.reshape(-1)
    view = buffer[elements:].view(t.shape)
    assert view.is_contiguous() and view.data_ptr() % 16 != 0
    return view


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_tensors_inside_buffers(gpu, dtype):
    """Tokens, masters and the norm's weight that start anywhere, and tokens with strides."""
    layer = _layer(gpu, expert_dtype="int8", n_groups=4, top_groups=2)
    norm = RMSNorm(D, device=gpu)
    x, r = _tokens(gpu, 1, dtype), _tokens(gpu, 2, dtype)
    want = layer.behind_norm(norm, x, r)
    plain = layer(x)[0]
    assert torch.equal(layer(_inside(x, 1))[0], plain)
    wide = torch.zeros((B, S, 2 * D), dtype=dtype, device=gpu)
    wide[:, :, ::2] = x
    for a, b in ((_inside(x, 1), _inside(r, 3)), (wide[:, :, ::2], r)):
        got = layer.behind_norm(norm, a, b)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    norm.scale.value = _inside(norm.scale.value, 1)
    for name in ("expert_w_gate", "expert_w_up", "expert_w_down"):
        param = getattr(layer, name)
        param.value = _inside(param.value, 2)
    assert torch.equal(layer.behind_norm(norm, x, r)[0], want[0])


@pytest.mark.parametrize("tokens,capacity", [(1, 1.25), (37, 0.5), (600, 1.25)])
def test_device_layer(gpu, tokens, capacity):
    wl = replace(W.WORKLOADS["full_bf16"], tokens=tokens, batch=1, d_model=256, d_ff=384, n_experts=12, top_k=3,
                 expert_dtype="int8", capacity_factor=capacity, weight_std=0.1)
    inp = W.make_inputs(wl, seed=2)
    r = DeviceLayer(inp, gpu).forward()
    plan = r["plan"]
    x_q, x_s = R.quantise(inp.x)
    assert np.array_equal(r["x_q"].cpu().numpy(), x_q) and np.array_equal(r["x_scale"].cpu().numpy(), x_s)
    off, src = plan.offsets.cpu().numpy(), plan.perm_src.cpu().numpy()
    kept = int(off[-1])
    h = R.bf16(np.zeros((len(src), 384), dtype=np.float32))
    got_q, got_s = r["h_q"].cpu().numpy(), r["h_scale"].cpu().numpy()
    ys = np.zeros((len(src), 256), dtype=np.float32)
    for e in range(12):
        lo, hi = off[e], off[e + 1]
        if lo == hi:
            continue
        rows = src[lo:hi] // 3
        q, s = R.quantise(R.gate_up_rows(inp.w_gate[e].T, inp.w_up[e].T))
        y = R.product(x_q[rows], x_s[rows], q, s).reshape(hi - lo, -1, 2, 32)
        want, bound = R.swiglu_with_bound(y[:, :, 0].reshape(hi - lo, -1), y[:, :, 1].reshape(hi - lo, -1))
        # h's codes stand for h rounded to bf16, then to half a code
        value = got_q[lo:hi] * got_s[lo:hi, None].astype(np.float64)
        off_by = bound + (np.abs(want) + bound) * 2.0**-8 + 0.5001 * got_s[lo:hi, None]
        assert (np.abs(value - want) <= off_by).all()
        q, s = R.quantise(inp.w_down[e].T)
        ys[lo:hi] = R.bf16(R.product(got_q[lo:hi], got_s[lo:hi], q, s))
    assert np.array_equal(r["ys"].float().cpu().numpy()[:kept], ys[:kept])
    g = R.bf16(r["gates"].cpu().numpy()).astype(np.float64)
    pos = plan.slot_pos.cpu().numpy().reshape(tokens, -1)
    out = sum(np.where(pos[:, k:k + 1] >= 0, g[:, k:k + 1] * ys[pos[:, k]].astype(np.float64), 0.0) for k in range(3))
    size = sum(np.where(pos[:, k:k + 1] >= 0, np.abs(g[:, k:k + 1] * ys[pos[:, k]]), 0.0) for k in range(3))
    assert (np.abs(r["out"].double().cpu().numpy() - out) <= 4 * 2.0**-24 * size).all()


def test_captured_and_replayed(gpu):
    """The block's half in a graph: replays on changed tokens, eager work between them, and a
    second graph of the same layer beside it."""
    layer = _layer(gpu, expert_dtype="int8", n_groups=4, top_groups=2)
    norm = RMSNorm(D, device=gpu)
    xs = [_tokens(gpu, s) for s in (1, 2, 3, 4)]
    want = [layer.behind_norm(norm, x, xs[0]) for x in xs]
    graphs = []
    for _ in range(2):
        x = xs[0].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            layer.behind_norm(norm, x, xs[0])
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = layer.behind_norm(norm, x, xs[0])
        graphs.append((graph, x, got))
    for i, w in enumerate(want):
        for graph, x, _ in graphs:
            x.copy_(xs[i])
            graph.replay()
        eager = layer.behind_norm(norm, xs[-1 - i], xs[0])
        torch.cuda.synchronize()
        for _, _, got in graphs:
            assert torch.equal(got[0], w[0]) and torch.equal(got[1], w[1])
        assert torch.equal(eager[0], want[-1 - i][0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_gradients_captured_and_replayed(gpu, dtype):
    """The norm's forward and backward in a graph, of two sizes of dw's sum, against eager runs
    between the replays; a second graph beside it has a workspace of its own."""
    rows, graphs = (1, 700), []
    norm = RMSNorm(D, device=gpu)
    norm.scale.value.requires_grad_(True)

    def step(x, r, dy):
        y, total = norm.with_sum(x, r)
        return torch.autograd.grad((y, total), (x, r, norm.scale.value), (dy, dy))

    def operands(n, seed):
        g = torch.Generator(device=gpu).manual_seed(seed)
        x, r, dy = (torch.randn((n, D), generator=g, device=gpu).to(dtype) for _ in range(3))
        return x.requires_grad_(True), r.requires_grad_(True), dy

    for n in rows:
        fixed = operands(n, 0)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*fixed)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step(*fixed)
        graphs.append((graph, n, fixed, got))
    for seed in (1, 2, 3):
        want = []
        for graph, n, fixed, _ in graphs:
            new = operands(n, seed)
            with torch.no_grad():
                for a, b in zip(fixed, new):
                    a.copy_(b)
            graph.replay()
            want.append(step(*new))
        torch.cuda.synchronize()
        for (_, _, _, got), w in zip(graphs, want):
            for a, b in zip(got, w):
                assert torch.equal(a, b)


def test_one_tensor_twice_and_broadcast_ones(gpu):
    """x as its own residual has both gradients; a row that is broadcast has its rows' sum."""
    norm = RMSNorm(D, device=gpu)
    g = torch.Generator(device=gpu).manual_seed(5)
    x = torch.randn((B, S, D), generator=g, device=gpu).requires_grad_(True)
    dy = torch.randn((B, S, D), generator=g, device=gpu)
    y, total = norm.with_sum(x, x)
    assert torch.equal(total, 2 * x.detach())
    both, = torch.autograd.grad((y, total), x, (dy, dy))
    other = x.detach().clone().requires_grad_(True)
    y, total = norm.with_sum(x, other)
    one, two = torch.autograd.grad((y, total), (x, other), (dy, dy))
    assert torch.equal(one, two) and torch.equal(both, one + two)
    row = torch.randn((1, 1, D), generator=g, device=gpu).requires_grad_(True)
    y, total = norm.with_sum(x, row.expand(B, S, D))
    each, summed = torch.autograd.grad((y, total), (x, row), (dy, dy))
    assert torch.equal(summed, each.sum((0, 1), keepdim=True))


def test_second_derivatives_are_refused(gpu):
    norm = RMSNorm(D, device=gpu)
    x = _tokens(gpu, 1, torch.float32).requires_grad_(True)
    dx, = torch.autograd.grad(norm(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.sum().backward()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_mxfp4_experts_of_groups(gpu, dtype):
    """The 4-bit experts with routing by groups, whose tokens are quantised in a launch of their
    own: the operators in a row."""
    layer = _layer(gpu, expert_dtype="mxfp4", n_groups=4, top_groups=2)
    x = _tokens(gpu, 1, dtype)
    out, aux = layer(x)
    t = x.view(-1, D)
    _, idx, gates = K.router(t, layer.router.value, layer.bias.value, TOP, 0, 2.5, 4, 2)
    plan = K.dispatch_plan(idx, N, t.shape[0] * TOP)
    gu = K.pack_mxfp4_gate_up(layer.expert_w_gate.value, layer.expert_w_up.value)
    dn = K.pack_mxfp4_down(layer.expert_w_down.value)
    h = K.grouped_gate_up_mxfp4_gather(*K.quantize_rows_mxfp4(t), plan, *gu)
    ys = K.grouped_down_mxfp4(*h, plan.offsets, *dn)
    part = layer._shared_ffn_promoted(t) if dtype == torch.float32 else layer._shared_ffn(t)
    assert torch.equal(out.view(-1, D), K.combine(ys, plan, gates, part, torch.float32))
    assert torch.equal(aux["expert_counts"], plan.counts)


def test_two_streams_at_once(gpu):
    layer = _layer(gpu, expert_dtype="int8", n_groups=4, top_groups=2)
    norm = RMSNorm(D, device=gpu)
    xs = [_tokens(gpu, s) for s in (1, 2)]
    want = [layer.behind_norm(norm, x, xs[0])[0] for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(layer.behind_norm(norm, xs[i], xs[0])[0])
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_no_tokens_and_one(gpu):
    """No tokens: the layer refuses them as without a norm (its losses are means over them), the
    operators give empty results."""
    layer = _layer(gpu, expert_dtype="int8", n_groups=4, top_groups=2)
    norm = RMSNorm(D, device=gpu)
    x = _tokens(gpu)[:1, :1]
    out, total, aux = layer.behind_norm(norm, x, x)
    assert out.shape == (1, 1, D) and int(aux["expert_counts"].sum()) == TOP
    none = x[:0]
    with pytest.raises(HmoeError, match="batch"):
        layer.behind_norm(norm, none, none)
    y, total = norm.with_sum(none, none)
    assert y.shape == total.shape == none.shape
    r = norm.rows(none, none, quant="int8")
    _, idx, _ = K.router(r.y, layer.router.value, layer.bias.value, TOP, 0, 2.5, 4, 2)
    gu = K.pack_i8_gate_up(layer.expert_w_gate.value, layer.expert_w_up.value)
    dn = K.pack_i8_down(layer.expert_w_down.value)
    off = torch.zeros(N + 1, dtype=torch.int32, device=gpu)
    h = K.grouped_gate_up_i8(r.q, r.scale, off, *gu)
    ys = K.grouped_down_i8(*K.quantize_rows_i8(h, off), off, *dn)
    assert idx.shape == (0, TOP) and h.shape == (0, F) and ys.shape == (0, D)

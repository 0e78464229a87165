"""The MXFP4 operators run together: the module, the measured layer and the capture."""
from dataclasses import replace

import numpy as np
import pytest
import torch

import mxfp4_reference as R
from hanuman_amd import MoE, _lib, kernels as K, workloads as W
from hanuman_amd.layer import DeviceLayer

pytestmark = pytest.mark.gpu


def _experts64(x_q, x_e, plan, wg, wu, wd, h_q, h_e):
    """float64 rows of the experts from the quantised tokens; h as the kernels rounded it
    (checked against its own sums), so that the down products are held to their own
    rounding alone."""
    x = R.values(x_q, x_e)
    off, src = plan.offsets.cpu().numpy(), plan.perm_src.cpu().numpy()
    N, D, F = wg.shape
    ys = np.zeros((len(src), D))
    bound = np.zeros((len(src), D))
    for e in range(N):
        lo, hi = off[e], off[e + 1]
        if lo == hi:
            continue
        a = x[src[lo:hi] // plan.top_k]
        g_w, u_w, d_w = (R.values(*R.quantise(w[e].T)) for w in (wg, wu, wd))
        g, u = a @ g_w.T, a @ u_w.T
        h, d = R.swiglu_with_bound(g, u, R.product_bound(a, g_w, D), R.product_bound(a, u_w, D))
        R.check_quantised(h_q[lo:hi], h_e[lo:hi], h, d, f"expert {e}")
        hv = R.values(h_q[lo:hi], h_e[lo:hi])
        ys[lo:hi] = hv @ d_w.T
        bound[lo:hi] = np.abs(ys[lo:hi]) * 2.0**-8 + 1.01 * R.product_bound(hv, d_w, F) + 1e-38
    return ys, bound


def _combined(ys, bound, plan, gates, T):
    """The combine of float64 rows: gates rounded to bf16, float32 sums over the slots."""
    g = torch.from_numpy(gates).bfloat16().double().numpy()
    pos = plan.slot_pos.cpu().numpy().reshape(T, -1)
    out, off = np.zeros((T, ys.shape[1])), np.zeros((T, ys.shape[1]))
    for k in range(pos.shape[1]):
        kept = pos[:, k] >= 0
        rows = pos[kept, k]
        out[kept] += g[kept, k:k + 1] * ys[rows]
        off[kept] += np.abs(g[kept, k:k + 1]) * (bound[rows] + (np.abs(ys[rows]) + bound[rows]) * 2.0**-20)
    return out, off + 1e-30


@pytest.mark.parametrize("tokens,capacity", [(1, 1.25), (37, 0.5), (600, 1.25)])
def test_device_layer(gpu, tokens, capacity):
    wl = replace(W.WORKLOADS["full_bf16"], tokens=tokens, batch=1, d_model=256, d_ff=384, n_experts=12, top_k=3,
                 expert_dtype="mxfp4", capacity_factor=capacity, weight_std=0.1)
    inp = W.make_inputs(wl, seed=2)
    r = DeviceLayer(inp, gpu).forward()
    plan = r["plan"]
    host = {k: r[k].cpu().numpy() for k in ("x_q", "x_exp", "h_q", "h_exp")}
    want_q, want_e = R.quantise(inp.x)
    assert np.array_equal(host["x_q"], want_q) and np.array_equal(host["x_exp"], want_e)
    ys, bound = _experts64(want_q, want_e, plan, inp.w_gate, inp.w_up, inp.w_down, host["h_q"], host["h_exp"])
    kept = int(plan.offsets[-1])
    got = r["ys"].double().cpu().numpy()
    assert (np.abs(got[:kept] - ys[:kept]) <= bound[:kept]).all()
    out, off = _combined(ys, bound, plan, r["gates"].cpu().numpy(), tokens)
    assert (np.abs(r["out"].double().cpu().numpy() - out) <= off).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("shared", [1, 2])
def test_module(gpu, dtype, shared):
    """Against the operators in a row, and against the bf16 module on the same weights."""
    B, S, D, F, N, Kk = 2, 31, 256, 128, 6, 2
    kw = dict(rngs=3, device=gpu, d_ff_shared=256)
    four = MoE(D, F, N, Kk, shared, 0.02, 2.5, "bfloat16", expert_dtype="mxfp4", **kw)
    full = MoE(D, F, N, Kk, shared, 0.02, 2.5, "bfloat16", **kw)
    x = torch.randn((B, S, D), generator=torch.Generator(device=gpu).manual_seed(1), device=gpu).to(dtype)
    out, aux = four(x)
    ref, ref_aux = full(x)
    assert out.shape == (B, S, D) and out.dtype == torch.float32
    for k in aux:
        assert torch.equal(aux[k], ref_aux[k])          # the router is the same
    x2 = x.reshape(B * S, D)
    logits, top_idx, gates = K.router(x2, four.router.value, four.bias.value, Kk, 0, 2.5)
    plan = K.dispatch_plan(top_idx, N, B * S * Kk)
    gu, dn = K.pack_mxfp4_gate_up(four.expert_w_gate.value, four.expert_w_up.value), K.pack_mxfp4_down(four.expert_w_down.value)
    ys = K.grouped_down_mxfp4(*K.grouped_gate_up_mxfp4_gather(*K.quantize_rows_mxfp4(x2), plan, *gu), plan.offsets, *dn)
    same = K.combine(ys, plan, gates, four._shared_ffn_promoted(x2) if dtype == torch.float32 else four._shared_ffn(x2),
                     torch.float32)
    assert torch.equal(out.reshape(B * S, D), same)
    # 4-bit operands: a rounding is off by up to a sixth of a value's size, about a tenth
    # of a block's root mean square; with tokens, two weights and h so rounded the outputs
    # are off by at most twice that and some, and by more than bf16 roundings alone (2^-8)
    err = float((out - ref).norm() / ref.norm())
    assert 0.005 < err < 0.3, err


def test_module_follows_its_masters(gpu):
    layer = MoE(256, 128, 4, 2, 1, 0.02, 1.0, "bfloat16", rngs=0, expert_dtype="mxfp4", device=gpu)
    x = torch.randn((1, 9, 256), device=gpu).bfloat16()
    a, _ = layer(x)
    assert torch.equal(a, layer(x)[0])
    with torch.no_grad():
        layer.expert_w_down.value.mul_(2.0)
    b, _ = layer(x)
    assert not torch.equal(a, b)
    state = layer.state()
    layer.load_state(state)
    assert torch.equal(layer(x)[0], b)


def test_module_refuses_autograd(gpu):
    layer = MoE(256, 128, 4, 2, 1, 0.02, 1.0, "bfloat16", rngs=0, expert_dtype="mxfp4", device=gpu)
    x = torch.randn((1, 4, 256), device=gpu).bfloat16().requires_grad_(True)
    with pytest.raises(NotImplementedError, match="backward"):
        layer(x)
    with torch.no_grad():
        assert layer(x)[0].shape == (1, 4, 256)


def test_layer_captured(gpu):
    """The measured layer in a graph, at a size of the tile forms, replayed with eager runs
    between."""
    wl = replace(W.WORKLOADS["full_bf16"], tokens=1500, batch=1, d_model=384, d_ff=640, n_experts=4, top_k=2,
                 expert_dtype="mxfp4", capacity_factor=None)
    layer = DeviceLayer(W.make_inputs(wl, seed=4), gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer.forward()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = layer.forward()
    for i in range(4):
        layer.x.copy_(torch.randn(layer.x.shape, generator=torch.Generator(device=gpu).manual_seed(i), device=gpu))
        graph.replay()
        got = {k: r[k].clone() for k in ("h_q", "h_exp", "ys", "out")}
        want = layer.forward()
        torch.cuda.synchronize()
        for k in got:
            assert torch.equal(got[k], want[k]), k


@pytest.mark.parametrize("T,D,N", [(1, 32, 8), (5, 96, 4), (37, 256, 16), (300, 4128, 32), (1000, 2048, 64),
                                   (6145, 1056, 16), (6151, 160, 12), (1537, 288, 64), (700, 64, 256),
                                   (4100, 64, 30)])
@pytest.mark.parametrize("wd", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_router_with_quantisation(gpu, T, D, N, wd):
    """The one launch gives the bits of the router and of the quantisation; rows of a wide
    range and one of zeros."""
    print(f"router quant T{T} D{D} N{N}", flush=True)
    g = torch.Generator(device="cpu").manual_seed(T + D)
    x = torch.randn(T, D, generator=g) * torch.exp(torch.rand(T, 1, generator=g) * 18 - 12)
    x[T // 3] = 0
    x = x.bfloat16().to(gpu)
    w = torch.randn(D, N, generator=g).mul(0.1).to(gpu, wd)
    bias = torch.randn(N, generator=g).mul(0.05).to(gpu)
    got = K.router_quant_mxfp4(x, w, bias, 3, _lib.ROUTE_SIGMOID_BIAS, 2.5)
    ref = (*K.router(x, w, bias, 3, _lib.ROUTE_SIGMOID_BIAS, 2.5), *K.quantize_rows_mxfp4(x))
    torch.cuda.synchronize()
    for i, (a, b) in enumerate(zip(got, ref)):
        assert a.dtype == b.dtype and torch.equal(a, b), i
    want_q, want_e = R.quantise(x.float().cpu().numpy())
    assert np.array_equal(got[3].cpu().numpy(), want_q) and np.array_equal(got[4].cpu().numpy(), want_e)


def test_module_captured(gpu):
    """The module in a graph after a first call (which packs the masters), replayed with
    eager calls between."""
    layer = MoE(256, 384, 6, 2, 1, 0.02, 1.0, "bfloat16", rngs=0, expert_dtype="mxfp4", device=gpu)
    x = torch.zeros((2, 150, 256), dtype=torch.bfloat16, device=gpu)
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            layer(x)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, aux = layer(x)
        for i in range(4):
            x.copy_(torch.randn(x.shape, generator=torch.Generator(device=gpu).manual_seed(i), device=gpu))
            graph.replay()
            got, counts = out.clone(), aux["expert_counts"].clone()
            want, want_aux = layer(x)
            torch.cuda.synchronize()
            assert torch.equal(got, want) and torch.equal(counts, want_aux["expert_counts"])

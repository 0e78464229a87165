"""The norm's gradients whose weight sum goes through a workspace: captured and replayed, two
graphs and two streams at a time; the sum of few rows within the bound of its runs."""
import pytest
import torch

from hanuman_amd import RMSNorm, _lib, kernels as K

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
# rows, columns: one launch; parts of a workgroup's rows each; of a wave's; rows of 1024 threads
SIZES = [(1, 256), (700, 256), (900, 256), (3000, 256), (900, 2056), (800, 8200)]


def _workspace(rows, cols):
    return _lib.lib().hmoe_add_rms_norm_bwd_workspace_bytes(rows, cols)


def _operands(gpu, rows, cols, dtype, seed):
    g = torch.Generator(device=gpu).manual_seed(seed)
    x, r, dy = (torch.randn((rows, cols), generator=g, device=gpu).to(dtype) for _ in range(3))
    return x.requires_grad_(True), r.requires_grad_(True), dy


def test_which_sizes_have_a_workspace(gpu):
    for rows, cols in SIZES:
        assert (_workspace(rows, cols) > 0) == (rows > 768)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("cols", sorted({c for _, c in SIZES}))
def test_captured_and_replayed(gpu, cols, dtype):
    """Graphs of every row count, two of each, replayed on changed operands one behind another and
    then on two streams, with eager calls between the replays; every replay against an eager run."""
    norm = RMSNorm(cols, device=gpu)
    norm.scale.value.requires_grad_(True)

    def step(x, r, dy):
        y, total = norm.with_sum(x, r)
        return torch.autograd.grad((y, total), (x, r, norm.scale.value), (dy, dy))

    graphs = []
    for rows in [r for r, c in SIZES if c == cols] * 2:
        fixed = _operands(gpu, rows, cols, dtype, 0)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*fixed)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step(*fixed)
        graphs.append((graph, rows, fixed, got))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for seed in (1, 2, 3, 4):
        new = [_operands(gpu, rows, cols, dtype, 10 * seed + i) for i, (_, rows, _, _) in enumerate(graphs)]
        want = [step(*n) for n in new]
        with torch.no_grad():
            for (_, _, fixed, _), n in zip(graphs, new):
                for a, b in zip(fixed, n):
                    a.copy_(b)
        torch.cuda.synchronize()
        for i, (graph, *_) in enumerate(graphs):
            if seed % 2:
                graph.replay()
                step(*new[i])
            else:
                with torch.cuda.stream(streams[i % 2]):
                    graph.replay()
        torch.cuda.synchronize()
        for (_, rows, _, got), w in zip(graphs, want):
            for a, b in zip(got, w):
                assert torch.equal(a, b), rows


@pytest.mark.parametrize("rows,cols", [s for s in SIZES if s[0] > 768])
def test_two_streams_at_once(gpu, rows, cols):
    norm = RMSNorm(cols, device=gpu)
    norm.scale.value.requires_grad_(True)
    ops = [_operands(gpu, rows, cols, BF16, seed) for seed in (1, 2)]

    def step(x, r, dy):
        y, total = norm.with_sum(x, r)
        return torch.autograd.grad((y, total), (x, norm.scale.value), (dy, dy))

    want = [step(*o) for o in ops]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(6):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(step(*ops[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for each in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(each, want[i]))


@pytest.mark.parametrize("rows,cols", [(1, 8), (31, 264), (33, 1032), (512, 2056), (768, 264), (768, 8192), (129, 8200),
                                       (768, 16392)])
@pytest.mark.parametrize("g_type,s_type", [(F32, F32), (BF16, BF16), (F32, BF16)])
def test_few_rows_sum(gpu, rows, cols, g_type, s_type):
    """The weight's gradient of up to 768 rows: 32 runs of rows (128 in workgroups of 1024
    threads, columns past 8192), each row's product added with one rounding, then the runs."""
    g = torch.Generator(device=gpu).manual_seed(rows + cols)
    s = torch.randn((rows, cols), generator=g, device=gpu).to(s_type)
    dy = torch.randn((rows, cols), generator=g, device=gpu).to(g_type)
    rstd = torch.rand(rows, generator=g, device=gpu) + 0.5
    assert _workspace(rows, cols) == 0
    _, dw = K.add_rms_norm_bwd(dy, s, torch.ones(cols, device=gpu), rstd)
    terms = dy.double() * (s.double() * rstd.double().unsqueeze(1))
    runs = 32 if cols <= 8192 else 128
    # n is rounded once, a run's sum once a row, the runs are added one after another
    off = 1 + -(-rows // runs) + (runs - 1)
    assert ((dw.double() - terms.sum(0)).abs() <= 1.001 * off * 2.0**-24 * terms.abs().sum(0)).all()

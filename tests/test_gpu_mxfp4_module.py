"""The module with MXFP4 experts on tensors that a program may hand it."""
import pytest
import torch

from hanuman_amd import MoE

pytestmark = pytest.mark.gpu


def _inside(t, elements):
    """The same values in a buffer of their own, `elements` behind its start."""
    buffer = torch.zeros(t.numel() + elements, dtype=t.dtype, device=t.device)
    buffer[elements:] = t.reshape(-1)
    view = buffer[elements:].view(t.shape)
    assert view.is_contiguous() and view.data_ptr() % 16 != 0
    return view


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_tensors_inside_buffers(gpu, dtype):
    """Tokens and masters that start anywhere in their buffers."""
    layer = MoE(256, 128, 6, 2, 1, 0.02, 2.5, "bfloat16", rngs=3, expert_dtype="mxfp4", device=gpu)
    x = torch.randn((2, 31, 256), generator=torch.Generator(device=gpu).manual_seed(1), device=gpu).to(dtype)
    want, aux = layer(x)
    got, got_aux = layer(_inside(x, 1))
    assert torch.equal(got, want) and all(torch.equal(got_aux[k], aux[k]) for k in aux)
    for name in ("expert_w_gate", "expert_w_up", "expert_w_down"):
        param = getattr(layer, name)
        param.value = _inside(param.value, 2)
    assert torch.equal(layer(x)[0], want)

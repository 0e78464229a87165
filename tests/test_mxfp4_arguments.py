"""What the Python layer of the MXFP4 calls says of their tensors, on the CPU: the checks
look at a tensor's class, type, size and device, never at its memory."""
import pytest
import torch

from hanuman_amd import kernels as K


class OnGpu(torch.Tensor):
    """A tensor subclass that says it is on a GPU, as the checks ask."""
    is_cuda = True


def _subclass(*shape, dtype):
    return torch.zeros(shape, dtype=dtype).as_subclass(OnGpu)


def test_index_arrays_of_a_subclass():
    """A Parameter's or a buffer's class does not matter: offsets and perm_src of the right
    type and size are taken, others refused for what is wrong with them."""
    t = _subclass(5, dtype=torch.int32)
    K._check_i32("call", "offsets", t, 5, t.device)
    for wrong in (_subclass(4, dtype=torch.int32), _subclass(5, dtype=torch.int64)):
        with pytest.raises(ValueError, match=r"offsets must be int32 \[5\]"):
            K._check_i32("call", "offsets", wrong, 5, t.device)
    with pytest.raises(ValueError, match="contiguous"):
        K._check_i32("call", "offsets", _subclass(10, dtype=torch.int32)[::2], 5, t.device)
    with pytest.raises(ValueError, match="tensors on"):
        K._check_i32("call", "offsets", t, 5, torch.device("cuda:1"))
    with pytest.raises(ValueError, match="GPU"):
        K._check_i32("call", "offsets", torch.zeros(5, dtype=torch.int32), 5, torch.device("cuda:0"))


def test_codes_of_a_subclass():
    t = _subclass(4, 32, dtype=torch.uint8)
    K._u8("call", t.device, t, (4, 32))
    with pytest.raises(ValueError, match="expected uint8"):
        K._u8("call", t.device, t, (4, 16))
    with pytest.raises(ValueError, match="tensors on"):
        K._u8("call", torch.device("cuda:1"), t, (4, 32))

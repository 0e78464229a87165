"""What the Python layer of the MXFP4 calls says of their tensors, on the CPU: the checks
look at a tensor's class, type, size and device, never at its memory."""
import ctypes

import pytest
import torch

from hanuman_amd import _lib, kernels as K


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


def _form(*sizes):
    return _lib.lib().hmoe_grouped_mxfp4_form(*sizes)


def test_form_of_sizes_that_the_products_refuse():
    """The query says -1 where the products refuse, at each limit and not below it."""
    top = 1 << 20
    assert _form(10, 1, top, 128, 256) >= 0 and _form(10, 1, top + 128, 128, 256) == -1
    assert _form(10, 1, 128, 2 * top, 256) >= 0 and _form(10, 1, 128, 2 * top + 128, 256) == -1
    # an expert's exponents of 2^31 bytes
    assert _form(10, 1, top, 1 << 15, 256) >= 0 and _form(10, 1, top, 1 << 16, 256) == -1
    # 2^30 tiles of 64 rows x 256 columns
    rows, cols = 1 << 30, 1 << 14
    assert _form(rows - 64, 1, 128, cols, 256) >= 0 and _form(rows, 1, 128, cols, 256) == -1


def test_products_refuse_those_sizes():
    """The same limits at the C entries, which look at no device before them."""
    p, top = ctypes.c_void_p(16), 1 << 20
    calls = {
        "hmoe_grouped_gate_up_mxfp4": lambda r, d, f: (p, p, p, 1, r, d, f, p, p, p, p, None),
        "hmoe_grouped_gate_up_mxfp4_gather": lambda r, d, f: (p, p, 64, 1, p, p, 1, r, d, f, p, p, p, p, None),
        "hmoe_grouped_down_mxfp4": lambda r, d, f: (p, p, p, 1, r, f, d, p, p, p, None),
    }
    for name, args in calls.items():
        for sizes, needle in (((10, top, top), "operand too large"), ((1 << 30, 1 << 15, 1 << 15), "too many tiles")):
            rc = getattr(_lib.lib(), name)(*args(*sizes))
            assert rc == _lib.ERR_INVALID and needle in _lib.lib().hmoe_last_error().decode(), name

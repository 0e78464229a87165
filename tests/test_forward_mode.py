"""Forward-mode derivatives of the norm and the layer are refused, before a device is touched."""
import pytest
import torch
from torch.autograd import forward_ad

from hanuman_amd import MoE, RMSNorm

D = 256


def _dual(*shape):
    return forward_ad.make_dual(torch.zeros(shape), torch.ones(shape))


def _layer():
    return MoE(D, 128, 8, 2, 1, 0.02, 1.0, "bfloat16", rngs=0, device="cpu")


def test_the_norm():
    norm = RMSNorm(D, device="cpu")
    plain = torch.zeros((3, D))
    with forward_ad.dual_level():
        for call in (lambda: norm(_dual(3, D)), lambda: norm.with_sum(_dual(3, D), plain),
                     lambda: norm.with_sum(plain, _dual(3, D)), lambda: norm(_dual(3, D).to(torch.bfloat16))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        with pytest.raises(ValueError, match="GPU"):       # nothing to refuse: on to the call
            norm(plain)
        norm.scale.value = _dual(D)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            norm(plain)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(RMSNorm(D, device="cpu"), (plain,), (torch.ones_like(plain),))


def test_the_layer():
    layer, norm = _layer(), RMSNorm(D, device="cpu")
    plain = torch.zeros((1, 4, D))
    with forward_ad.dual_level():
        for call in (lambda: layer(_dual(1, 4, D)), lambda: layer.behind_norm(norm, _dual(1, 4, D)),
                     lambda: layer.behind_norm(norm, plain, _dual(1, 4, D))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        layer.router.value = _dual(D, 8)
        for call in (lambda: layer(plain), lambda: layer.behind_norm(norm, plain)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()

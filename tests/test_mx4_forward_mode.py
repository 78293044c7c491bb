"""The 4-bit operators and the loss have backward derivatives alone: a dual tensor is refused, where its tangent would
have been dropped without a word.  The refusal comes before any look at the device."""
import pytest
import torch
from torch.autograd import forward_ad

import _native
import distill
import mxfp4

BF = torch.bfloat16


def _refused(call):
    with pytest.raises(_native.NativeError, match="forward-mode"):
        call()


def test_dual_logits_are_refused():
    z, idx, t = torch.zeros(4, 64), torch.zeros(4, 1, dtype=torch.int32), torch.zeros(4, 1)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(z, torch.ones_like(z))
        _refused(lambda: distill.topk_kl(d, idx, t))
        _refused(lambda: distill.topk_kl_rows(d, idx, t))
        with pytest.raises(_native.NativeError, match="GPU"):
            distill.topk_kl(z, idx, t)
    with pytest.raises(_native.NativeError, match="GPU"):
        distill.topk_kl(d, idx, t)  # the level has ended: no tangent any more


@pytest.mark.gpu
def test_dual_activations_are_refused(gpu):
    w = torch.zeros(64, 128, dtype=BF, device=gpu)
    W, G = mxfp4.Weight(w), mxfp4.GatedWeight(w, w)
    add = torch.zeros(128, dtype=BF, device=gpu)
    for rows in (1, 40):
        x = torch.zeros(rows, 128, dtype=BF, device=gpu)
        with forward_ad.dual_level():
            d, da = forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(add, torch.ones_like(add))
            _refused(lambda: mxfp4.mx4_linear(d, W))
            _refused(lambda: mxfp4.mx4_gated(d, G))
            _refused(lambda: mxfp4.mx4_gated(x, G, add=da))
            assert mxfp4.mx4_linear(x, W).shape == (rows, 64)

"""The per-step copies of the adapters' weights (fused_linear._cast) belong to the parameters they were made from: a model
built after another one is gone takes none of its copies, whatever object ids come back, also without new_step()."""
import gc
import weakref

import torch

import fused_linear
from test_group_host import _frozen, _lora


def test_models_one_after_the_other_without_a_new_step():
    g = torch.Generator().manual_seed(3)
    K, T = 32, 3
    x = torch.randn(T, K, generator=g)
    for i in range(200):
        n = 128 if i % 3 else 192  # also of another shape
        mods = [_lora(n, K, 8, g), _lora(64, K, 8, g), _frozen(16, K, g)]
        with torch.no_grad():
            got = fused_linear.group_linear(x, mods)
            want = [m(x) for m in mods]
        for a, b in zip(got, want):
            torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-6)
        del mods


def test_adapters_that_share_a_and_not_b():
    g = torch.Generator().manual_seed(4)
    one, two = _lora(128, 32, 8, g), _lora(128, 32, 8, g)
    two.lora_A["default"].weight = one.lora_A["default"].weight
    x = torch.randn(3, 32, generator=g)
    with torch.no_grad():
        for m in (one, two):
            torch.testing.assert_close(fused_linear.group_linear(x, [m])[0], m(x), rtol=1e-5, atol=1e-6)


def test_a_copy_goes_with_its_source_and_stays_with_a_live_one():
    made = []

    def make():
        made.append(torch.zeros(4))
        return made[-1]

    a, b = torch.zeros(3), torch.zeros(3)
    key = ((id(a), id(b)), "copy")
    first = fused_linear._cast(key, make, a, b)
    assert fused_linear._cast(key, make, a, b) is first and len(made) == 1
    kept = weakref.ref(first)
    del first, b
    made.clear()
    gc.collect()
    assert kept() is None and key not in fused_linear._CAST  # nothing left under an id that may come back
    c = torch.zeros(3)
    second = fused_linear._cast(key, make, a, c)
    assert second is made[0]
    fused_linear.new_step()
    third = fused_linear._cast(key, make, a, c)
    del c
    gc.collect()
    assert third is made[1] and key not in fused_linear._CAST

"""enable_mxfp4 and disable_mxfp4 beside the 8-bit switches, on stand-ins of the quantized weights (the quantizer runs on the
GPU alone): each pair undoes its own work only, and a call that fails leaves the model as it was."""
import types

import pytest
import torch

import distill_mxfp4
import mxfp4
import mxfp8


class _Weight:
    def __init__(self, *w):
        self.w = [t.detach().clone() for t in w]


@pytest.fixture
def model(monkeypatch):
    monkeypatch.setattr(mxfp4, "Weight", _Weight)
    monkeypatch.setattr(mxfp4, "GatedWeight", _Weight)
    return distill_mxfp4.Model(2, 64, 96, 32, 8, True)


def _state(model):
    """What the switches may touch: weights, and the attributes of every module."""
    return ({n: p.detach().clone() for n, p in model.named_parameters()},
            {n: {k for k in m.__dict__ if not k.startswith("_parameters")} for n, m in model.named_modules()})


def _same(a, b):
    return a[1] == b[1] and a[0].keys() == b[0].keys() and all(torch.equal(a[0][n], b[0][n]) for n in a[0])


def test_there_and_back(model):
    before = _state(model)
    for _ in range(2):
        assert mxfp4.enable_mxfp4(model) == 6
        assert not _same(_state(model), before)
        mxfp4.disable_mxfp4(model)
        assert _same(_state(model), before)
    mxfp4.disable_mxfp4(model)  # nothing to undo
    assert _same(_state(model), before)


def test_the_eight_bit_switches_leave_four_bit_layers_alone(model):
    before = _state(model)
    mxfp4.enable_mxfp4(model)
    on = _state(model)
    mxfp8.disable_mxfp8(model)
    assert _same(_state(model), on)
    with pytest.raises(ValueError, match="MXFP4"):
        mxfp8.enable_mxfp8(model)
    assert _same(_state(model), on)
    mxfp4.disable_mxfp4(model)
    assert _same(_state(model), before)


def test_the_four_bit_switches_leave_eight_bit_layers_alone(model):
    lin = model.model.layers[0].mlp.down_proj.base_layer
    lin._mx_w, lin._bf16_cpu = torch.zeros(1), torch.zeros(1)  # as enable_mxfp8 marks it
    on = _state(model)
    with pytest.raises(ValueError):
        mxfp4.enable_mxfp4(model)
    mxfp4.disable_mxfp4(model)
    assert _same(_state(model), on)


def test_forwards_patched_before_come_back(model):
    mlp = model.model.layers[0].mlp
    lin = model.model.layers[1].mlp.down_proj.base_layer
    calls = []
    mlp.forward = types.MethodType(lambda self, x: calls.append("mlp") or x, mlp)
    lin.forward = types.MethodType(lambda self, x: calls.append("lin") or x, lin)
    mxfp4.enable_mxfp4(model)
    assert mlp.forward.__func__ is mxfp4.mlp and lin.forward.__func__ is mxfp4._linear_forward
    mxfp4.disable_mxfp4(model)
    mlp(1)
    lin(1)
    assert calls == ["mlp", "lin"]


@pytest.mark.parametrize("fail_at", [0, 1, 2, 3])
def test_a_call_that_fails_leaves_the_model_as_it_was(model, monkeypatch, fail_at):
    """Two MLPs are taken whole; without their act_fn, six linears one by one."""
    if fail_at >= 2:
        for layer in model.model.layers:
            layer.mlp.act_fn = torch.nn.ReLU()
    before, made = _state(model), []

    def weight(*w):
        if len(made) == fail_at:
            raise MemoryError
        made.append(1)
        return _Weight(*w)

    monkeypatch.setattr(mxfp4, "Weight", weight)
    with pytest.raises(MemoryError):
        mxfp4.enable_mxfp4(model)
    assert _same(_state(model), before)

"""bench.py's side figures run their steps as a training program does."""
import pytest

import bench
import fused_linear

pytestmark = pytest.mark.gpu


def test_unfused_mlp_steps_begin_with_new_step(gpu, monkeypatch):
    """Each step casts its adapters' weights anew, after the attention figures of another model too."""
    calls, new_step = [], fused_linear.new_step
    monkeypatch.setattr(fused_linear, "new_step", lambda: (calls.append(1), new_step()))
    bench._grouped_linears(256, 2048, 16, 32, gpu, steps=1)
    calls.clear()
    out = bench._unfused_mlp(256, 2048, 6144, 16, gpu, steps=2)
    assert out["unfused step"]["ms_per_step"] > 0
    assert len(calls) == 5  # three to warm up

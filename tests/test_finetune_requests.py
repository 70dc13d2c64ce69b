"""Requests that fine-tuning refuses on the host, before anything reaches the GPU (CPU)."""
import importlib
from types import SimpleNamespace

import pytest


@pytest.fixture
def engine(jc):
    def forward_trace(*a, **k):
        raise AssertionError("a request that should have been refused reached the engine")
    cfg = jc.default_config(d_model=128, inter=128, n_layers=3, vocab=500, head_ff=128, scorer_hidden=64,
                            max_positions=128)
    return SimpleNamespace(cfg=cfg, forward_trace=forward_trace, head_length=0)


@pytest.mark.parametrize("bad,why", [
    (([3, 500], [0], 0), "token id 500 is past the vocabulary"), (([-1], [0], 0), "token id -1"),
    (([2 ** 32 + 1, 2], [0], 0), "past the vocabulary"), (([1, 2, 3], [0, 3], 0), "a marker is past the sequence"),
    (([1, 2, 3], [-1], 0), "a marker is past the sequence"), (([], [], 0), "no tokens"),
    (([1, 2], [0], 3), "no question type 3"), (([1, 2], [0], -1), "no question type -1")])
def test_features_refuse(jc, engine, bad, why):
    ft = importlib.import_module("julia-cuda_b200.finetune")
    with pytest.raises(jc.JuliaCudaError, match=f"sequence 1: .*{why}"):
        ft.features(engine, [([1, 2, 3], [0, 2], 0), bad])

"""The trainer's sync point asks whether a bounded device wait ran out."""
import pytest
import torch

from vibecheck_nn_b200 import _lib, train


def test_layers_are_not_handed_over_after_a_fault(monkeypatch):
    t = train.MlpTrainer.__new__(train.MlpTrainer)
    t.weights, t.biases = [torch.ones(3, 2)], [torch.zeros(3)]
    asked = []
    monkeypatch.setattr(_lib, 'fault_check', lambda device=None: asked.append(device))
    (W, b), = t.layers()
    assert W.shape == (3, 2) and b.shape == (3,) and asked == [t.weights[0].device]

    def fault(device=None):
        raise TimeoutError('linear layer: a bounded device-side wait expired')
    monkeypatch.setattr(_lib, 'fault_check', fault)
    for call in (t.layers, t.gg):
        with pytest.raises(TimeoutError):
            call()

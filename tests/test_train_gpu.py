"""The training step as a whole against float64, and what is trained bounded.

One step's loss and gradients of a 6 -> [40] x 3 -> 5 network in float32 pass
four products and their gradients, each within 4e-6 of its scale (the linear
layer's tolerance): 5e-5 of a gradient's largest entry covers the chain.
"""
import numpy as np
import pytest
import torch

from vibecheck_nn_b200 import train, workloads as wk

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


def network(dims, seed=0):
    return wk.mlp_params(dims, np.random.default_rng(seed))


def reference(layers, x, y):
    ps = [torch.tensor(a, dtype=torch.float64, requires_grad=True) for l in layers for a in l]
    h = x.double().cpu()
    for i in range(0, len(ps), 2):
        h = h @ ps[i].t() + ps[i + 1]
        if i + 2 < len(ps):
            h = torch.relu(h)
    value = torch.nn.functional.cross_entropy(h, y.cpu())
    value.backward()
    return float(value.detach()), [p.grad for p in ps[::2]] + [p.grad for p in ps[1::2]]


@pytest.mark.parametrize('rows', [1, 33, 700])
def test_one_step_against_float64(rows):
    layers = network((6, 40, 40, 40, 5))
    x, y = train.nearest_centre_data(rows, 6, 5)
    t = train.MlpTrainer(layers)
    value, grads = t.gradients(x, y)
    want, wgrads = reference(layers, x, y)
    assert abs(float(value) - want) <= 1e-5 * max(1.0, want)
    for g, w in zip(grads, wgrads):
        assert float((g.double().cpu() - w).abs().max()) <= 5e-5 * float(w.abs().max())


@pytest.mark.parametrize('dtype,bits', [(torch.float32, 32), (torch.float32, 8),
                                        (torch.bfloat16, 8)])
def test_training_learns_and_the_result_is_bounded(dtype, bits):
    """The loss falls by half, and CROWN's margins hold on points sampled in
    the boxes (up to float32 rounding of an output, 1e-4 here)."""
    x, y = train.nearest_centre_data(2048, 5, 5)
    t = train.MlpTrainer(network((5, 50, 50, 50, 5)), dtype=dtype, lr=2e-3, state_bits=bits, seed=1)
    first = float(t.step(x.to(dtype), y))
    for _ in range(150):
        last = t.step(x.to(dtype), y)
    assert float(last) < 0.5 * first
    eps = 0.02
    m = train.certified(t.gg(), x[:256], y[:256], eps)
    assert m.shape == (256, 5) and bool(torch.isinf(m[torch.arange(256), y[:256]]).all())
    f32 = train.MlpTrainer(t.layers())
    gen = torch.Generator(DEV).manual_seed(0)
    for _ in range(20):
        p = x[:256] + eps * (2 * torch.rand(256, 5, device=DEV, generator=gen) - 1)
        out = f32.logits(p)
        margin = out.gather(1, y[:256, None]) - out
        margin[torch.arange(256), y[:256]] = float('inf')
        assert bool((margin >= m - 1e-4).all())
    assert 0 < int((m > 0).all(1).sum()) < 256


def test_steps_repeat_bit_for_bit():
    x, y = train.nearest_centre_data(512, 6, 5)
    runs = []
    for _ in range(2):
        t = train.MlpTrainer(network((6, 64, 64, 5)), state_bits=8, seed=4)
        losses = [t.step(x, y) for _ in range(5)]
        runs.append((torch.stack(losses), [w.clone() for w in t.weights + t.biases]))
    assert torch.equal(runs[0][0], runs[1][0])
    assert all(torch.equal(a, b) for a, b in zip(runs[0][1], runs[1][1]))

"""The loss under autograd: its gradient is rounded to the logits' type once, after the upstream
factor.

Bounds as for the loss itself (a probability 4e-6 relative, 4e-7 of the factor over the labelled
rows for what cancels at the label) times the factor, plus one rounding of the result and half of
float16's smallest step: none of them is multiplied by the factor afterwards.
"""
import pytest
import torch

from vibecheck_nn_b200 import loss

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
ROUND = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-38, torch.bfloat16: 1e-38, torch.float16: 2.0 ** -25}


def make(R, C, dtype):
    gen = torch.Generator(DEV).manual_seed(R + C)
    x = torch.randn((R, C), device=DEV, generator=gen).to(dtype)
    y = torch.randint(0, C, (R,), device=DEV, generator=gen)
    y[1::7] = -100
    return x, y


def gradient64(x, y, factor):
    x = x.double()
    live = y != -100
    p = torch.softmax(x, 1)
    p[torch.arange(len(y), device=DEV), torch.where(live, y, 0)] -= 1
    return p * live[:, None] * (factor / max(1, int(live.sum())))


# a row in 8 lanes, in a warp, in a warp's vectors, over a cluster; one launch and two
@pytest.mark.parametrize('dtype', list(ROUND))
@pytest.mark.parametrize('R,C', [(20, 10), (3000, 10), (600, 100), (2048, 1000), (50, 4001),
                                 (2048, 20001), (5, 131072)])
@pytest.mark.parametrize('factor', [1.0, 65536.0, 1e-3])
def test_upstream_factor_comes_before_the_rounding(R, C, dtype, factor):
    x, y = make(R, C, dtype)
    leaf = x.clone().requires_grad_(True)
    (loss.cross_entropy(leaf, y) * factor).backward()
    want = gradient64(x, y, factor)
    n = max(1, int((y != -100).sum()))
    err = (leaf.grad.double() - want).abs()
    bound = (4e-6 + ROUND[dtype]) * want.abs() + 4e-7 * factor / n + TINY[dtype]
    assert leaf.grad.dtype == dtype and bool((err <= bound).all()), float((err - bound).max())


def test_loss_scaling_keeps_small_float16_gradients():
    """Off the label entries are about 1 / (R C) = 6e-9, below float16's smallest step: unscaled
    they are 0, scaled by 2^16 none may be."""
    x, y = make(4096, 40000, torch.float16)
    leaf = x.clone().requires_grad_(True)
    (loss.cross_entropy(leaf, y) * 65536).backward()
    live = leaf.grad[y != -100]
    want = gradient64(x, y, 65536.0)[y != -100].float()
    assert float(((live != 0) | (want.abs() < 2.0 ** -25)).float().mean()) == 1.0
    assert abs(float(live.float().abs().sum()) / float(want.abs().sum()) - 1) <= 1e-3


@pytest.mark.parametrize('R,C', [(20, 10), (3000, 10), (40, 129), (50, 4001), (7, 60000)])
def test_value_and_gradient_are_those_of_one_pass(R, C):
    for dtype in ROUND:
        x, y = make(R, C, dtype)
        value, grad = loss.cross_entropy_grad(x, y)
        leaf = x.clone().requires_grad_(True)
        got = loss.cross_entropy(leaf, y)
        got.backward()
        assert torch.equal(got.detach(), value) and torch.equal(leaf.grad, grad)
        assert torch.equal(loss.cross_entropy(x, y), value)


def test_upstream_of_another_stream_and_shape():
    x, y = make(12, 40, torch.bfloat16)
    leaf = x.reshape(3, 4, 40).clone().requires_grad_(True)
    value = loss.cross_entropy(leaf, y.reshape(3, 4))
    factor = torch.tensor(0.5, device=DEV, requires_grad=True)
    (value * factor).backward()
    assert leaf.grad.shape == leaf.shape and torch.equal(factor.grad, value.detach())
    want = gradient64(x, y, 0.5)
    assert float((leaf.grad.reshape(12, 40).double() - want).abs().max()) <= 2.0 ** -8 / 10

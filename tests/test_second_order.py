"""Second derivatives through the training-step operators: their gradients are made by kernels
that autograd does not see, so asking for a graph through them has to fail, not drop terms."""
import pytest
import torch

from vibecheck_nn_b200 import linear, loss


@pytest.fixture
def on_the_host(monkeypatch):
    """The operators' kernels replaced by detached products of CPU tensors."""
    def forward(x, w, b=None, act='none', residual=None, keep=False):
        z = x.detach() @ w.detach().t()
        return (z, z) if keep else z

    def backward(dy, x, w, z=None, act='none', bias=True, need=(True, True)):
        dy, x, w = dy.detach(), x.detach(), w.detach()
        return dy @ w, dy.t() @ x, dy.sum(0) if bias else None

    def value_and_gradient(x, y, ignore_index, scale=None, want_loss=True, want_grad=True):
        x = x.detach()
        p = torch.softmax(x, 1)
        p[torch.arange(len(y)), y] -= 1
        return torch.nn.functional.cross_entropy(x, y), p / len(y) * (1 if scale is None else scale)

    monkeypatch.setattr(linear, 'linear_forward', forward)
    monkeypatch.setattr(linear, 'linear_backward', backward)
    monkeypatch.setattr(loss, '_run', value_and_gradient)


def penalties():
    x = torch.randn(4, 6, requires_grad=True)
    w = torch.randn(5, 6, requires_grad=True)
    y = torch.randint(0, 5, (4,))
    return (x, w), (lambda: linear.linear(x, w, None, 'gelu').square().sum(),
                    lambda: loss.cross_entropy(x @ w.t(), y),
                    lambda: linear.linear(x, w).sum())  # an upstream that is constant


@pytest.mark.parametrize('k', [0, 1, 2])
def test_double_backward_is_refused(on_the_host, k):
    torch.manual_seed(0)
    (x, w), values = penalties()
    value = values[k]()
    gx, = torch.autograd.grad(value, x, create_graph=True)
    with pytest.raises(RuntimeError, match='differentiable once'):
        (value + gx.square().sum()).backward()


@pytest.mark.parametrize('k', [0, 1, 2])
def test_one_backward_works(on_the_host, k):
    torch.manual_seed(0)
    (x, w), values = penalties()
    values[k]().backward()
    assert x.grad is not None and w.grad is not None and bool(x.grad.any())


@pytest.mark.parametrize('k', [0, 1, 2])
def test_a_graph_that_is_not_used_does_no_harm(on_the_host, k):
    torch.manual_seed(0)
    (x, w), values = penalties()
    want, = torch.autograd.grad(values[k](), x)
    got, = torch.autograd.grad(values[k](), x, create_graph=True)
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_on_the_gpu(dtype):
    gen = torch.Generator('cuda').manual_seed(0)
    x = torch.randn(40, 64, device='cuda', generator=gen).to(dtype).requires_grad_(True)
    w = torch.randn(32, 64, device='cuda', generator=gen).to(dtype).requires_grad_(True)
    y = torch.randint(0, 32, (40,), device='cuda', generator=gen)
    for value in (lambda: linear.linear(x, w, None, 'silu').float().square().sum(),
                  lambda: loss.cross_entropy(x @ w.t(), y)):
        want, = torch.autograd.grad(value(), x)
        got, = torch.autograd.grad(value(), x, create_graph=True)
        assert torch.equal(got, want)
        with pytest.raises(RuntimeError, match='differentiable once'):
            got.float().square().sum().backward()
    r = torch.randn(40, 32, device='cuda', generator=gen).to(dtype).requires_grad_(True)
    g, = torch.autograd.grad(linear.linear(x, w, residual=r).float().square().sum(), r,
                             create_graph=True)
    assert g.requires_grad  # the residual's gradient is the upstream's, to any order

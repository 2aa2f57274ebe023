"""AdamW's host side with launches recorded instead of made: what a step checks of its
parameters, and which launches it makes."""
import types

import pytest
import torch

from vibecheck_nn_b200 import _lib, linear, optim


@pytest.fixture
def host_adamw(monkeypatch):
    """An optimiser of CPU tensors whose launches are recorded, not made."""
    made = []
    monkeypatch.setattr(optim, 'type_of', lambda t, name: linear.TYPES[t.dtype])
    monkeypatch.setattr(_lib, 'launch', lambda *args: made.append(args) or 0)

    def build(*params, **kw):
        opt = optim.AdamW(params, **kw)
        opt.device = types.SimpleNamespace(index=-1)  # what get_device() says of a CPU tensor
        return opt
    return build, made


@pytest.mark.parametrize('first,then', [(torch.float32, torch.float16), (torch.bfloat16, torch.float32),
                                        (torch.float16, torch.bfloat16)])
def test_adamw_refuses_parameters_of_another_type_than_at_its_construction(host_adamw, first, then):
    build, made = host_adamw
    p = torch.nn.Parameter(torch.ones(6, dtype=first))
    opt = build(p)
    p.data = p.data.to(then)  # what module.half() and the like do
    for g in (torch.ones(6), torch.ones(6, dtype=first), torch.ones(6, dtype=then)):
        with pytest.raises(ValueError):
            opt.step([g])
    assert not made and opt.t == 0
    p.data = p.data.to(first)
    opt.step([torch.ones(6, dtype=first)])
    assert len(made) == 1 and opt.t == 1


def test_adamw_refuses_parameters_that_changed_their_layout_or_size(host_adamw):
    build, made = host_adamw
    for data in (torch.ones(4, 4).t().contiguous().t(), torch.ones(4, 4, dtype=torch.float32)[:, :2],
                 torch.ones(2, 8), torch.ones(1, 1).expand(4, 4), torch.ones(0)):
        p, q = (torch.nn.Parameter(torch.ones(4, 4)) for _ in range(2))
        opt = build(p, q)
        q.data = data
        for grads in ([torch.ones(4, 4)] * 2, [None, torch.ones(4, 4)], [None, torch.ones(data.shape)]):
            with pytest.raises(ValueError):
                opt.step(grads)
        assert not made and opt.t == 0


@pytest.mark.gpu
def test_adamw_refuses_parameters_converted_on_the_gpu():
    layer = torch.nn.Linear(30, 20).cuda()
    opt = optim.AdamW(layer.parameters())
    grads = [torch.ones_like(p) for p in layer.parameters()]
    opt.step(grads)
    before = [p.detach().clone() for p in layer.parameters()]
    for change in (layer.half, layer.bfloat16, layer.cpu):
        change()
        with pytest.raises(ValueError):
            opt.step(grads)
        layer.float().cuda()
        for p, b in zip(layer.parameters(), before):
            p.data.copy_(b)
    opt.step(grads)
    assert opt.t == 2 and all(bool((p < b).all()) for p, b in zip(layer.parameters(), before))

"""AdamW's host side with launches recorded instead of made: what a step checks of its
parameters, and which launches it makes."""
import ctypes
import types

import pytest
import torch

from vibecheck_nn_b200 import _lib, linear, optim


@pytest.fixture
def host_adamw(monkeypatch):
    """An optimiser of CPU tensors whose launches are recorded, not made."""
    made = []
    monkeypatch.setattr(optim, 'type_of', lambda t, name: linear.TYPES[t.dtype])
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: False)
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


def test_bias_corrections_count_each_parameters_own_steps(host_adamw):
    build, made = host_adamw
    opt = build(*(torch.ones(4) for _ in range(3)), lr=1e-3, betas=(0.9, 0.99))
    g = torch.ones(4)
    for _ in range(100):
        opt.step([g, None, g])
    del made[:]
    opt.step([g, g, g])
    f32 = lambda x: ctypes.c_float(x).value  # noqa: E731
    sizes = {a[2]: a[-1]._obj.size for a in made}  # tensors of the launch -> lr / (1 - b1^t)
    assert sizes == {2: f32(1e-3 / (1 - 0.9 ** 101)), 1: f32(1e-3 / (1 - 0.9))}
    roots = {a[2]: a[-1]._obj.root for a in made}
    assert roots == {2: f32((1 - 0.99 ** 101) ** -0.5), 1: f32((1 - 0.99) ** -0.5)}


def test_equal_counts_make_one_launch(host_adamw):
    build, made = host_adamw
    opt = build(*(torch.ones(4) for _ in range(3)))
    g = torch.ones(4)
    opt.step([g, g, g])
    opt.step([None, None, None])  # nothing to do, nothing counted
    opt.step([g, None, g])
    opt.step([None, g, None])
    opt.step([g, g, g])
    assert [a[2] for a in made] == [3, 2, 1, 3] and opt.t == 5


def test_counts_travel_with_the_state(host_adamw):
    build, made = host_adamw
    opt, other = (build(torch.ones(4), torch.ones(4)) for _ in range(2))
    g = torch.ones(4)
    for _ in range(5):
        opt.step([g, None])
    state = opt.state_dict()
    other.load_state_dict(state)
    del made[:]
    other.step([g, g])
    assert len(made) == 2 and other.t == 6
    del state['steps']  # a state of one count
    other.load_state_dict(state)
    del made[:]
    other.step([g, g])
    assert len(made) == 1
    with pytest.raises(ValueError):
        other.load_state_dict({**state, 'steps': [1]})


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


@pytest.mark.gpu
@pytest.mark.parametrize('bits', [32, 8])
def test_a_parameter_that_starts_late_steps_as_torch_would(bits):
    """First steps are about lr long whenever they come; float32 moments agree with
    torch.optim.AdamW to a few roundings (1e-6 of a weight or a step)."""
    gen = torch.Generator('cuda').manual_seed(1)
    ps = [torch.randn(300, device='cuda', generator=gen) for _ in range(2)]
    qs = [p.clone().requires_grad_(True) for p in ps]
    hyper = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01)
    opt, ref = optim.AdamW(ps, state_bits=bits, **hyper), torch.optim.AdamW(qs, **hyper)
    for step in range(60):
        grads = [torch.randn(300, device='cuda', generator=gen) for _ in range(2)]
        if step < 50:
            grads[1] = None
        before = ps[1].clone()
        opt.step(list(grads))
        for q, g in zip(qs, grads):
            q.grad = g
        ref.step()
        if step == 50:
            moved = (ps[1] - before * (1 - 1e-4)).abs()
            assert float((moved - 1e-2).abs().max()) <= 1e-6
        if bits == 32:
            for p, q in zip(ps, qs):
                assert float((p - q.detach()).abs().max()) <= 1e-6 * (step + 1) * 4


def test_adamw_refuses_to_be_captured(host_adamw, monkeypatch):
    build, made = host_adamw
    opt = build(torch.ones(4))
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: True)
    with pytest.raises(RuntimeError, match='captured'):
        opt.step([torch.ones(4)])
    assert not made and opt.t == 0

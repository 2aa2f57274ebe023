"""The training-step operators in CUDA graphs: a replay computes what the calls compute."""
import pytest
import torch

from vibecheck_nn_b200 import linear, loss, optim

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


# few rows, the FP32 units, the tensor cores with the contraction cut, unaligned and in pairs
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('M,N,K', [(1, 512, 300), (100, 256, 784), (600, 640, 512), (300, 1001, 301),
                                   (2048, 2048, 2048), (12_000, 512, 100)])
def test_replay_of_a_training_pass(M, N, K, dtype):
    gen = torch.Generator(DEV).manual_seed(1)
    new = lambda *s: torch.randn(s, device=DEV, generator=gen).to(dtype)  # noqa: E731
    x, w, b = new(M, K), new(N, K) * K ** -0.5, new(N)
    labels = torch.randint(0, N, (M,), device=DEV, generator=gen)

    def step():
        y, z = linear.linear_forward(x, w, b, 'gelu', keep=True)
        value, dy = loss.cross_entropy_grad(y, labels)
        return [y, z, value, dy, *linear.linear_backward(dy, x, w, z, 'gelu')]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        x.copy_(new(M, K))
        labels.copy_(torch.randint(0, N, (M,), device=DEV, generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, step()):
            assert torch.equal(got, want)


def test_an_optimiser_step_is_not_captured():
    """Its constants go by the step count on the host: a replay would repeat one step's."""
    p = torch.ones(300, device=DEV)
    opt = optim.AdamW([p])
    g = torch.ones_like(p)
    opt.step([g])
    before = p.clone()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match='captured'):
        with torch.cuda.graph(graph):
            opt.step([g])
    torch.cuda.synchronize()
    assert opt.t == 1 and torch.equal(p, before)
    opt.step([g])
    assert opt.t == 2

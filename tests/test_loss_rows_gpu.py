"""Rows of logits that the other tests do not hold: longer than a cluster's shared memory, and cut
out of padded rows.  Bounds as in the tests of the loss (a probability 4e-6 relative, 4e-7 over the
labelled rows at the label, one rounding of a 16-bit gradient)."""
import pytest
import torch

from vibecheck_nn_b200 import loss

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
ROUND = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-38, torch.bfloat16: 1e-38, torch.float16: 2.0 ** -25}


def check(x, y):
    value, grad = loss.cross_entropy_grad(x, y)
    live = y != -100
    n = max(1, int(live.sum()))
    total = 0.0
    for r in range(x.shape[0]):
        row = x[r].double()
        if not live[r]:
            assert not bool(grad[r].any())
            continue
        lse = torch.logsumexp(row, 0)
        total += float(lse - row[y[r]])
        p = torch.exp(row - lse)
        p[y[r]] -= 1
        want = p / n
        err = (grad[r].double() - want).abs()
        bound = (4e-6 + ROUND[x.dtype]) * want.abs() + 4e-7 / n + TINY[x.dtype]
        assert bool((err <= bound).all()), float((err - bound).max())
    assert abs(float(value) - total / n) <= 4e-6 * max(1.0, abs(total / n))


# a cluster holds 8 x 216 KB: 442,368 float32 or 884,736 16-bit logits
@pytest.mark.parametrize('dtype,C', [(torch.float32, 442_368), (torch.float32, 442_369),
                                     (torch.float32, 700_001), (torch.bfloat16, 884_736),
                                     (torch.bfloat16, 884_745), (torch.float16, 1_300_003)])
@pytest.mark.parametrize('pad', [0, 3])
def test_rows_longer_than_a_cluster_can_stage(C, dtype, pad):
    gen = torch.Generator(DEV).manual_seed(C)
    x = (torch.randn((5, C + pad), device=DEV, generator=gen) * 2).to(dtype)[:, :C]
    y = torch.tensor([0, C - 1, -100, C // 2, 12345], device=DEV)
    x[3, C // 3:C // 2] = float('-inf')
    x[4, :] = torch.finfo(dtype).min
    x[4, 12345] = 1.0
    check(x, y)
    x[1] = float('-inf')  # a row without any class
    value, grad = loss.cross_entropy_grad(x, y)
    assert float(value) == float('inf') and not bool(grad[1].any())
    assert bool(torch.isfinite(grad).all())


@pytest.mark.parametrize('dtype', list(ROUND))
@pytest.mark.parametrize('C,width', [(10, 16), (100, 128), (1000, 1024), (3999, 4096), (50_257, 50_304)])
def test_logits_cut_out_of_padded_rows(C, width, dtype):
    gen = torch.Generator(DEV).manual_seed(C)
    whole = torch.full((20, width), float('nan'), device=DEV).to(dtype)
    whole[:, :C] = torch.randn((20, C), device=DEV, generator=gen).to(dtype)
    y = torch.randint(0, C, (20,), device=DEV, generator=gen)
    y[3] = -100
    check(whole[:, :C], y)
    assert bool(torch.isnan(whole[:, C:]).all())

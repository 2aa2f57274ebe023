"""Cross-entropy and its gradient against the definition in float64.

A softmax probability comes from a difference of logits times log2(e) in
float32 (relative error 2^-24 times that exponent, here below 40) and one
exponential (2^-22): 4e-6 relative; the loss is a float32 logarithm of a
float32 sum, 4e-6 of its size.  16-bit gradients add one rounding (and
float16's smallest step).
"""
import pytest
import torch

from vibecheck_nn_b200 import _lib, loss

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
ROUND = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-38, torch.bfloat16: 1e-38, torch.float16: 2.0 ** -25}


def definition(x, y, ignore=-100):
    x = x.double()
    # relative to the row's largest logit: beside 3e38 float64 has no place for log C
    top = x.amax(1, keepdim=True)
    x = x - torch.where(torch.isinf(top), torch.zeros_like(top), top)
    live = y != ignore
    n = max(1, int(live.sum()))
    lse = torch.logsumexp(x, 1)
    at = torch.where(live, y, torch.zeros_like(y))[:, None]
    rows = torch.where(torch.isinf(lse) & (lse < 0), torch.full_like(lse, float('inf')),
                       lse - x.gather(1, at)[:, 0])
    empty = (lse == float('-inf'))[:, None]
    p = torch.where(empty, torch.zeros_like(x), torch.exp(x - lse[:, None]))
    p = p - torch.where(empty, 0.0, 1.0) * torch.zeros_like(x).scatter_(1, at, 1.0)
    return float(rows[live].sum()) / n, p * live[:, None] / n


def check(x, y, ignore=-100):
    got, grad = loss.cross_entropy_grad(x, y, ignore)
    want, wgrad = definition(x, y, ignore)
    assert got.dtype == torch.float32 and grad.dtype == x.dtype and grad.shape == x.shape
    if want == float('inf'):
        assert float(got) == want
    else:
        assert abs(float(got) - want) <= 4e-6 * max(1.0, abs(want)), (float(got), want)
    n = max(1, int((y != ignore).sum()))
    err = (grad.double() - wgrad).abs()
    bound = (4e-6 + ROUND[x.dtype]) * wgrad.abs() + 4e-7 / n + TINY[x.dtype]
    assert bool((err <= bound).all()), float((err - bound).max())


def make(R, C, dtype, pad=0, scale=2.0, ignored=0.2, seed=0):
    gen = torch.Generator(DEV).manual_seed(seed + R + C)
    x = (torch.randn((R, C + pad), device=DEV, generator=gen) * scale).to(dtype)[:, :C]
    y = torch.randint(0, C, (R,), device=DEV, generator=gen)
    y[torch.rand(R, device=DEV, generator=gen) < ignored] = -100
    return x, y


@pytest.mark.parametrize('dtype', list(ROUND))
@pytest.mark.parametrize('R,C', [(1, 1), (1, 2), (3, 10), (65, 31), (300, 32), (40, 33), (7, 128),
                                 (33, 129), (9, 1000), (5, 1024), (4, 1025), (6, 4099), (3, 50001),
                                 (2, 131072), (2, 300007), (5000, 10)])
def test_against_definition(R, C, dtype):
    for pad in (0, 3, 8):
        check(*make(R, C, dtype, pad))


@pytest.mark.parametrize('C', [10, 900, 5001, 40000])
def test_masked_logits_empty_rows_and_extremes(C):
    for dtype in ROUND:
        x, y = make(12, C, dtype, ignored=0.0)
        x = x.clone()
        x[0] = float('-inf')                       # nothing left: loss inf, gradient 0
        assert float(loss.cross_entropy_grad(x, y)[0]) == float('inf')
        check(x, y)
        y[0] = -100                                # ... unless the row is ignored
        x[1, C // 2:] = float('-inf')
        y[1] = 0
        x[2] = torch.finfo(dtype).min              # all at the lowest value: uniform
        x[3, 1:] = torch.finfo(dtype).min          # one logit left
        y[3] = 0
        x[4] = 100.0 + x[4]
        check(x, y)
        x[5, 1] = float('nan')
        y[5] = 0
        got, grad = loss.cross_entropy_grad(x, y)
        assert bool(torch.isnan(got)) and bool(torch.isnan(grad[5]).all())
        assert bool(torch.isfinite(grad[6:]).all()) and not grad[0].any()


@pytest.mark.parametrize('C', [10, 2000])
def test_labels(C):
    x, y = make(20, C, torch.float32)
    all_out = torch.full_like(y, -100)
    got, grad = loss.cross_entropy_grad(x, all_out)
    assert float(got) == 0.0 and not grad.any()
    check(x, torch.where(y == -100, 7, y), ignore=7)
    for bad in (C, -1, -2 ** 62, 2 ** 40):
        y2 = y.clone()
        y2[3] = bad
        got, grad = loss.cross_entropy_grad(x, y2)
        assert bool(torch.isnan(got)) and bool(torch.isnan(grad[3]).all())
        rest = torch.arange(20, device=DEV) != 3
        assert bool(torch.isfinite(grad[rest]).all())


def test_no_rows_and_leading_axes():
    got, grad = loss.cross_entropy_grad(torch.empty(0, 5, device=DEV),
                                        torch.empty(0, dtype=torch.int64, device=DEV))
    assert float(got) == 0.0 and grad.shape == (0, 5)
    x, y = make(12, 40, torch.bfloat16)
    a, ga = loss.cross_entropy_grad(x, y)
    b, gb = loss.cross_entropy_grad(x.reshape(3, 4, 40), y.reshape(3, 4))
    assert torch.equal(a, b) and torch.equal(ga, gb.reshape(12, 40))


def test_gradient_is_the_slope_of_the_loss():
    """Differences at h = 1e-2: the loss's float32 error 4e-6 / 2h and the
    third derivative's h^2 keep below 1e-3."""
    for C in (20, 3000):
        x, y = make(16, C, torch.float32)
        x = x.clone().requires_grad_(True)
        (3 * loss.cross_entropy(x, y)).backward()
        gen = torch.Generator(DEV).manual_seed(1)
        d = torch.randn(x.shape, device=DEV, generator=gen)
        h = 1e-2
        up, dn = (float(loss.cross_entropy_grad(x.detach() + s * h * d, y)[0]) for s in (1, -1))
        an = float((x.grad.double() * d).sum())
        assert abs(3 * (up - dn) / (2 * h) - an) <= 3e-3 * max(1.0, abs(an))


def test_repeats_bit_for_bit_on_another_stream():
    x, y = make(500, 7001, torch.bfloat16)
    a = loss.cross_entropy_grad(x, y)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        b = loss.cross_entropy_grad(x, y)
    s.synchronize()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_refusals():
    x, y = torch.ones(2, 4, device=DEV), torch.zeros(2, dtype=torch.int64, device=DEV)
    with pytest.raises(_lib.UnsupportedInput):
        loss.cross_entropy_grad(x.cpu(), y.cpu())
    with pytest.raises(_lib.UnsupportedInput):
        loss.cross_entropy_grad(x.double(), y)
    for bad in (lambda: loss.cross_entropy_grad(x, y.int()), lambda: loss.cross_entropy_grad(x, y[:1]),
                lambda: loss.cross_entropy_grad(x, y.cpu()),
                lambda: loss.cross_entropy_grad(x[:, :0], y)):
        with pytest.raises(ValueError):
            bad()
    lib = _lib.lib()
    p = x.data_ptr()
    assert lib.vcb_cross_entropy(300, 4, 0, p, 4, y.data_ptr(), -100, p, p, 4, None, 0, None) \
        == _lib.VCB_ERR_INVALID
    assert lib.vcb_cross_entropy(2, 4, 0, p, 3, y.data_ptr(), -100, p, p, 4, p, 1 << 20, None) \
        == _lib.VCB_ERR_INVALID

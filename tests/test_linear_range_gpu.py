"""Float32 products whose rows hold entries of very different size.

Bound.  An output sum_k x_k w_k in float32 errs in proportion to its own sum_k |x_k w_k|: every
product may lose 2^-24 of itself, and K additions in float32 lose 2^-24 sqrt(K) of their size
typically, whatever their order; 2^-19 is 32 such roundings (K = 1024).  Entries below 2^-110 may
be held to 2^-134 apart.  Rows' norms do not enter: an entry that meets a zero costs nothing.
"""
import pytest
import torch

from vibecheck_nn_b200 import _lib, linear

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
LARGEST = torch.finfo(torch.float32).max

# few rows, the FP32 units, the tensor cores with the contraction cut and in pairs
SIZES = [(4, 300, 512), (40, 130, 1024), (600, 640, 512), (1024, 1000, 250), (2048, 2048, 1024)]


def within(got, a, b, absolute=0.0):
    """got ~ a b^T entry by entry, in float64."""
    a, b = a.double(), b.double()
    err = (got.double() - a @ b.t()).abs()
    bound = 2.0 ** -19 * (a.abs() @ b.abs().t()) + absolute
    assert bool(torch.isfinite(got).all()) and bool((err <= bound).all()), \
        float((err / bound).max())


def rand(gen, *shape):
    return torch.randn(shape, device=DEV, generator=gen)


@pytest.mark.parametrize('M,N,K', SIZES)
@pytest.mark.parametrize('size', [2.0 ** 20, 2.0 ** 30, 1.7e12, 2.0 ** 60])
def test_one_large_column(M, N, K, size):
    """An unscaled feature beside ordinary ones, with a weight of 0 and with its reciprocal."""
    gen = torch.Generator(DEV).manual_seed(1)
    x, w = rand(gen, M, K), rand(gen, N, K)
    x[:, 0] *= size
    w[::2, 0] = 0
    w[1::2, 0] /= size
    within(linear.linear_forward(x, w), x, w)
    dy = rand(gen, M, N)
    dx, dw, db = linear.linear_backward(dy, x, w)
    within(dx, dy, w.t())
    within(dw, dy.t(), x.t())


@pytest.mark.parametrize('M,N,K', SIZES)
def test_one_token_with_large_gradients(M, N, K):
    """Half of the features are off in that token: their weights' gradients come from the others."""
    gen = torch.Generator(DEV).manual_seed(2)
    x, w, dy, z = rand(gen, M, K), rand(gen, N, K), rand(gen, M, N), rand(gen, M, N)
    dy[M // 2] *= 2.0 ** 35
    x[M // 2, ::2] = 0
    dx, dw, db = linear.linear_backward(dy, x, w, z, 'relu')
    dz = torch.where(z > 0, dy, 0.0)
    within(dx, dz, w.t())
    within(dw, dz.t(), x.t())
    within(db[:, None], dz.t(), torch.ones(1, M, device=DEV))


@pytest.mark.parametrize('M,N,K', SIZES)
def test_the_ends_of_the_range(M, N, K):
    gen = torch.Generator(DEV).manual_seed(3)
    x, w = rand(gen, M, K), rand(gen, N, K)
    x[1], w[:, 1] = x[1].abs(), w[:, 1].abs()
    x[:, 0], w[:, 0] = -LARGEST, 0          # a mask of the lowest value that meets nothing
    x[0, 1:], w[3, 0] = 0, 1                # ... and one that is handed through
    x[2, 0], w[3, 1:] = LARGEST, 0
    y = linear.linear_forward(x, w)
    within(y, x, w)
    assert float(y[0, 3]) == -LARGEST and float(y[2, 3]) == LARGEST
    x, w = rand(gen, M, K) * 1e-30, rand(gen, N, K) * torch.logspace(-6, 30, K, device=DEV)
    within(linear.linear_forward(x, w), x, w, 2.0 ** -133 * float(w.double().abs().sum(1).max()))
    x, w = rand(gen, M, K) * 1e-37, rand(gen, N, K)
    within(linear.linear_forward(x, w), x, w, 2.0 ** -133 * float(w.double().abs().sum(1).max()))


@pytest.mark.parametrize('M,N,K', SIZES)
def test_every_bit_of_an_entry_counts(M, N, K):
    """One product per output: the result is the float32 product to one rounding or so."""
    gen = torch.Generator(DEV).manual_seed(4)
    x, w = torch.zeros(M, K, device=DEV), torch.zeros(N, K, device=DEV)
    at = torch.arange(M, device=DEV) % K
    x[torch.arange(M, device=DEV), at] = rand(gen, M)
    w[:] = rand(gen, N, K)
    y = linear.linear_forward(x, w)
    want = x.double() @ w.double().t()
    assert bool(((y.double() - want).abs() <= 2.0 ** -22 * want.abs()).all())


def test_not_finite_entries_stay_in_their_rows():
    gen = torch.Generator(DEV).manual_seed(5)
    for M, N, K in SIZES:
        x, w = rand(gen, M, K), rand(gen, N, K)
        x[1, 2], x[2, 1], w[5, 0] = float('nan'), float('inf'), float('-inf')
        bad = ~torch.isfinite(linear.linear_forward(x, w))
        assert bool(bad[1].all()) and bool(bad[2].all()) and bool(bad[:, 5].all())
        bad[1], bad[2], bad[:, 5] = False, False, False
        assert not bool(bad.any())
    _lib.fault_check()

"""Millions of rows through the linear layer: points of a small network come in such numbers.

Tolerance.  db and dW sum M terms: a float32 sum of random signs errs by some 2^-24 sqrt(M) of
the terms' size, 1e-4 of an entry of order sqrt(M) at most; 1e-5 of the largest entry is allowed,
the rest as for few rows (4e-6)."""
import pytest
import torch

from vibecheck_nn_b200 import _lib, linear

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


@pytest.mark.parametrize('M,N,K', [(2_200_000, 50, 5), (2_097_121, 5, 50), (40, 2_200_003, 3)])
def test_float32_backward(M, N, K):
    gen = torch.Generator(DEV).manual_seed(1)
    x, w, dy, z = (torch.randn(s, device=DEV, generator=gen) for s in ((M, K), (N, K), (M, N), (M, N)))
    dx, dw, db = linear.linear_backward(dy, x, w, z, 'relu')
    dz = torch.where(z > 0, dy, 0.0).double()
    for got, want, tol in ((dx, dz @ w.double(), 4e-6), (dw, dz.t() @ x.double(), 1e-5),
                           (db, dz.sum(0), 1e-5)):
        assert got.shape == want.shape
        assert float((got.double() - want).abs().max()) <= tol * float(want.abs().max())
    _lib.fault_check()

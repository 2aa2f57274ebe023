"""Long contractions of one sign in 16 bits: the sum may not drift.

The tensor cores cut low-order bits in every accumulation.  An accumulator takes 8,192 entries,
512 accumulations, each of which loses at most 2^-23 of what has been summed so far, half of it
on average: 2^-14 of the result at most.  With the float32 sums of those parts 2^-13 is allowed
beside the one rounding of the output (2^-11 float16, 2^-8 bfloat16).
"""
import pytest
import torch

from vibecheck_nn_b200 import _lib, linear

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def positive(gen, rows, cols, terms, dtype, pad=0):
    """Entries of 0.5 to 1.5 times what makes a sum of squares of `terms` of them 8 or so."""
    t = (torch.rand((rows, cols + pad), device=DEV, generator=gen) + 0.5) * (8.0 / terms) ** 0.5
    return t.to(dtype)[:, :cols]


def product64(a, b):
    """a^T b over many rows."""
    out = torch.zeros(a.shape[1], b.shape[1], dtype=torch.float64, device=DEV)
    for i in range(0, a.shape[0], 65536):
        out += a[i:i + 65536].double().t() @ b[i:i + 65536].double()
    return out


def within(got, want):
    rel = (got.double() - want).abs() / want.abs()
    assert float(rel.max()) <= HALF[got.dtype] + 2.0 ** -13, float(rel.max())


# dW sums over the rows: cut over a cluster and not, in pairs, rows that TMA cannot read
@pytest.mark.parametrize('dtype', list(HALF))
@pytest.mark.parametrize('M,N,K,pad', [(8192, 512, 512, 0), (12_000, 2048, 1500, 0),
                                       (40_000, 1100, 1030, 0), (131_072, 64, 64, 0),
                                       (131_072, 2048, 2048, 0), (70_001, 131, 67, 3),
                                       (1_048_576, 200, 64, 0)])
def test_weight_gradients(M, N, K, pad, dtype):
    gen = torch.Generator(DEV).manual_seed(1)
    dy, x = positive(gen, M, N, M, dtype, pad), positive(gen, M, K, M, dtype, pad)
    w = torch.zeros(N, K, device=DEV, dtype=dtype)
    for need in ((False, True), (True, True)):
        dx, dw, db = linear.linear_backward(dy, x, w, None, 'none', True, need)
        within(dw, product64(dy, x))
        assert dx is None or not bool(dx.any())
    within(db[:, None], product64(dy, torch.ones(M, 1, device=DEV)))
    _lib.fault_check()


@pytest.mark.parametrize('dtype', list(HALF))
@pytest.mark.parametrize('M,N,K,pad', [(300, 260, 100_000, 0), (2048, 1999, 20_000, 0),
                                       (50, 1000, 70_001, 1), (2304, 2304, 9_000, 0)])
def test_forward_with_its_epilogue(M, N, K, pad, dtype):
    gen = torch.Generator(DEV).manual_seed(2)
    x, w = positive(gen, M, K, K, dtype, pad), positive(gen, N, K, K, dtype, pad)
    b, r = positive(gen, 1, N, 8, dtype)[0], positive(gen, M, N, 8, dtype, pad)
    z = product64(x.t(), w.t()) + b.double()
    for act in ('relu', 'silu'):
        got, gz = linear.linear_forward(x, w, b, act, r, keep=True)
        within(gz, z)
        within(got, (z if act == 'relu' else z * torch.sigmoid(z)) + r.double())
    _lib.fault_check()


@pytest.mark.parametrize('dtype', list(HALF))
@pytest.mark.parametrize('M,N,K', [(200, 100_000, 180), (2048, 20_000, 2048), (9_000, 9_500, 600)])
def test_input_gradients(M, N, K, dtype):
    """dX sums over the outputs; at 9,000 rows both contractions are long."""
    gen = torch.Generator(DEV).manual_seed(3)
    dy, w = positive(gen, M, N, N, dtype), positive(gen, N, K, N, dtype)
    x = positive(gen, M, K, N, dtype)
    want = product64(dy.t(), w)
    for need in ((True, False), (True, True)):
        dx, dw, _ = linear.linear_backward(dy, x, w, None, 'none', False, need)
        within(dx, want)
    z = torch.ones(M, N, device=DEV, dtype=dtype)
    dx, _, _ = linear.linear_backward(dy, x, w, z, 'relu')
    within(dx, want)
    _lib.fault_check()


@pytest.mark.parametrize('dtype', list(HALF))
def test_the_sizes_above_reach_what_they_mean(dtype):
    t = linear.TYPES[dtype]
    path = lambda M, N, K, product, aligned=1: \
        _lib.lib().vcb_linear_path(M, N, K, t, product, 0, aligned)  # noqa: E731
    cut, pairs = 4, 5
    assert path(8192, 512, 512, 2) < cut  # the longest of one accumulator
    assert path(131_072, 64, 64, 2) == cut and path(1_048_576, 200, 64, 2) == cut
    assert path(12_000, 2048, 1500, 2) in (cut, pairs) and path(131_072, 2048, 2048, 2) == pairs
    assert path(70_001, 131, 67, 2, 0) == cut
    assert path(300, 260, 100_000, 0) == cut and path(2048, 1999, 20_000, 0) == pairs
    assert path(200, 100_000, 180, 1) == cut and path(2048, 20_000, 2048, 1) == pairs
    assert path(9_000, 9_500, 600, 1) >= cut and path(9_000, 9_500, 600, 2) >= cut

"""The kernels of the large products: CTA pairs, persistent over several tiles.

What each case means to reach is asserted (``vcb_linear_path``).  Tolerances are those of the
smaller products: 4e-6 of the largest output in float32 (a few 2^-24 sqrt(K) of the rows' norms),
one rounding of the output in 16 bits, one more for dz behind an activation.
"""
import pytest
import torch

from vibecheck_nn_b200 import _lib, linear

gpu = pytest.mark.gpu
DEV = 'cuda:0'
TOL = {torch.float32: 4e-6, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
PAIRS = 3

# one tile per pair; ragged tiles, rows that TMA cannot read (16 bits) and, a row further, that it
# can; two rounds of one stage or two; three tiles and more per pair, so that rings wrap between
# tiles and accumulators are used again
FORWARD = [(2048, 2048, 2048), (2047, 2050, 1999), (2047, 2050, 2000), (6061, 3731, 72),
           (4096, 4096, 4096), (4100, 4600, 1000)]
BACKWARD = [(2048, 2048, 2048), (2047, 2050, 1999), (2047, 2056, 2000), (4096, 4096, 4096)]


def path(M, N, K, dtype, product, act='none', aligned=True):
    return _lib.lib().vcb_linear_path(M, N, K, linear.TYPES[dtype], product, linear.ACTS[act],
                                      int(aligned))


def act64(z, act):
    return {'none': lambda: z, 'relu': lambda: torch.relu(z),
            'gelu': lambda: z * torch.special.ndtr(z), 'silu': lambda: z * torch.sigmoid(z)}[act]()


def slope64(z, act):
    z = z.clone().requires_grad_(True)
    act64(z, act).sum().backward()
    return z.grad


def rand(gen, *shape, dtype, scale=1.0):
    return (torch.randn(shape, device=DEV, generator=gen) * scale).to(dtype)


def close(got, want, dtype, roundings=1):
    assert got.dtype == dtype and got.shape == want.shape
    tol = TOL[dtype] * (roundings if dtype != torch.float32 else 1)
    err, scale = float((got.double() - want).abs().max()), float(want.abs().max())
    assert err <= tol * scale, (err, scale)


@gpu
@pytest.mark.parametrize('dtype', list(TOL))
@pytest.mark.parametrize('M,N,K', FORWARD)
def test_forward(M, N, K, dtype):
    assert path(M, N, K, dtype, 0, aligned=K % 8 == 0) == PAIRS
    gen = torch.Generator(DEV).manual_seed(M + N + K)
    x, w = rand(gen, M, K, dtype=dtype), rand(gen, N, K, dtype=dtype, scale=K ** -0.5)
    b, r = rand(gen, N, dtype=dtype), rand(gen, M, N, dtype=dtype)
    z0 = x.double() @ w.double().t()
    for i, act in enumerate(linear.ACTS):
        bias, res = (b if i != 1 else None), (r if i >= 2 else None)
        z = z0 if bias is None else z0 + b.double()
        y = act64(z, act) + (0 if res is None else r.double())
        got, gz = linear.linear_forward(x, w, bias, act, res, keep=True)
        close(got, y, dtype)
        close(gz, z, dtype)
        again = linear.linear_forward(x, w, bias, act, res)
        assert torch.equal(again, got)
    _lib.fault_check()


@gpu
@pytest.mark.parametrize('dtype', list(TOL))
@pytest.mark.parametrize('M,N,K', BACKWARD)
def test_backward(M, N, K, dtype):
    aligned = N % 8 == 0 and K % 8 == 0
    gen = torch.Generator(DEV).manual_seed(M * 3 + N + K)
    x, w = rand(gen, M, K, dtype=dtype), rand(gen, N, K, dtype=dtype, scale=K ** -0.5)
    dy, z = rand(gen, M, N, dtype=dtype), rand(gen, M, N, dtype=dtype)
    for act in linear.ACTS:
        assert [path(M, N, K, dtype, p, act, aligned) for p in (1, 2)] == [PAIRS, PAIRS]
        dz = dy.double() * slope64(z.double(), act)
        dx, dw, db = linear.linear_backward(dy, x, w, z if act != 'none' else None, act)
        n = 1 if act == 'none' else 2
        close(dx, dz @ w.double(), dtype, n)
        close(dw, dz.t() @ x.double(), dtype, n)
        close(db, dz.sum(0), dtype, n)
        for need in ((True, False), (False, True)):  # a product alone in its launch
            one = linear.linear_backward(dy, x, w, z if act != 'none' else None, act, False, need)
            for got, whole in zip(one, (dx, dw)):
                assert got is None or torch.equal(got, whole)
    _lib.fault_check()


@gpu
@pytest.mark.parametrize('dtype', list(TOL))
def test_one_product_in_pairs_and_one_cut(dtype):
    """dX of 4096 x 1024 x 1024 goes to the pairs, dW is cut over a cluster: two launches."""
    M, N, K = 4096, 1024, 1024
    assert [path(M, N, K, dtype, p, 'gelu') for p in (1, 2)] == [PAIRS, 2]
    gen = torch.Generator(DEV).manual_seed(8)
    x, w = rand(gen, M, K, dtype=dtype), rand(gen, N, K, dtype=dtype, scale=K ** -0.5)
    dy, z = rand(gen, M, N, dtype=dtype), rand(gen, M, N, dtype=dtype)
    dz = dy.double() * slope64(z.double(), 'gelu')
    for _ in range(3):
        dx, dw, db = linear.linear_backward(dy, x, w, z, 'gelu')
        close(dx, dz @ w.double(), dtype, 2)
        close(dw, dz.t() @ x.double(), dtype, 2)
        close(db, dz.sum(0), dtype, 2)
    _lib.fault_check()


@gpu
@pytest.mark.parametrize('dtype', list(TOL))
def test_large_calls_on_two_streams_repeat_bit_for_bit(dtype):
    gen = torch.Generator(DEV).manual_seed(9)
    M = N = K = 2048
    assert path(M, N, K, dtype, 0) == PAIRS
    x, w = rand(gen, M, K, dtype=dtype), rand(gen, N, K, dtype=dtype, scale=K ** -0.5)
    dy, z = rand(gen, M, N, dtype=dtype), rand(gen, M, N, dtype=dtype)

    def step():
        return [linear.linear_forward(x, w, act='silu'), *linear.linear_backward(dy, x, w, z, 'silu')]
    first = step()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(step())
    torch.cuda.synchronize()
    for out in outs:
        for a, b in zip(first, out):
            assert torch.equal(a, b)
    _lib.fault_check()


def test_path_query_of_calls_that_are_refused_or_small():
    f = _lib.lib().vcb_linear_path
    assert f(-1, 4, 4, 0, 0, 0, 1) == -1 and f(4, 4, 4, 3, 0, 0, 1) == -1
    assert f(4, 4, 4, 0, 3, 0, 1) == -1
    assert f(1, 4096, 4096, 1, 0, 0, 1) == 0 and f(1, 4096, 4096, 1, 2, 0, 1) == 0
    for t in (0, 1, 2):
        assert f(64, 50, 50, t, 0, 0, 1) == 1 and f(64, 50, 0, t, 1, 0, 1) == 1
        assert f(0, 50, 50, t, 0, 0, 1) == 1

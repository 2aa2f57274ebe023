"""Linear layer with epilogue and gradients against the definition in float64.

Tolerances.  With N(0, 1) inputs and weights of variance 1 / K, outputs and
gradients are of order 1 (``scale`` below is each reference's largest entry).
A product of K terms in float32 errs by at most a few 2^-24 sqrt(K) of a row's
norms, below 2e-6 of the scale for every size here; 16-bit types add one
rounding of the output (2^-8 bfloat16, 2^-11 float16, relative) and, in a
backward pass through an activation, one rounding of dz, whose errors in a sum
of independent terms stay below the same figure of the scale.
"""
import numpy as np
import pytest
import torch

from vibecheck_nn_b200 import _lib, linear

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
TOL = {torch.float32: 4e-6, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = list(TOL)
ACTS = list(linear.ACTS)


def act64(z, act):
    return {'none': lambda: z, 'relu': lambda: torch.relu(z),
            'gelu': lambda: z * torch.special.ndtr(z), 'silu': lambda: z * torch.sigmoid(z)}[act]()


def slope64(z, act):
    z = z.detach().clone().requires_grad_(True)
    act64(z, act).sum().backward()
    return z.grad


def close(got, want, dtype, roundings=1):
    want = want.double()
    assert got.dtype == dtype and got.shape == want.shape
    if not want.numel():
        return
    err = float((got.double() - want).abs().max())
    scale = float(want.abs().max())
    tol = TOL[dtype] * (roundings if dtype != torch.float32 else 1)
    assert err <= tol * max(scale, 1e-30), (err, scale)


def rand(gen, *shape, dtype, pad=0, scale=1.0):
    *lead, c = shape
    t = (torch.randn((*lead, c + pad), device=DEV, generator=gen) * scale).to(dtype)
    return t[..., :c]


SIZES = [(1, 1, 1), (1, 5, 3), (3, 64, 17), (1, 4096, 1024), (1, 1000, 4097), (2, 130, 264),
         (5, 50, 50), (17, 96, 128), (37, 500, 200), (64, 128, 64), (100, 256, 784),
         (129, 257, 65), (200, 1000, 72), (513, 384, 1000), (300, 2050, 512), (1024, 1024, 256)]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('M,N,K', SIZES)
def test_forward(M, N, K, dtype):
    gen = torch.Generator(DEV).manual_seed(M * 31 + N + K)
    for i, act in enumerate(ACTS):
        pad = (0, 3, 8, 1)[i]
        x = rand(gen, M, K, dtype=dtype, pad=pad)
        w = rand(gen, N, K, dtype=dtype, pad=pad % 3, scale=K ** -0.5)
        b = rand(gen, N, dtype=dtype) if i != 1 else None
        r = rand(gen, M, N, dtype=dtype, pad=pad) if i >= 2 else None
        z = x.double() @ w.double().t() + (0 if b is None else b.double())
        y = act64(z, act) + (0 if r is None else r.double())
        got, gz = linear.linear_forward(x, w, b, act, r, keep=True)
        close(got, y, dtype)
        close(gz, z, dtype)
        close(linear.linear_forward(x, w, b, act, r), y, dtype)
    _lib.fault_check()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('M,N,K', SIZES)
def test_backward(M, N, K, dtype):
    gen = torch.Generator(DEV).manual_seed(M * 37 + N + K)
    for i, act in enumerate(ACTS):
        pad = (0, 8, 3, 2)[i]
        x = rand(gen, M, K, dtype=dtype, pad=pad)
        w = rand(gen, N, K, dtype=dtype, scale=K ** -0.5)
        dy = rand(gen, M, N, dtype=dtype, pad=pad)
        z = rand(gen, M, N, dtype=dtype, pad=pad % 4)
        dz = dy.double() * slope64(z.double(), act)
        dx, dw, db = linear.linear_backward(dy, x, w, z if act != 'none' else None, act)
        n = 1 if act == 'none' else 2
        close(dx, dz @ w.double(), dtype, n)
        close(dw, dz.t() @ x.double(), dtype, n)
        close(db, dz.sum(0), dtype, n)
    _lib.fault_check()


def test_backward_parts_agree_with_the_whole():
    gen = torch.Generator(DEV).manual_seed(5)
    for M, N, K, dtype in ((33, 70, 90, torch.float32), (600, 520, 640, torch.bfloat16),
                           (600, 520, 640, torch.float32)):
        x, w = rand(gen, M, K, dtype=dtype), rand(gen, N, K, dtype=dtype)
        dy, z = rand(gen, M, N, dtype=dtype), rand(gen, M, N, dtype=dtype)
        dx, dw, db = linear.linear_backward(dy, x, w, z, 'relu')
        for bias in (True, False):
            for need in ((True, False), (False, True), (False, False)):
                got = linear.linear_backward(dy, x, w, z, 'relu', bias, need)
                want = (dx if need[0] else None, dw if need[1] else None, db if bias else None)
                for g, t in zip(got, want):
                    assert (g is None) == (t is None)
                    if t is not None:
                        close(g, t, dtype)


@pytest.mark.parametrize('dtype', TYPES)
def test_empty_axes(dtype):
    w, b = torch.ones(4, 6, device=DEV, dtype=dtype), torch.full((4,), 2.0, device=DEV, dtype=dtype)
    assert linear.linear_forward(torch.ones(0, 6, device=DEV, dtype=dtype), w, b).shape == (0, 4)
    none = torch.ones(3, 0, device=DEV, dtype=dtype)
    y = linear.linear_forward(none, torch.ones(4, 0, device=DEV, dtype=dtype), b, 'relu')
    assert torch.equal(y, b.expand(3, 4))
    dx, dw, db = linear.linear_backward(torch.ones(0, 4, device=DEV, dtype=dtype),
                                        torch.ones(0, 6, device=DEV, dtype=dtype), w)
    assert dx.shape == (0, 6) and not dw.any() and not db.any() and dw.shape == (4, 6)
    dx, dw, db = linear.linear_backward(torch.ones(3, 4, device=DEV, dtype=dtype), none,
                                        torch.ones(4, 0, device=DEV, dtype=dtype))
    assert dx.shape == (3, 0) and dw.shape == (4, 0) and torch.equal(db, torch.full_like(db, 3))
    dx, dw, db = linear.linear_backward(torch.ones(3, 0, device=DEV, dtype=dtype),
                                        torch.ones(3, 6, device=DEV, dtype=dtype),
                                        torch.ones(0, 6, device=DEV, dtype=dtype))
    assert not dx.any() and dx.shape == (3, 6) and dw.shape == (0, 6) and db.shape == (0,)


@pytest.mark.parametrize('M,N,K', [(7, 20, 12), (260, 300, 280)])
def test_gradient_is_the_slope_of_the_forward(M, N, K):
    """<dL/dp, d> against (L(p + h d) - L(p - h d)) / 2h with L summed in
    float64, every direction moving z by about h (a weight's by h / sqrt K per
    entry); float32 forward errors of 1e-6 over h = 1e-2 and the third
    derivative's h^2 stay below 2e-3 of the slope's size."""
    gen = torch.Generator(DEV).manual_seed(9)
    f32 = torch.float32
    x, w = rand(gen, M, K, dtype=f32), rand(gen, N, K, dtype=f32, scale=K ** -0.5)
    b, r = rand(gen, N, dtype=f32), rand(gen, M, N, dtype=f32)
    up = rand(gen, M, N, dtype=f32)
    for act in ('gelu', 'silu', 'none'):
        ps = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
        y = linear.linear(ps[0], ps[1], ps[2], act, ps[3])
        y.backward(up)
        for k in range(4):
            d = torch.randn(ps[k].shape, device=DEV, generator=gen) * (K ** -0.5 if k == 1 else 1)
            h = 1e-2

            def at(s):
                q = [t.detach() for t in ps]
                q[k] = q[k] + s * h * d
                return float((linear.linear_forward(q[0], q[1], q[2], act, q[3]).double()
                              * up.double()).sum())
            fd = (at(1) - at(-1)) / (2 * h)
            an = float((ps[k].grad.double() * d.double()).sum())
            size = float(up.double().norm()) * float(d.double().norm()) / d.numel() ** 0.5
            assert abs(fd - an) <= 2e-3 * max(size, abs(an)), (act, k, fd, an)


def test_autograd_matches_backward_and_leading_axes():
    gen = torch.Generator(DEV).manual_seed(2)
    x = rand(gen, 2, 3, 40, dtype=torch.bfloat16).contiguous().requires_grad_(True)
    w = rand(gen, 24, 40, dtype=torch.bfloat16).contiguous().requires_grad_(True)
    b = rand(gen, 24, dtype=torch.bfloat16).contiguous().requires_grad_(True)
    y = linear.linear(x, w, b, 'relu')
    assert y.shape == (2, 3, 24)
    up = rand(gen, 2, 3, 24, dtype=torch.bfloat16)
    y.backward(up)
    _, z = linear.linear_forward(x.detach(), w.detach(), b.detach(), 'relu', keep=True)
    dx, dw, db = linear.linear_backward(up, x.detach(), w.detach(), z, 'relu')
    assert torch.equal(x.grad, dx) and torch.equal(w.grad, dw) and torch.equal(b.grad, db)


@pytest.mark.parametrize('M,N,K', [(4, 40, 30), (300, 400, 320)])
def test_not_finite_inputs_reach_their_rows_only(M, N, K):
    for dtype in TYPES:
        gen = torch.Generator(DEV).manual_seed(3)
        x, w = rand(gen, M, K, dtype=dtype), rand(gen, N, K, dtype=dtype)
        x = x.clone()
        x[1, 2], x[2, 1] = float('nan'), float('inf')
        y = linear.linear_forward(x, w)
        bad = ~torch.isfinite(y)
        assert bad[1].all() and bad[2].all() and int(bad.any(1).sum()) == 2


def test_large_and_small_float32_rows_keep_their_precision():
    """Rows and weights of very different size: each output is within 4e-6 of
    its own row's and weight's norms."""
    gen = torch.Generator(DEV).manual_seed(4)
    for M, N, K in ((6, 80, 64), (300, 320, 512)):
        x, w = rand(gen, M, K, dtype=torch.float32), rand(gen, N, K, dtype=torch.float32)
        x = x * torch.logspace(-25, 12, M, device=DEV)[:, None]
        w = w * torch.logspace(12, -9, N, device=DEV)[:, None]
        want = x.double() @ w.double().t()
        err = (linear.linear_forward(x, w).double() - want).abs()
        size = x.double().norm(dim=1)[:, None] * w.double().norm(dim=1)[None]
        assert float((err / size).max()) <= 4e-6
        dy = rand(gen, M, N, dtype=torch.float32) * torch.logspace(-10, 10, M, device=DEV)[:, None]
        dx, dw, _ = linear.linear_backward(dy, x, w)
        for got, a, b in ((dx, dy, w.t()), (dw, dy.t(), x.t())):
            a, b = a.double(), b.double()
            size = a.norm(dim=1)[:, None] * b.norm(dim=1)[None]
            assert float(((got.double() - a @ b.t()).abs() / size).max()) <= 4e-6


def test_runs_on_the_current_stream_and_repeats_bit_for_bit():
    gen = torch.Generator(DEV).manual_seed(6)
    for dtype, (M, N, K) in ((torch.bfloat16, (40, 1000, 2000)), (torch.float32, (500, 600, 700)),
                             (torch.float16, (700, 640, 512))):
        x, w = rand(gen, M, K, dtype=dtype), rand(gen, N, K, dtype=dtype)
        z, dy = rand(gen, M, N, dtype=dtype), rand(gen, M, N, dtype=dtype)
        first = [linear.linear_forward(x, w), *linear.linear_backward(dy, x, w, z, 'silu')]
        torch.cuda.synchronize()
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            again = [linear.linear_forward(x, w), *linear.linear_backward(dy, x, w, z, 'silu')]
        s.synchronize()
        for a, b in zip(first, again):
            assert torch.equal(a, b)
    _lib.fault_check()


def test_refusals():
    x, w = torch.ones(2, 4, device=DEV), torch.ones(3, 4, device=DEV)
    with pytest.raises(_lib.UnsupportedInput):
        linear.linear_forward(x.cpu(), w.cpu())
    with pytest.raises(_lib.UnsupportedInput):
        linear.linear_forward(x.double(), w.double())
    for bad in (lambda: linear.linear_forward(x, w.half()),
                lambda: linear.linear_forward(x, torch.ones(3, 5, device=DEV)),
                lambda: linear.linear_forward(x, w, torch.ones(2, device=DEV)),
                lambda: linear.linear_forward(x, w, act='tanh'),
                lambda: linear.linear_forward(x, w, residual=torch.ones(3, device=DEV)),
                lambda: linear.linear_backward(torch.ones(2, 4, device=DEV), x, w),
                lambda: linear.linear_backward(torch.ones(2, 3, device=DEV), x, w, act='relu')):
        with pytest.raises(ValueError):
            bad()
    lib = _lib.lib()
    p = x.data_ptr()
    assert lib.vcb_linear_forward(2, 3, 4, 9, p, 4, p, 4, None, 0, None, 0, p, 3, None, 0, None, 0,
                                  None) == _lib.VCB_ERR_INVALID
    assert lib.vcb_linear_forward(2, 3, 4, 0, p, 3, p, 4, None, 0, None, 0, p, 3, None, 0, None, 0,
                                  None) == _lib.VCB_ERR_INVALID
    assert lib.vcb_linear_forward(2, 3, 4, 0, None, 4, p, 4, None, 0, None, 0, p, 3, None, 0, None,
                                  0, None) == _lib.VCB_ERR_INVALID
    assert lib.vcb_linear_backward(2, 3, 4, 0, p, 3, p, 4, p, 4, None, 0, 1, p, 4, p, 4, p, None, 0,
                                   None) == _lib.VCB_ERR_INVALID


# Rows of every kernel: few rows, small products cut unevenly, copies of unaligned operands,
# pairs with a short contraction, narrow gradients.
VIEW_SIZES = [(1, 300, 1001), (2, 1025, 515), (4, 520, 2050), (6, 1001, 515), (8, 130, 100),
              (16, 600, 500), (50, 33, 5), (900, 40, 70), (2314, 5, 10), (1500, 131, 300),
              (700, 1200, 40)]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('M,N,K', VIEW_SIZES)
@pytest.mark.parametrize('first,pad', [(1, 0), (1, 3), (3, 8)])
def test_rows_that_start_anywhere(M, N, K, first, pad, dtype):
    """Operands are columns first.. of wider matrices, so that rows start on odd elements; the
    neighbours are NaN and may not be read into any result."""
    gen = torch.Generator(DEV).manual_seed(M + 7 * N + 31 * K + first)

    def view(rows, cols, scale=1.0):
        t = torch.full((rows, first + cols + pad), float('nan'), dtype=dtype, device=DEV)
        t[:, first:first + cols] = rand(gen, rows, cols, dtype=dtype, scale=scale)
        return t[:, first:first + cols]

    x, w, r = view(M, K), view(N, K, K ** -0.5), view(M, N)
    b = rand(gen, N + 1, dtype=dtype)[1:]
    z = x.double() @ w.double().t() + b.double()
    got, gz = linear.linear_forward(x, w, b, 'silu', r, keep=True)
    close(got, act64(z, 'silu') + r.double(), dtype)
    close(gz, z, dtype)
    dy, zz = view(M, N), view(M, N)
    dz = dy.double() * slope64(zz.double(), 'gelu')
    dx, dw, db = linear.linear_backward(dy, x, w, zz, 'gelu')
    close(dx, dz @ w.double(), dtype, 2)
    close(dw, dz.t() @ x.double(), dtype, 2)
    close(db, dz.sum(0), dtype, 2)
    _lib.fault_check()


@pytest.mark.parametrize('dtype', TYPES)
def test_calls_in_a_row_share_the_workspace(dtype):
    """Each call prepares its operands in the memory that the call before it used: the product of
    one has to be over before the preparation of the next, and after its own."""
    gen = torch.Generator(DEV).manual_seed(11)
    M, N, K = 520, 515, 513
    xs = [rand(gen, M, K, dtype=dtype) for _ in range(4)]
    w, dy = rand(gen, N, K, dtype=dtype, scale=K ** -0.5), rand(gen, M, N, dtype=dtype)
    alone = []
    for x in xs:
        y, z = linear.linear_forward(x, w, None, 'gelu', keep=True)
        alone.append((y, z, *linear.linear_backward(dy, x, w, z, 'gelu')))
        torch.cuda.synchronize()
    for _ in range(5):
        together = []
        for x in xs:
            y, z = linear.linear_forward(x, w, None, 'gelu', keep=True)
            together.append((y, z, *linear.linear_backward(dy, x, w, z, 'gelu')))
        torch.cuda.synchronize()
        for got, want in zip(together, alone):
            for g, t in zip(got, want):
                assert torch.equal(g, t)
    _lib.fault_check()

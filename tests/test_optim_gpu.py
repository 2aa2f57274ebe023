"""AdamW against the definition in float64.

One step in float32 errs by a few 2^-24 of the weight, of the two terms of each
moment and of the step that the terms of m would make (m itself may cancel):
1e-6 of each is allowed (16-bit weights: one rounding more).  A code
of an 8-bit state may lie one step from the code that float64 would choose
where the noise falls on the other side of a probability that float32 rounds:
at most 1e-3 of the elements; everywhere else codes are equal.
"""
import numpy as np
import pytest
import torch

from vibecheck_nn_b200 import _lib, optim

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
SHAPES = [(50, 5), (50,), (7,), (1,), (256,), (257,), (3, 4099), (0,), (2048,), (130, 2049)]
ROUND = {torch.float32: 2.0 ** -23, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -10}


def noise(i, key):
    m = 0xFFFFFFFF
    x = ((i + key) & m) * 0x9E3779B9 & m
    x = (x ^ (x >> 16)) * 0x6A09E667 & m
    x = (x ^ (x >> 15)) * 0xBB67AE85 & m
    return x ^ (x >> 16)


def values(code, scale, levels, power):
    c = code.double()
    return torch.sign(c) * (c.abs() / levels) ** power * scale.double().repeat_interleave(256)


def tensors(dtype, seed=0, shapes=SHAPES, gdtype=None, shift=0):
    gen = torch.Generator(DEV).manual_seed(seed)

    def make(s, i, dt, scale):
        n = int(np.prod(s))
        t = (torch.randn(n + shift, device=DEV, generator=gen) * scale).to(dt)
        return t[shift:].view(s)
    return ([make(s, i, dtype, 0.1) for i, s in enumerate(shapes)],
            [[make(s, i, gdtype or dtype, 10.0 ** (-i % 4)) for i, s in enumerate(shapes)]
             for _ in range(3)])


def flat(ts, opt):
    out = torch.zeros(opt.m.numel(), dtype=torch.float64, device=DEV)
    for t, at in zip(ts, opt.offsets):
        out[at:at + t.numel()] = t.reshape(-1).double()
    return out


@pytest.mark.parametrize('dtype,gdtype', [(torch.float32, None), (torch.bfloat16, None),
                                          (torch.float16, None), (torch.bfloat16, torch.float32),
                                          (torch.float16, torch.float32)])
@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('shift', [0, 1])
def test_three_steps(dtype, gdtype, bits, shift):
    ps, grads = tensors(dtype, 1, gdtype=gdtype, shift=shift)
    opt = optim.AdamW(ps, state_bits=bits, seed=11, **HYPER)
    b1, b2 = HYPER['betas']
    for t in (1, 2, 3):
        p0, g = flat(ps, opt), flat(grads[t - 1], opt)
        m0, v0 = (s.double().clone() for s in opt.moments())
        opt.step(grads[t - 1])
        m = b1 * m0 + (1 - b1) * g
        v = b2 * v0 + (1 - b2) * g * g
        rate = HYPER['lr'] / (1 - b1 ** t) / (torch.sqrt(v / (1 - b2 ** t)) + HYPER['eps'])
        step = rate * m
        terms = rate * (b1 * m0.abs() + (1 - b1) * g.abs())
        p = p0 * (1 - HYPER['lr'] * HYPER['weight_decay']) - step
        err = (flat(ps, opt) - p).abs()
        # float16: half of its smallest step as well
        bound = ROUND[dtype] * p.abs() + 1e-6 * (p0.abs() + terms) + \
            (2.0 ** -25 if dtype == torch.float16 else 0)
        assert bool((err <= bound).all()), float((err - bound).max())
        gm, gv = (s.double() for s in opt.moments())
        if bits == 32:
            assert bool(((gm - m).abs() <= 1e-6 * (m0.abs() + g.abs())).all())
            assert bool(((gv - v).abs() <= 1e-6 * v).all())
            continue
        key = (11 * 0xBB67AE85 + t * 0x6A09E667) & 0xFFFFFFFF
        h = noise(torch.arange(m.numel(), device=DEV), key)
        for val, r, codes, scale, levels, power in (
                (m, h >> 16, opt.m, opt.m_scale, 127, 2), (v, h & 0xFFFF, opt.v, opt.v_scale, 255, 4)):
            top = val.abs().view(-1, 256).amax(1)
            assert bool(((scale.double() - top).abs() <= 1e-6 * top).all())
            a = torch.where(top > 0, val.abs().view(-1, 256).T / top, torch.zeros(())
                            .to(val)).T.reshape(-1)
            low = torch.floor(a ** (1 / power) * levels + 1e-9).clamp(max=levels - 1)
            lo, hi = (low / levels) ** power, ((low + 1) / levels) ** power
            want = low + (r.double() / 65536 * (hi - lo) < a - lo).double()
            if power == 4:
                want = torch.where((a > 0) & (want < 1), torch.ones_like(want), want)
            want = torch.sign(val) * want
            off = (codes.double() - want).abs()
            assert float(off.max()) <= 1 and float((off > 0).double().mean()) <= 1e-3
            assert not codes[flat([torch.ones_like(q) for q in ps], opt) == 0].any()
            got = values(codes, scale, levels, power)
            assert bool(((got - (gm if power == 2 else gv)).abs() <= 1e-6 * got.abs()).all())


def test_many_tensors_are_the_same_as_one_by_one():
    """More tensors than one launch's table holds; 8-bit noise goes by the
    place in the state, so 32-bit states are compared bit for bit."""
    shapes = [(1 + i % 300,) for i in range(1500)]
    ps, grads = tensors(torch.float32, 3, shapes)
    qs = [p.clone() for p in ps]
    opt = optim.AdamW(ps, **HYPER)
    opt.step(grads[0])
    for q, g, p in list(zip(qs, grads[0], ps))[::37]:
        one = optim.AdamW([q], **HYPER)
        one.step([g])
        assert torch.equal(q, p)


def test_eight_bit_codes_keep_the_mean():
    """One gradient repeated: m and v must reach their 32-bit values on
    average.  512 blocks of one value beside its block's largest: with random
    rounding the mean over 511 x 256 elements is within 1 %; with codes that
    only ever round to the nearest, v would stop far below."""
    n = 256 * 512
    g = torch.full((n,), 0.02, device=DEV)
    g[::256] = 1.0
    ps = [torch.zeros(n, device=DEV)], [torch.zeros(n, device=DEV)]
    a = optim.AdamW(ps[0], betas=(0.9, 0.999), state_bits=32)
    b = optim.AdamW(ps[1], betas=(0.9, 0.999), state_bits=8, seed=5)
    for _ in range(300):
        a.step([g])
        b.step([g])
    small = torch.ones(n, dtype=torch.bool, device=DEV)
    small[::256] = False
    for x, y in zip(a.moments(), b.moments()):
        want, got = float(x[small].double().mean()), float(y[small].double().mean())
        assert abs(got - want) <= 0.01 * want, (got, want)
    assert not bool((b.v[small] == 0).any())
    # 1 / sqrt(v) of a v that scatters by a quarter around its mean is 2 % up on average
    want, got = (float(p[0][small].double().mean()) for p in ps)
    assert abs(got - want) <= 0.1 * abs(want), (got, want)


def test_none_gradients_zero_gradients_and_not_finite_ones():
    for bits in (32, 8):
        ps, grads = tensors(torch.float32, 4, [(300,), (600,), (256,)])
        keep = ps[1].clone()
        opt = optim.AdamW(ps, state_bits=bits, **HYPER)
        opt.step([grads[0][0], None, torch.zeros_like(ps[2])])
        assert torch.equal(ps[1], keep) and not opt.m[512:1536].any()
        assert bool(torch.isfinite(ps[2]).all()) and not opt.v[1280:].any()
        g = grads[1][1]
        g[10] = float('nan')
        g[300] = float('inf')
        opt.step([None, g, None])
        m, v = opt.moments()
        bad = ~torch.isfinite(ps[1])
        assert bool(bad[10]) and int(bad.sum()) <= 2
        hit = torch.isnan(m[512:512 + 600])
        assert bool(hit[10]) and not bool(hit[512:].any())
        assert bool(torch.isfinite(m[:512]).all())


def test_tiny_and_huge_gradients():
    """Blocks at the ends of float32's range stay finite and ordered."""
    ps = [torch.zeros(256 * 4, device=DEV)]
    g = torch.ones(256 * 4, device=DEV)
    g[:256], g[256:512], g[512:768], g[768:] = 1e-30, 1e-18, 1e15, 1e18
    opt = optim.AdamW(ps, lr=0.1, weight_decay=0.0, state_bits=8)
    opt.step([g])
    m, v = opt.moments()
    assert bool(torch.isfinite(ps[0]).all()) and bool(torch.isfinite(m).all())
    assert bool((m.view(4, 256).diff(dim=0) >= 0).all()) and bool(torch.isfinite(v).all())
    assert torch.allclose(ps[0][512:], torch.full_like(ps[0][512:], -0.1), rtol=1e-5)


def test_resume_continues_bit_for_bit():
    for bits in (32, 8):
        ps, grads = tensors(torch.float32, 6)
        opt = optim.AdamW(ps, state_bits=bits, seed=3, **HYPER)
        opt.step(grads[0])
        saved, qs = opt.state_dict(), [p.clone() for p in ps]
        opt.step(grads[1])
        again = optim.AdamW(qs, state_bits=bits, **HYPER)
        again.load_state_dict(saved)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            again.step(grads[1])
        s.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(ps, qs))
        assert torch.equal(opt.m, again.m) and torch.equal(opt.v, again.v)


def test_uses_grad_fields_and_strided_gradients():
    p = torch.ones(6, 8, device=DEV, requires_grad=True)
    q = p.detach().clone()
    version = p._version
    g = torch.arange(48.0, device=DEV).view(8, 6).t()
    p.grad = g
    optim.AdamW([p], **HYPER).step()
    optim.AdamW([q], **HYPER).step([g.contiguous()])
    assert torch.equal(p.detach(), q) and p._version > version


def test_refusals():
    p = torch.ones(4, device=DEV)
    with pytest.raises(_lib.UnsupportedInput):
        optim.AdamW([p.cpu()])
    with pytest.raises(_lib.UnsupportedInput):
        optim.AdamW([p.double()])
    opt = optim.AdamW([p])
    for bad in (lambda: optim.AdamW([]), lambda: optim.AdamW([p], state_bits=4),
                lambda: optim.AdamW([p], betas=(1.0, 0.9)),
                lambda: optim.AdamW([torch.ones(4, 4, device=DEV).t()]),
                lambda: opt.step([]), lambda: opt.step([torch.ones(5, device=DEV)]),
                lambda: opt.step([torch.ones(4)]),
                lambda: opt.load_state_dict({'step': 1, 'm': p, 'v': p})):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(_lib.UnsupportedInput):
        opt.step([torch.ones(4, device=DEV, dtype=torch.float16)])
    assert opt.t == 0
    lib = _lib.lib()
    o = _lib.VcbAdamwOpts()
    import ctypes
    none = (None,) * 4
    assert lib.vcb_adamw(1, *none, 0, 0, 32, None, None, None, None, ctypes.byref(o), None) \
        == _lib.VCB_ERR_INVALID
    assert lib.vcb_adamw(0, *none, 0, 0, 16, None, None, None, None, ctypes.byref(o), None) \
        == _lib.VCB_ERR_INVALID

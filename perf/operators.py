"""Measured cases of the training-step operators: a linear layer with its
epilogue and gradients, the softmax cross-entropy with its gradient, and the
AdamW step over many tensors.

``listed()`` names the cases, ``draw(rng)`` makes more of the same ranges,
``prepare(case, seed)`` builds what a training or serving program holds before
the call, ``run(state)`` makes one pass.  With ``own`` false a pass is the
operator's plain form in elementary 32-bit torch operations, with ``own`` true
it is the package's public call.  ``exact(case, seed)`` is the definition
evaluated in 64 bits.
"""
import math

import numpy as np
import torch

own = False

DEV = 'cuda'
TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
ACTS = ('none', 'relu', 'gelu', 'silu')
IGNORE = -100
BLOCK = 256           # elements that share one scale of an 8-bit state
GOLDEN, ROOT2, ROOT3 = 0x9E3779B9, 0x6A09E667, 0xBB67AE85   # the noise's multipliers
MASK32 = 0xFFFFFFFF
V_LEVELS = float(np.float32(255.0 ** 4))
LARGEST_LINEAR = 8192 * 8192 * 4096


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _linear(name, way, dtype, M, N, K, act='none', bias=True, residual=False, keep=False, pad=0):
    return {'name': name, 'op': 'linear', 'way': way, 'dtype': dtype, 'M': M, 'N': N, 'K': K,
            'act': act, 'bias': bias, 'residual': residual, 'keep': keep, 'pad': pad}


def _loss(name, dtype, R, C, ignored=0.1, masked=0.0, pad=0):
    return {'name': name, 'op': 'loss', 'dtype': dtype, 'R': R, 'C': C, 'ignored': ignored,
            'masked': masked, 'pad': pad}


def _adamw(name, dtype, bits, tensors, width, shape):
    return {'name': name, 'op': 'adamw', 'dtype': dtype, 'bits': bits, 'tensors': tensors,
            'width': width, 'shape': shape}


def listed():
    return [
        # one token through a wide layer: the weight is read once, nothing else matters
        _linear('linear one token', 'forward', 'bf16', 1, 4096, 4096, 'silu', True, True),
        # a batch of decoding requests, rows and columns off every tile
        _linear('linear 37 tokens f16', 'forward', 'f16', 37, 5000, 2048, 'gelu', True, False),
        # the 784 -> 256 layer of the ReLU-split workload in a training batch
        _linear('linear 784-256 backward', 'backward', 'f32', 100, 256, 784, 'relu', True),
        # a training forward at the largest batch, pre-activation kept for the backward pass
        _linear('linear bf16 training', 'forward', 'bf16', 8192, 8192, 4096, 'gelu', True, True, True),
        # both gradients at sizes that no tile divides and rows that are not 16-byte aligned
        _linear('linear bf16 ragged backward', 'backward', 'bf16', 2047, 2050, 1999, 'silu', True),
        # a 32-bit training forward: what is trained to be bounded in 32 bits
        _linear('linear f32 training', 'forward', 'f32', 4096, 4096, 4096, 'relu', True, False, True),
        # a classifier's ten classes in a small batch
        _loss('loss 10 classes', 'f32', 100, 10),
        # a mid-sized table of outputs, odd width, some of them masked off
        _loss('loss 50001 bf16', 'bf16', 2048, 50001, 0.1, 0.01),
        # the longest rows: one row does not fit an SM
        _loss('loss 131072 bf16', 'bf16', 8192, 131072, 0.3),
        # the tensors of the 5 -> [50] x 6 -> 5 network: one launch's latency
        _adamw('adamw 5-50-5 network', 'f32', 32, 14, 50, 'mlp'),
        # a deeper network of ragged layers in 16 bits with 8-bit states
        _adamw('adamw bf16 8-bit states', 'bf16', 8, 24, 1021, 'ragged'),
        # a large model's share on one GPU, 32-bit weights and 8-bit states
        _adamw('adamw f32 8-bit large', 'f32', 8, 16, 4096, 'ragged'),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.5 else max(lo, n // 8 * 8)


def draw(rng):
    op = rng.choice(['linear', 'linear', 'loss', 'adamw'])
    dtype = rng.choice(['f32', 'bf16', 'f16'])
    if op == 'linear':
        limit = 4096 ** 3 if dtype == 'f32' else LARGEST_LINEAR
        way = rng.choice(['forward', 'backward'])
        limit //= 2 if way == 'backward' else 1
        M, N, K = _log(rng, 1, 8192), _width(rng, 5, 8192), _width(rng, 5, 8192)
        while M * N * K > limit:
            M = max(1, M // 2)
        case = _linear('', way, dtype, M, N, K, rng.choice(ACTS), rng.random() < 0.8,
                       way == 'forward' and rng.random() < 0.5,
                       way == 'forward' and rng.random() < 0.5, rng.choice([0, 0, 8, 3]))
    elif op == 'loss':
        R, C = _log(rng, 1, 8192), _width(rng, 2, 131072)
        case = _loss('', dtype, R, C, rng.choice([0.0, 0.1, 0.5]), rng.choice([0.0, 0.01, 0.3]),
                     rng.choice([0, 0, 8, 3]))
        while case['R'] * case['C'] * (2 if dtype == 'f32' else 1) > 8192 * 131072:
            case['R'] = max(1, case['R'] // 2)
    else:
        case = _adamw('', dtype, rng.choice([8, 32]), rng.randint(1, 40), _log(rng, 5, 2500),
                      rng.choice(['mlp', 'ragged']))
        while sum(_sizes(case)) > sum(_sizes(listed()[-1])) // 2:
            case['width'] = case['width'] * 3 // 4
    del case['name']
    return case


def _shapes(case):
    """The tensors of a network: weights and biases in turn; 'ragged' layers differ in width."""
    n, w = case['tensors'], case['width']
    if case['shape'] == 'mlp':
        d = [5] + [w] * max(0, (n + 1) // 2 - 1) + [5]
    else:
        d = [w + (37 * i) % 101 for i in range((n + 1) // 2 + 1)]
    both = [s for i in range((n + 1) // 2) for s in ((d[i + 1], d[i]), (d[i + 1],))]
    return both[:n]


def _sizes(case):
    return [int(np.prod(s)) for s in _shapes(case)]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _rows(R, C, pad, dtype, gen, scale=1.0):
    """(R, C) normal values; with `pad` a slice of rows that are wider than what is used."""
    t = torch.randn((R, C + pad), device=DEV, generator=gen).mul_(scale).to(dtype)
    return t[:, :C]


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 13)
    s = {'case': dict(case)}
    dt = TYPES[case['dtype']]
    if case['op'] == 'linear':
        M, N, K = case['M'], case['N'], case['K']
        s['x'] = _rows(M, K, case['pad'], dt, gen)
        s['w'] = _rows(N, K, 0, dt, gen, K ** -0.5)
        s['b'] = _rows(1, N, 0, dt, gen, 0.1)[0] if case['bias'] else None
        s['r'] = _rows(M, N, 0, dt, gen) if case['residual'] else None
        if case['way'] == 'backward':
            z = s['x'].float() @ s['w'].float().t()
            s['z'] = (z + s['b'].float() if case['bias'] else z).to(dt)
            s['dy'] = _rows(M, N, case['pad'], dt, gen, 0.05)
        if own:
            from vibecheck_nn_b200 import linear
            s['call'] = linear
    elif case['op'] == 'loss':
        R, C = case['R'], case['C']
        s['logits'] = _rows(R, C, case['pad'], dt, gen, 2.0)
        labels = torch.randint(0, C, (R,), device=DEV, generator=gen)
        if case['masked']:
            off = torch.rand((R, C), device=DEV, generator=gen) < case['masked']
            off[torch.arange(R, device=DEV), labels] = False
            s['logits'].masked_fill_(off, float('-inf'))
        labels[torch.rand(R, device=DEV, generator=gen) < case['ignored']] = IGNORE
        s['labels'] = labels
        if own:
            from vibecheck_nn_b200 import loss
            s['call'] = loss
    else:
        _prepare_adamw(case, s, gen, dt, int(seed))
    return s


def _prepare_adamw(case, s, gen, dt, seed):
    shapes = _shapes(case)
    s['params'] = [(torch.randn(sh, device=DEV, generator=gen) * 0.05).to(dt) for sh in shapes]
    # gradients of a network differ in size between its tensors and between its neurons
    s['grads'] = [(torch.randn(sh, device=DEV, generator=gen)
                   * torch.exp(torch.randn(sh[:1] + (1,) * (len(sh) - 1), device=DEV, generator=gen))
                   * 10.0 ** (-2 - i % 3)).to(dt) for i, sh in enumerate(shapes)]
    starts, total = [], 0
    for sh in shapes:
        starts.append(total)
        total += -(-int(np.prod(sh)) // BLOCK) * BLOCK
    live = torch.zeros(total, device=DEV, dtype=torch.bool)
    for at, sh in zip(starts, shapes):
        live[at:at + int(np.prod(sh))] = True
    state = {'step': 100}
    if case['bits'] == 32:
        state['m'] = torch.randn(total, device=DEV, generator=gen).mul_(1e-3) * live
        state['v'] = torch.rand(total, device=DEV, generator=gen).mul_(1e-5) * live
    else:
        blocks = total // BLOCK
        state['m'] = (torch.randint(-127, 128, (total,), device=DEV, generator=gen) * live).to(torch.int8)
        state['v'] = (torch.randint(1, 256, (total,), device=DEV, generator=gen) * live).to(torch.uint8)
        state['m_scale'] = torch.rand(blocks, device=DEV, generator=gen).add_(0.1).mul_(1e-3)
        state['v_scale'] = torch.rand(blocks, device=DEV, generator=gen).add_(0.1).mul_(1e-5)
    s['hyper'] = {'lr': 1e-3, 'betas': (0.9, 0.999), 'eps': 1e-8, 'weight_decay': 0.01}
    s['noise'] = seed & 0x7FFFFFFF
    if own:
        from vibecheck_nn_b200 import optim
        s['opt'] = optim.AdamW(s['params'], state_bits=case['bits'], seed=s['noise'], **s['hyper'])
        s['opt'].load_state_dict(state)
    else:
        s['starts'], s['state'] = starts, state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    return {'linear': _run_linear, 'loss': _run_loss, 'adamw': _run_adamw}[s['case']['op']](s)


def _run_linear(s):
    c = s['case']
    if own:
        if c['way'] == 'forward':
            return s['call'].linear_forward(s['x'], s['w'], s['b'], act=c['act'], residual=s['r'],
                                            keep=c['keep'])
        return s['call'].linear_backward(s['dy'], s['x'], s['w'], z=s['z'], act=c['act'],
                                         bias=c['bias'])
    dt = s['x'].dtype
    x, w = s['x'].float(), s['w'].float()
    if c['way'] == 'forward':
        z = x @ w.t()
        z = z + s['b'].float() if c['bias'] else z
        y = _act(z, c['act'])
        y = y + s['r'].float() if c['residual'] else y
        return (y.to(dt), z.to(dt)) if c['keep'] else y.to(dt)
    dz = s['dy'].float() * _act_slope(s['z'].float(), c['act'])
    return ((dz @ w).to(dt), (dz.t() @ x).to(dt), dz.sum(0).to(dt) if c['bias'] else None)


def _act(z, act):
    if act == 'relu':
        return torch.clamp(z, min=0)
    if act == 'gelu':
        return 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))
    return z / (1 + torch.exp(-z)) if act == 'silu' else z


def _act_slope(z, act):
    if act == 'relu':
        return (z > 0).to(z.dtype)
    if act == 'gelu':
        return 0.5 * (1 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    if act == 'silu':
        g = 1 / (1 + torch.exp(-z))
        return g * (1 + z * (1 - g))
    return torch.ones_like(z)


def _run_loss(s):
    if own:
        return s['call'].cross_entropy_grad(s['logits'], s['labels'], ignore_index=IGNORE)
    x, labels = s['logits'].float(), s['labels']
    live = labels != IGNORE
    at = torch.where(live, labels, torch.zeros_like(labels)).unsqueeze(1)
    e = torch.exp(x - x.amax(1, keepdim=True))
    total = e.sum(1, keepdim=True)
    row = torch.log(total[:, 0]) - (x.gather(1, at) - x.amax(1, keepdim=True))[:, 0]
    count = live.sum().clamp(min=1).float()
    zero = torch.zeros_like(row)
    grad = e / total
    grad.scatter_add_(1, at, torch.full_like(at, -1, dtype=grad.dtype))
    grad = torch.where(live.unsqueeze(1), grad / count, zero.unsqueeze(1))
    return torch.where(live, row, zero).sum() / count, grad.to(s['logits'].dtype)


def _run_adamw(s):
    if own:
        s['opt'].step(s['grads'])
        return (s['params'], *s['opt'].moments())
    st = s['state']
    st['step'] += 1
    k = _adam_constants(s['hyper'], st['step'])
    key = _noise_key(s['noise'], st['step'])
    done = [_adamw_one(p, g, st, at, k, key) for p, g, at in zip(s['params'], s['grads'], s['starts'])]
    if 'm_scale' not in st:
        return s['params'], st['m'], st['v']
    m, v = torch.zeros_like(st['m'], dtype=torch.float32), torch.zeros_like(st['v'], dtype=torch.float32)
    m.view(-1, BLOCK).copy_(st['m_scale'].unsqueeze(1) * _m_level(st['m'].view(-1, BLOCK)))
    v.view(-1, BLOCK).copy_(st['v_scale'].unsqueeze(1) * _v_level(st['v'].view(-1, BLOCK)))
    return s['params'], m, v


def _adam_constants(h, step):
    """The step's constants, each rounded once to 32 bits."""
    b1, b2 = h['betas']
    f = lambda x: float(np.float32(x))  # noqa: E731
    return {'b1': f(b1), 'c1': f(1 - b1), 'b2': f(b2), 'c2': f(1 - b2), 'eps': f(h['eps']),
            'size': f(h['lr'] / (1 - b1 ** step)), 'root': f((1 - b2 ** step) ** -0.5),
            'keep': f(1 - h['lr'] * h['weight_decay'])}


def _noise_key(seed, step):
    return (seed * ROOT3 + step * ROOT2) & MASK32


def _noise(index, key):
    """32 noise bits for each element's place in the state, as int64."""
    x = ((index + key) & MASK32) * GOLDEN & MASK32
    x = (x ^ (x >> 16)) * ROOT2 & MASK32
    x = (x ^ (x >> 15)) * ROOT3 & MASK32
    return x ^ (x >> 16)


def _m_level(code):
    c = code.to(torch.float32)
    return c * c.abs() * float(np.float32(1 / 16129.0))


def _v_level(code):
    q = code.to(torch.float32)
    q = q * q
    return q * q * float(np.float32(1 / 255.0 ** 4))


def _adamw_one(p, g, st, at, k, key):
    n = p.numel()
    end = at + -(-n // BLOCK) * BLOCK
    g32 = g.reshape(-1).float()
    if 'm_scale' not in st:
        m, v = st['m'][at:at + n], st['v'][at:at + n]
        m1 = m * k['b1'] + g32 * k['c1']
        v1 = v * k['b2'] + g32 * k['c2'] * g32
        m.copy_(m1)
        v.copy_(v1)
    else:
        lo, hi = at // BLOCK, end // BLOCK
        gb = torch.zeros(end - at, device=g.device).view(-1, BLOCK)
        gb.view(-1)[:n] = g32
        m = st['m_scale'][lo:hi, None] * _m_level(st['m'][at:end].view(-1, BLOCK))
        v = st['v_scale'][lo:hi, None] * _v_level(st['v'][at:end].view(-1, BLOCK))
        m = m * k['b1'] + gb * k['c1']
        v = v * k['b2'] + gb * k['c2'] * gb
        h = _noise(torch.arange(at, end, device=g.device).view(-1, BLOCK), key)
        big, most = m.abs().amax(1, keepdim=True), v.amax(1, keepdim=True)
        big, most = (torch.where(t < torch.finfo(torch.float32).tiny, torch.zeros_like(t), t) for t in (big, most))
        st['m'][at:end] = _m_code(m, big, (h >> 16).float() * 2.0 ** -16).view(-1)
        st['v'][at:end] = _v_code(v, most, (h & 0xFFFF).float() * 2.0 ** -16).view(-1)
        st['m_scale'][lo:hi] = big[:, 0]
        st['v_scale'][lo:hi] = most[:, 0]
        m1, v1 = m.view(-1)[:n], v.view(-1)[:n]
    d = m1 / (torch.sqrt(v1) * k['root'] + k['eps'])
    q = p.reshape(-1).float() * k['keep'] - d * k['size']
    p.copy_(q.view(p.shape))


def _m_code(m, big, r):
    """Codes c of m ~ big sign(c) (c / 127)^2, up or down with the probability that keeps the mean."""
    y = torch.where(big > 0, m.abs() * (1 / big) * 16129.0, torch.zeros_like(m))
    c = torch.floor(torch.sqrt(y)).clamp(max=126)
    c = c - (c * c > y).float()
    up = r * (2 * c + 1) < y - c * c
    return (torch.where(m < 0, -1.0, 1.0) * (c + up.float())).to(torch.int8)


def _v_code(v, most, r):
    """Codes c of v ~ most (c / 255)^4; what is not zero gets no code that stands for zero."""
    y = torch.where(most > 0, v * (1 / most) * V_LEVELS, torch.zeros_like(v))
    four = lambda c: (c * c) * (c * c)  # noqa: E731
    c = torch.floor(torch.sqrt(torch.sqrt(y))).clamp(max=254)
    c = c - (four(c) > y).float()
    c = c + ((four(c + 1) <= y) & (c < 254)).float()
    up = r * (four(c + 1) - four(c)) < y - four(c)
    c = c + up.float()
    return torch.where((y > 0) & (c < 1), torch.ones_like(c), c).to(torch.uint8)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    if case['op'] == 'linear':
        b = 4 if case['dtype'] == 'f32' else 2
        M, N, K = case['M'], case['N'], case['K']
        if case['way'] == 'forward':
            moved = M * K + N * K + M * N * (1 + case['residual'] + case['keep']) + N * case['bias']
            return {'bytes': b * moved, 'flops': 2.0 * M * N * K}
        moved = 2 * (M * K + N * K) + M * N * (2 if case['act'] != 'none' else 1) + N * case['bias']
        return {'bytes': b * moved, 'flops': 4.0 * M * N * K}
    if case['op'] == 'loss':
        b = 4 if case['dtype'] == 'f32' else 2
        return {'bytes': 2.0 * b * case['R'] * case['C'] + 8 * case['R'], 'flops': 4.0 * case['R'] * case['C']}
    b, n = (4 if case['dtype'] == 'f32' else 2), float(sum(_sizes(case)))
    # weights in and out, gradients, both moments in and out; of 8-bit states also a block's two
    # scales in and out, and the values they stand for, which are written anew
    return {'bytes': n * (3 * b + 16) if case['bits'] == 32 else n * (3 * b + 4 + 16 / BLOCK + 8),
            'flops': 14 * n}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {'linear': _exact_linear, 'loss': _exact_loss, 'adamw': _exact_adamw}[case['op']](case, s)


def _exact_linear(case, s):
    x, w = s['x'].double(), s['w'].double()
    phi = lambda t: torch.special.ndtr(t)  # noqa: E731
    if case['way'] == 'forward':
        z = torch.einsum('mk,nk->mn', x, w)
        if case['bias']:
            z += s['b'].double()
        y = {'none': lambda: z, 'relu': lambda: torch.relu(z), 'gelu': lambda: z * phi(z),
             'silu': lambda: z * torch.sigmoid(z)}[case['act']]()
        y = y + s['r'].double() if case['residual'] else y
        return (y, z) if case['keep'] else y
    z = s['z'].double()
    slope = {'none': lambda: torch.ones_like(z), 'relu': lambda: torch.where(z > 0, 1.0, 0.0).double(),
             'gelu': lambda: phi(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi),
             'silu': lambda: torch.sigmoid(z) + z * torch.sigmoid(z) * torch.sigmoid(-z)}[case['act']]()
    dz = s['dy'].double() * slope
    return (torch.einsum('mn,nk->mk', dz, w), torch.einsum('mn,mk->nk', dz, x),
            torch.einsum('mn->n', dz) if case['bias'] else None)


def _exact_loss(case, s):
    R = case['R']
    grad = torch.empty((R, case['C']), dtype=torch.float64, device=DEV)
    live = s['labels'] != IGNORE
    n = max(1, int(live.sum()))
    total = 0.0
    for a in range(0, R, 1024):
        x, lab, on = s['logits'][a:a + 1024].double(), s['labels'][a:a + 1024], live[a:a + 1024]
        lp = torch.log_softmax(x, 1)
        rows = torch.nonzero(on)[:, 0]
        total += float(-lp[rows, lab[rows]].sum())
        p = torch.exp(lp)
        p[rows, lab[rows]] -= 1.0
        grad[a:a + 1024] = p * on[:, None] / n
    return torch.tensor(total / n, dtype=torch.float64, device=DEV), grad


def _exact_adamw(case, s):
    h, st = s['hyper'], s['state']
    t = st['step'] + 1
    b1, b2 = h['betas']
    total = st['m'].numel()
    g = torch.zeros(total, dtype=torch.float64, device=DEV)
    for x, at in zip(s['grads'], s['starts']):
        g[at:at + x.numel()] = x.reshape(-1).double()
    m, v = st['m'].double(), st['v'].double()
    if case['bits'] == 8:
        m = torch.sign(m) * (m / 127) ** 2 * st['m_scale'].double().repeat_interleave(BLOCK)
        v = (v / 255) ** 4 * st['v_scale'].double().repeat_interleave(BLOCK)
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    step = h['lr'] * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + h['eps'])
    new = [p.double() * (1 - h['lr'] * h['weight_decay']) - step[at:at + p.numel()].view(p.shape)
           for p, at in zip(s['params'], s['starts'])]
    if case['bits'] == 32:
        return new, m, v
    key = (s['noise'] * ROOT3 + t * ROOT2) % 2 ** 32
    x = torch.arange(total, device=DEV, dtype=torch.int64)
    x = ((x + key) % 2 ** 32 * GOLDEN) & MASK32
    for by, mul in ((16, ROOT2), (15, ROOT3)):
        x = ((x ^ (x >> by)) * mul) & MASK32
    x = x ^ (x >> 16)
    out = []
    for val, r, levels, power in ((m, x >> 16, 127, 2), (v, x & 0xFFFF, 255, 4)):
        top = val.abs().view(-1, BLOCK).amax(1).repeat_interleave(BLOCK)
        a = torch.where(top > 0, val.abs() / top, torch.zeros_like(val))
        low = torch.floor(a ** (1 / power) * levels + 1e-12).clamp(max=levels - 1)
        below, above = (low / levels) ** power, ((low + 1) / levels) ** power
        code = low + (r.double() / 65536 * (above - below) < a - below).double()
        if power == 4:
            code = torch.where((a > 0) & (code < 1), torch.ones_like(code), code)
        out.append(torch.sign(val) * (code / levels) ** power * top)
    return new, out[0], out[1]

"""AdamW over all tensors of a network in one launch, moments in 32 or 8 bits.

    m = b1 m + (1 - b1) g            v = b2 v + (1 - b2) g^2
    p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)

with t counted per parameter: the steps in which it had a gradient.

The moments of all tensors lie in one flat buffer; tensor i starts at
``offsets[i]``, a multiple of 256.  ``state_bits=8`` keeps codes with one
float32 scale per 256 elements (``m = s sgn(c) (c/127)^2``, ``v = s
(c/255)^4``): 2 bytes per weight instead of 8.  Codes are rounded up or down
with the probability that keeps a moment's mean, from a hash of the element's
place, the step t and ``seed``, so a run is repeatable.  A gradient that is not
finite makes its block of 256 moments NaN.

Weights are updated in place, in float32 arithmetic, rounded once to their own
type (float32, bfloat16, float16: in 16 bits a step below half a unit in the
last place is lost); gradients have the weights' type or float32.  A parameter
keeps the type, shape, device and contiguous layout that it had when the optimiser
was built; a step refuses (``ValueError``) one that a conversion of its module
has changed.  The step's constants are computed on the host, so a step refuses to be
captured in a CUDA graph (``RuntimeError``).
"""
from __future__ import annotations

import ctypes
from array import array

import torch

from . import _lib
from .linear import TYPES, type_of

BLOCK = 256
_MASK32 = 0xFFFFFFFF


class AdamW:
    """Optimiser of the CUDA tensors ``params`` (contiguous, one device)."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01,
                 state_bits=32, seed=0):
        self.params = list(params)
        if not self.params:
            raise ValueError('no parameters')
        if state_bits not in (8, 32):
            raise ValueError(f'state_bits {state_bits}: 8 or 32')
        if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1 and eps >= 0 and lr >= 0):
            raise ValueError(f'lr {lr}, betas {betas}, eps {eps}')
        self.lr, self.betas, self.eps, self.weight_decay = lr, tuple(betas), eps, weight_decay
        self.state_bits, self.seed, self.t = state_bits, int(seed), 0
        self._counts = [0] * len(self.params)  # of each parameter's own steps
        self.device = self.params[0].device
        self._types = [type_of(p, f'parameter {i}') for i, p in enumerate(self.params)]
        self._one_type = len(set(self._types)) == 1
        self._shapes = [p.shape for p in self.params]
        self._dtypes = [p.dtype for p in self.params]
        self._sizes, self.offsets, total = [], [], 0
        for i, p in enumerate(self.params):
            if p.device != self.device or not p.is_contiguous():
                raise ValueError(f'parameter {i}: must be contiguous on {self.device}')
            self.offsets.append(total)
            self._sizes.append(p.numel())
            total += -(-p.numel() // BLOCK) * BLOCK
        self._all = range(len(self.params))
        self._arrays = array('q', self._sizes), array('q', self.offsets)
        new = lambda n, dt: torch.zeros(n, dtype=dt, device=self.device)  # noqa: E731
        if state_bits == 32:
            self.m, self.v = new(total, torch.float32), new(total, torch.float32)
            self.m_scale = self.v_scale = None
        else:
            self.m, self.v = new(total, torch.int8), new(total, torch.uint8)
            self.m_scale = new(total // BLOCK, torch.float32)
            self.v_scale = new(total // BLOCK, torch.float32)

    def _opts(self, t):
        b1, b2 = self.betas
        return _lib.VcbAdamwOpts(b1, 1 - b1, b2, 1 - b2, self.eps, self.lr / (1 - b1 ** t),
                                 (1 - b2 ** t) ** -0.5, 1 - self.lr * self.weight_decay,
                                 (self.seed * 0xBB67AE85 + t * 0x6A09E667) & _MASK32)

    def step(self, grads=None):
        """One step with ``grads`` (by default every parameter's ``.grad``); a
        parameter whose gradient is None stays as it is, moments and step count
        (the t of its bias corrections) included."""
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError('AdamW.step cannot be captured in a CUDA graph: its constants go by '
                               'the step count on the host')
        ps = self.params
        grads = [p.grad for p in ps] if grads is None else list(grads)
        if len(grads) != len(ps):
            raise ValueError(f'{len(grads)} gradients for {len(ps)} parameters')
        self._check_params()
        groups = self._groups(grads)
        self.t += 1
        m, v = self.m.data_ptr(), self.v.data_ptr()
        ms, vs = _p(self.m_scale), _p(self.v_scale)
        step = _lib.lib().vcb_adamw
        counts = self._counts
        for pt, gt, t, idx, gp in groups:
            opts = self._opts(t)
            for i in idx:
                counts[i] = t
            if idx is self._all:
                pp, (sizes, offsets) = array('Q', [p.data_ptr() for p in ps]), self._arrays
            else:
                pp = array('Q', [ps[i].data_ptr() for i in idx])
                sizes = array('q', [self._sizes[i] for i in idx])
                offsets = array('q', [self.offsets[i] for i in idx])
            gp = array('Q', gp)
            rc = _lib.launch(self.device.index, step, len(gp), pp.buffer_info()[0],
                             gp.buffer_info()[0], sizes.buffer_info()[0],
                             offsets.buffer_info()[0], pt, gt, self.state_bits, m, v, ms, vs,
                             ctypes.byref(opts))
            if rc:
                _lib.check(rc, 'vcb_adamw')
        torch.autograd.graph.increment_version(ps)

    def _check_params(self):
        """A parameter keeps its identity when a module is converted or moved
        (its ``data`` is replaced): what the state was laid out for must still
        hold before a pointer is taken."""
        here = self.device.index
        if [p.dtype for p in self.params] == self._dtypes \
                and [p.shape for p in self.params] == self._shapes \
                and all([p.get_device() == here and p.is_contiguous() for p in self.params]):
            return
        for i, p in enumerate(self.params):
            if p.dtype != self._dtypes[i] or p.shape != self._shapes[i] \
                    or p.get_device() != here or not p.is_contiguous():
                raise ValueError(f'parameter {i}: {p.dtype} {tuple(p.shape)} strides {p.stride()} on '
                                 f'{p.device}, contiguous {self._dtypes[i]} '
                                 f'{tuple(self._shapes[i])} on {self.device} when this optimiser '
                                 'was built')

    def _groups(self, grads):
        """[(weights' type, gradients' type, step count, indices, gradient
        pointers)], one entry per launch."""
        here = self.device.index
        counts = self._counts
        if not any([g is None for g in grads]):  # usually one type, and nothing to copy
            first = grads[0].dtype
            if self._one_type and counts.count(counts[0]) == len(counts) and (first == torch.float32 or first == self._dtypes[0]) \
                    and [g.shape for g in grads] == self._shapes \
                    and all([g.dtype is first and g.get_device() == here and g.is_contiguous()
                             for g in grads]):
                return [(self._types[0], TYPES[first], counts[0] + 1, self._all,
                         [g.data_ptr() for g in grads])]
        groups = {}
        for i, (g, shape) in enumerate(zip(grads, self._shapes)):
            if g is None:
                continue
            if g.shape != shape or g.get_device() != here:
                raise ValueError(f'gradient {i}: {tuple(g.shape)} on {g.device}, expected '
                                 f'{tuple(shape)} on {self.device}')
            if not g.is_contiguous():
                grads[i] = g = g.contiguous()  # grads keeps it until the launch
            key = (self._types[i], g.dtype, counts[i] + 1)
            group = groups.get(key)
            if group is None:
                if g.dtype != torch.float32 and g.dtype != self._dtypes[i]:
                    raise _lib.UnsupportedInput(f'vibecheck_nn_b200: gradient {i} of type '
                                                f'{g.dtype}; the weight\'s or float32')
                group = groups[key] = (key[0], TYPES[g.dtype], key[2], [], [])
            group[3].append(i)
            group[4].append(g.data_ptr())
        return groups.values()

    def moments(self):
        """(m, v) of all tensors as flat float32 buffers (the state itself
        with 32-bit states, the values the codes stand for with 8-bit ones)."""
        if self.state_bits == 32:
            return self.m, self.v
        n = self.m.numel()
        m = torch.empty(n, dtype=torch.float32, device=self.device)
        v = torch.empty(n, dtype=torch.float32, device=self.device)
        rc = _lib.launch(self.device.index, _lib.lib().vcb_adamw_values, n, self.m.data_ptr(),
                         self.v.data_ptr(), self.m_scale.data_ptr(), self.v_scale.data_ptr(),
                         m.data_ptr(), v.data_ptr())
        _lib.check(rc, 'vcb_adamw_values')
        return m, v

    def _buffers(self):
        names = ('m', 'v') if self.state_bits == 32 else ('m', 'v', 'm_scale', 'v_scale')
        return {k: getattr(self, k) for k in names}

    def state_dict(self):
        """The step counts (of the optimiser and of each parameter), the seed and
        copies of the state's buffers."""
        return {'step': self.t, 'steps': list(self._counts), 'seed': self.seed,
                **{k: t.clone() for k, t in self._buffers().items()}}

    def load_state_dict(self, state):
        """Takes over a state of the same tensors and ``state_bits``; one without
        ``steps`` counts ``step`` for every parameter."""
        counts = [int(n) for n in state.get('steps', [state['step']] * len(self.params))]
        if len(counts) != len(self.params):
            raise ValueError(f'state of {len(counts)} parameters, expected {len(self.params)}')
        for k, t in self._buffers().items():
            s = state[k]
            if s.shape != t.shape or s.dtype != t.dtype:
                raise ValueError(f'state {k}: {s.dtype} {tuple(s.shape)}, expected {t.dtype} '
                                 f'{tuple(t.shape)}')
        for k, t in self._buffers().items():
            t.copy_(state[k])
        self.t, self._counts = int(state['step']), counts
        self.seed = int(state.get('seed', self.seed))


def _p(t):
    return None if t is None else t.data_ptr()

"""Linear layer with its epilogue, and its gradients: the layers of a network
that is trained here and bounded by the rest of the package.

* ``linear_forward`` -- ``y = act(x W^T + b) + r`` in one product; with
  ``keep`` also the pre-activation ``z = x W^T + b`` for the backward pass;
* ``linear_backward`` -- ``dz = dy * act'(z)``, ``dx = dz W``, ``dW = dz^T x``
  and ``db``;
* ``linear`` -- the same for autograd, differentiable once.

``x`` is (..., K), ``weight`` (N, K) as in a ``gg`` dict's fc layer.  float32,
bfloat16 and float16, one type per call; sums are held in float32 and each
output is rounded once.  In float32 a product keeps float32 accuracy: entries are
split into three bfloat16 parts, not rounded, for the tensor cores, and an output's
error goes by its own sum of |x w|, whatever else lies in the rows (entries below
2^-110 are held to 2^-134).  An entry that is not finite makes the outputs that it
meets infinite or NaN.  ``act`` is one of 'none',
'relu', 'gelu' (with erf) and 'silu'; a ReLU's slope at 0 is 0.  Work runs on
the current stream of ``x``'s device; like the tensor-core bounds, a caller
can ask ``_lib.fault_check`` whether a bounded device wait ran out.
"""
from __future__ import annotations

import functools
import struct

import torch

from . import _lib

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
# argument lists of the packed entry points
_FORWARD, _BACKWARD = struct.Struct('19q').pack, struct.Struct('21q').pack
ACTS = {'none': 0, 'relu': 1, 'gelu': 2, 'silu': 3}


def type_of(t, name):
    """vcb_dtype of a CUDA tensor; refuses what the kernels do not take."""
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        _lib.require_cuda(t, name)
    code = TYPES.get(t.dtype)
    if code is None:
        raise _lib.UnsupportedInput(f'vibecheck_nn_b200: {name} must be float32, bfloat16 or '
                                    f'float16 (got {t.dtype})')
    return code


def rows_of(t, cols, like, name):
    """``t`` (..., cols) as rows with unit column stride -> (tensor, row
    stride); copies only what no row stride describes."""
    if t.dtype != like.dtype or t.get_device() != like.get_device():
        raise ValueError(f'{name}: {t.dtype} on {t.device}, expected {like.dtype} on {like.device}')
    dim = t.dim()
    if dim < 1 or t.shape[-1] != cols:
        raise ValueError(f'{name}: shape {tuple(t.shape)}, expected (..., {cols})')
    if ((t.shape[0] if dim == 2 else t.shape[:-1].numel()) | cols) >> 31:
        raise _lib.UnsupportedInput(f'vibecheck_nn_b200: {name} {tuple(t.shape)}: rows and columns '
                                    'are counted in 32 bits')
    if dim == 2 and t.is_contiguous():
        return t, cols
    if dim != 2:
        t = t.reshape(t.shape[:-1].numel(), cols)
    rows = t.shape[0]
    ld = t.stride(0) if rows > 1 else cols
    if (cols > 1 and t.stride(1) != 1) or ld < cols:
        t = t.contiguous()
        ld = cols
    return t, ld


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(entry, *sizes):
    return getattr(_lib.lib(), entry)(*sizes)


def _act(act):
    code = ACTS.get(act)
    if code is None:
        raise ValueError(f'act {act!r}: one of {sorted(ACTS)}')
    return code


def _weight(x, weight):
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        raise ValueError('weight must be (N, K)')
    return weight.shape


def linear_forward(x, weight, bias=None, act='none', residual=None, keep=False):
    """``act(x W^T + bias) + residual``, shape (..., N); with ``keep`` the pair
    (y, z)."""
    ty = type_of(x, 'x')
    code = _act(act)
    N, K = _weight(x, weight)
    x2, ldx = rows_of(x, K, x, 'x')
    w2, ldw = rows_of(weight, K, x, 'weight')
    M = x2.shape[0]
    flat = x2.dim() == x.dim()
    if bias is not None:
        bias = _vector(bias, N, x, 'bias')
    r2, ldr = None, 0
    if residual is not None:
        if residual.shape[:-1] != x.shape[:-1]:
            raise ValueError(f'residual: shape {tuple(residual.shape)}, expected '
                             f'{(*x.shape[:-1], N)}')
        r2, ldr = rows_of(residual, N, x, 'residual')
    y = x.new_empty((M, N))
    z = x.new_empty((M, N)) if keep else None
    xp, wp = x2.data_ptr(), w2.data_ptr()
    size = x.element_size()
    nbytes = _workspace_bytes('vcb_linear_forward_workspace', M, N, K, ty,
                              not (xp | wp | ldx * size | ldw * size) & 15)
    ws = _lib.workspace(nbytes, x.device)
    rc = _lib.launch_packed(x.get_device(), _lib.lib().vcb_linear_forward_packed, _FORWARD,
                            M, N, K, ty, xp, ldx, wp, ldw, _p(bias), code, _p(r2), ldr,
                            y.data_ptr(), N, _p(z), N, _p(ws), nbytes)
    if rc:
        _lib.check(rc, 'vcb_linear_forward')
    if not flat:
        y = y.view(*x.shape[:-1], N)
        z = z.view(*x.shape[:-1], N) if keep else None
    return (y, z) if keep else y


def linear_backward(dy, x, weight, z=None, act='none', bias=True, need=(True, True)):
    """Gradients (dx, dW, db) of ``linear_forward`` for the upstream ``dy``
    (..., N); ``z`` is the pre-activation (not needed for act 'none').  db is
    None unless ``bias``; ``need`` switches dx and dW off.  The residual's
    gradient is ``dy`` itself."""
    ty = type_of(x, 'x')
    code = _act(act)
    N, K = _weight(x, weight)
    if dy.shape[:-1] != x.shape[:-1] or dy.shape[-1:] != (N,):
        raise ValueError(f'dy: shape {tuple(dy.shape)}, expected {(*x.shape[:-1], N)}')
    g2, ldg = rows_of(dy, N, x, 'dy')
    x2, ldx = rows_of(x, K, x, 'x')
    w2, ldw = rows_of(weight, K, x, 'weight')
    z2, ldz = None, 0
    if code:
        if z is None or z.shape != dy.shape:
            raise ValueError(f'act {act!r} needs z of shape {tuple(dy.shape)}')
        z2, ldz = rows_of(z, N, x, 'z')
    M = x2.shape[0]
    dx = x.new_empty((M, K)) if need[0] else None
    dw = x.new_empty((N, K)) if need[1] else None
    db = x.new_empty((N,)) if bias else None
    gp, xp, wp = g2.data_ptr(), x2.data_ptr(), w2.data_ptr()
    size = x.element_size()
    nbytes = _workspace_bytes('vcb_linear_backward_workspace', M, N, K, ty, code,
                              not (gp | xp | wp | (ldg | ldx | ldw) * size) & 15)
    ws = _lib.workspace(nbytes, x.device)
    rc = _lib.launch_packed(x.get_device(), _lib.lib().vcb_linear_backward_packed, _BACKWARD,
                            M, N, K, ty, gp, ldg, xp, ldx, wp, ldw, _p(z2), ldz, code, _p(dx), K,
                            _p(dw), K, _p(db), _p(ws), nbytes)
    if rc:
        _lib.check(rc, 'vcb_linear_backward')
    if dx is not None and x.dim() != 2:
        dx = dx.view(x.shape)
    return dx, dw, db


def _vector(t, n, like, name):
    if t.dtype != like.dtype or t.get_device() != like.get_device() or t.shape != (n,):
        raise ValueError(f'{name}: {t.dtype} {tuple(t.shape)} on {t.device}, expected '
                         f'{like.dtype} ({n},) on {like.device}')
    return t.contiguous()


def _p(t):
    return 0 if t is None else t.data_ptr()


class _Refuse(torch.autograd.Function):
    @staticmethod
    def forward(ctx, anchor, what, *outs):
        ctx.what = what
        return outs

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(f'vibecheck_nn_b200: {ctx.what} is differentiable once (its gradients '
                           'come from kernels that autograd does not see)')


def first_order(what, outs):
    """Gradients ``outs`` (tensors or None) of ``what``: where a graph of the
    backward pass is asked for, a second derivative through them raises instead of
    missing its terms."""
    if not torch.is_grad_enabled():
        return outs
    anchor = torch.zeros((), requires_grad=True)
    made = iter(_Refuse.apply(anchor, what, *[t for t in outs if t is not None]))
    return tuple(None if t is None else next(made) for t in outs)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, act, residual):
        keep = act != 'none' and any(ctx.needs_input_grad[:3])
        out = linear_forward(x, weight, bias, act, residual, keep)
        y, z = out if keep else (out, None)
        ctx.act = act
        ctx.save_for_backward(x, weight, z)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, weight, z = ctx.saved_tensors
        gx, gw, gb = ctx.needs_input_grad[:3]
        dx = dw = db = None
        if gx or gw or gb:
            with torch.no_grad():
                outs = linear_backward(dy, x, weight, z, ctx.act, gb, (gx, gw))
            dx, dw, db = first_order('linear', outs)
        return dx, dw, db, None, dy if ctx.needs_input_grad[4] else None


def linear(x, weight, bias=None, act='none', residual=None):
    """``linear_forward``, differentiable once (gradients of x, weight, bias and
    residual; a second derivative through them raises ``RuntimeError``)."""
    return _Linear.apply(x, weight, bias, act, residual)

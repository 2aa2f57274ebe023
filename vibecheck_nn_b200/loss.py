"""Softmax cross-entropy with its gradient in one pass over the logits.

* ``cross_entropy_grad`` -- (loss, dlogits) of the mean over labelled rows;
* ``cross_entropy`` -- the same loss for autograd, differentiable once.

Logits (..., C) in float32, bfloat16 or float16, int64 labels (...).  Rows
labelled ``ignore_index`` count for nothing and get gradient 0; with no
labelled row the loss is 0.  A row whose logits are all ``-inf`` has loss
``inf`` and gradient 0.  Labels are not read back to the host: one outside
[0, C) makes its row's gradient and the loss NaN.

``cross_entropy`` reads the logits once for the loss; its backward pass makes
the gradient from them, times the upstream factor, before the one rounding to
their type: a loss scale reaches entries that float16 alone would lose.
"""
from __future__ import annotations

import struct

import torch

from . import _lib
from .linear import _p, _workspace_bytes, first_order, rows_of, type_of

_ARGS = struct.Struct('14q').pack


def _run(logits, labels, ignore_index, scale=None, want_loss=True, want_grad=True):
    """(loss or None, gradient times ``scale`` (a device scalar) or None)."""
    ty = type_of(logits, 'logits')
    shape = logits.shape
    if not shape or shape[-1] == 0:
        raise ValueError(f'logits: shape {tuple(shape)}, expected (..., C) with C > 0')
    dev = logits.get_device()
    if not isinstance(labels, torch.Tensor) or labels.dtype != torch.int64 \
            or labels.get_device() != dev or labels.shape != shape[:-1]:
        raise ValueError(f'labels must be int64 {tuple(shape[:-1])} on {logits.device}')
    C = shape[-1]
    x2, ld = rows_of(logits, C, logits, 'logits')
    labels = labels.contiguous()
    R = x2.shape[0]
    grad = logits.new_empty((R, C)) if want_grad else None
    loss = logits.new_empty((), dtype=torch.float32) if want_loss else None
    nbytes = _workspace_bytes('vcb_cross_entropy_workspace', R, C)
    ws = _lib.workspace(nbytes, logits.device)
    rc = _lib.launch_packed(dev, _lib.lib().vcb_cross_entropy_scaled_packed, _ARGS, R, C, ty,
                            x2.data_ptr(), ld, labels.data_ptr(), int(ignore_index), _p(scale),
                            _p(loss), _p(grad), C, _p(ws), nbytes)
    if rc:
        _lib.check(rc, 'vcb_cross_entropy')
    return loss, grad if grad is None or len(shape) == 2 else grad.view(shape)


def cross_entropy_grad(logits, labels, ignore_index=-100):
    """(loss, d loss / d logits): loss a float32 scalar on the device, the
    gradient in the logits' type and shape."""
    return _run(logits, labels, ignore_index)


class _CrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, ignore_index):
        ctx.ignore_index = ignore_index
        ctx.save_for_backward(logits, labels)
        return _run(logits, labels, ignore_index, want_grad=False)[0]

    @staticmethod
    def backward(ctx, g):
        logits, labels = ctx.saved_tensors
        with torch.no_grad():
            out = _run(logits, labels, ctx.ignore_index, g.float(), want_loss=False)[1:]
        return (*first_order('cross_entropy', out), None, None)


def cross_entropy(logits, labels, ignore_index=-100):
    """Mean cross-entropy over the labelled rows, differentiable once (a second
    derivative through its gradient raises ``RuntimeError``)."""
    return _CrossEntropy.apply(logits, labels, ignore_index)

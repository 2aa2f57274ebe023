"""Sizes that 32 bits do not hold: the packed entry points of the training-step operators carry
64 bits per argument, and a size may not be cut on the way."""
import struct

import pytest
import torch

from vibecheck_nn_b200 import _lib, linear, loss

P = 1 << 12  # a pointer that is never dereferenced


def forward(M, N, K):
    return _lib.lib().vcb_linear_forward_packed(struct.pack(
        '19q', M, N, K, 0, P, K, P, K, 0, 0, 0, 0, P, N, 0, 0, 0, 0, 0))


def backward(M, N, K):
    return _lib.lib().vcb_linear_backward_packed(struct.pack(
        '21q', M, N, K, 0, P, N, P, K, P, K, 0, 0, 0, P, K, P, K, P, 0, 0, 0))


def cross_entropy(R, C):
    return _lib.lib().vcb_cross_entropy_packed(struct.pack(
        '13q', R, C, 0, P, C, P, -100, P, P, C, 0, 0, 0))


@pytest.mark.parametrize('size', [1 << 32, 1 << 31, (1 << 33) + (1 << 32), -(1 << 32)])
def test_c_refuses_sizes_that_32_bits_do_not_hold(size):
    """Cut to 32 bits each would be 0 (nothing to do) or negative."""
    for at in range(3):
        sizes = [4, 4, 4]
        sizes[at] = size
        if at < 2:  # K = 0 is work: one column of biases
            assert forward(*sizes) == _lib.VCB_ERR_UNSUPPORTED
    assert backward(4, 4, size) == _lib.VCB_ERR_UNSUPPORTED
    assert forward(0, 4, size) == _lib.VCB_ERR_UNSUPPORTED
    assert cross_entropy(4, size) == _lib.VCB_ERR_UNSUPPORTED
    assert cross_entropy(size, 4) == _lib.VCB_ERR_UNSUPPORTED
    for act in (size, 1 << 32):
        args = [0, 4, 4, 0, P, 4, P, 4, 0, act, 0, 0, P, 4, 0, 0, 0, 0, 0]
        assert _lib.lib().vcb_linear_forward_packed(struct.pack('19q', *args)) \
            == _lib.VCB_ERR_UNSUPPORTED


@pytest.mark.parametrize('shape', [((1 << 32) + 5, 2), (2, 1 << 31), (1 << 16, 1 << 16, 2)])
def test_python_refuses_them_before_it_allocates(shape, monkeypatch):
    x = torch.empty(shape, device='meta')
    monkeypatch.setattr(linear, 'type_of', lambda t, name: 0)
    monkeypatch.setattr(loss, 'type_of', lambda t, name: 0)
    w = torch.empty(3, shape[-1], device='meta')
    labels = torch.empty(shape[:-1], dtype=torch.int64, device='meta')
    for call in (lambda: linear.linear_forward(x, w),
                 lambda: linear.linear_backward(x.new_empty(*shape[:-1], 3), x, w),
                 lambda: linear.linear_forward(w, x.reshape(-1, shape[-1])),
                 lambda: loss.cross_entropy_grad(x, labels)):
        with pytest.raises(_lib.UnsupportedInput, match='32 bits'):
            call()

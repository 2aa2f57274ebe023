"""CPU checks of the training-step operators: refusals and size queries, before
any kernel runs."""
import ctypes

import pytest
import torch

from vibecheck_nn_b200 import _lib, linear, loss, optim


def test_cpu_tensors_are_refused():
    x, w = torch.ones(2, 4), torch.ones(3, 4)
    for call in (lambda: linear.linear_forward(x, w),
                 lambda: linear.linear_backward(torch.ones(2, 3), x, w),
                 lambda: linear.linear(x, w),
                 lambda: loss.cross_entropy_grad(x, torch.zeros(2, dtype=torch.int64)),
                 lambda: loss.cross_entropy(x, torch.zeros(2, dtype=torch.int64)),
                 lambda: optim.AdamW([x])):
        with pytest.raises(_lib.UnsupportedInput):
            call()


def test_c_abi_refuses_before_it_touches_memory():
    lib = _lib.lib()
    p = 4096  # never dereferenced
    bad = [
        lib.vcb_linear_forward(2, 3, 4, 0, None, 4, p, 4, None, 0, None, 0, p, 3, None, 0, None, 0,
                               None),
        lib.vcb_linear_forward(2, 3, 4, 3, p, 4, p, 4, None, 0, None, 0, p, 3, None, 0, None, 0,
                               None),
        lib.vcb_linear_forward(2, 3, 4, 0, p, 4, p, 4, None, 4, None, 0, p, 3, None, 0, None, 0,
                               None),
        lib.vcb_linear_forward(-1, 3, 4, 0, p, 4, p, 4, None, 0, None, 0, p, 3, None, 0, None, 0,
                               None),
        lib.vcb_linear_forward(2, 3, 4, 0, p + 2, 4, p, 4, None, 0, None, 0, p, 3, None, 0, None, 0,
                               None),
        lib.vcb_linear_forward(2, 3, 4, 0, p, 4, p, 4, None, 0, p, 2, p, 3, None, 0, None, 0, None),
        lib.vcb_linear_forward(4096, 4096, 4096, 0, p, 4096, p, 4096, None, 0, None, 0, p, 4096,
                               None, 0, None, 0, None),  # no workspace
        lib.vcb_linear_backward(2, 3, 4, 0, p, 3, p, 4, p, 4, None, 0, 1, p, 4, p, 4, p, None, 0,
                                None),  # an activation without z
        lib.vcb_linear_backward(2, 3, 4, 0, p, 2, p, 4, p, 4, None, 0, 0, p, 4, p, 4, p, None, 0,
                                None),
        lib.vcb_cross_entropy(2, 0, 0, p, 4, p, -100, p, p, 4, None, 0, None),
        lib.vcb_cross_entropy(2, 4, 0, p, 3, p, -100, p, p, 4, None, 0, None),
        lib.vcb_cross_entropy(4000, 4, 0, p, 4, p, -100, p, p, 4, None, 0, None),
        lib.vcb_adamw_values(100, p, p, p, p, p, p, None),
        lib.vcb_adamw_values(256, None, p, p, p, p, p, None),
    ]
    assert bad == [_lib.VCB_ERR_INVALID] * len(bad), bad
    opts = _lib.VcbAdamwOpts()
    one = (ctypes.c_int64 * 1)
    ptr, n, off = one(p), one(4), one(100)
    adr = ctypes.addressof
    for bits, o in ((32, off), (16, one(0))):
        assert lib.vcb_adamw(1, adr(ptr), adr(ptr), adr(n), adr(o), 0, 0, bits, p, p, None, None,
                             ctypes.byref(opts), None) == _lib.VCB_ERR_INVALID
    assert lib.vcb_adamw(1, adr(ptr), adr(ptr), adr(n), adr(one(0)), 0, 0, 8, p, p, None, None,
                         ctypes.byref(opts), None) == _lib.VCB_ERR_INVALID  # no scales
    assert lib.vcb_adamw(1, adr(ptr), adr(ptr), adr(n), adr(one(0)), 0, 1, 32, p, p, None, None,
                         ctypes.byref(opts), None) == _lib.VCB_ERR_INVALID  # 16-bit gradient


def test_nothing_to_do_is_ok():
    lib = _lib.lib()
    assert lib.vcb_linear_forward(0, 3, 4, 0, None, 4, None, 4, None, 0, None, 0, None, 3, None, 0,
                                  None, 0, None) == _lib.VCB_OK
    opts = _lib.VcbAdamwOpts()
    assert lib.vcb_adamw(0, None, None, None, None, 0, 0, 32, None, None, None, None,
                         ctypes.byref(opts), None) == _lib.VCB_OK
    assert lib.vcb_adamw_values(0, None, None, None, None, None, None, None) == _lib.VCB_OK


def test_workspace_queries():
    lib = _lib.lib()
    f, b = lib.vcb_linear_forward_workspace, lib.vcb_linear_backward_workspace
    assert f(1, 50, 50, 0, 0) == 0 and f(4096, 4096, 4096, 1, 1) == 0
    # copies of both operands, rows padded to 8 elements
    assert f(256, 1000, 1001, 1, 0) >= 2 * 1008 * (256 + 1000)
    # two halves of both operands
    assert f(4096, 4096, 4096, 0, 1) >= 4 * 4096 * 4096 * 2
    assert b(4096, 4096, 4096, 1, 0, 1) == 0
    assert b(4096, 4096, 4096, 1, 1, 1) >= 2 * 4096 * 4096
    assert b(4096, 4096, 4096, 0, 1, 1) >= 4 * 4 * 4096 * 4096
    assert lib.vcb_cross_entropy_workspace(100, 10) == 0
    assert lib.vcb_cross_entropy_workspace(10000, 10) >= 10000 * 8

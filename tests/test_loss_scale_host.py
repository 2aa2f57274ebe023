"""Which arguments the scaled loss refuses before it touches memory."""
from vibecheck_nn_b200 import _lib

P = 4096  # never dereferenced


def test_refusals():
    f = _lib.lib().vcb_cross_entropy_scaled
    bad = [f(2, 0, 0, P, 4, P, -100, None, P, P, 4, None, 0, None),       # no classes
           f(2, 4, 0, P, 3, P, -100, None, P, P, 4, None, 0, None),       # rows overlap
           f(2, 4, 0, P, 4, P, -100, None, P, P, 3, None, 0, None),
           f(2, 4, 7, P, 4, P, -100, None, P, P, 4, None, 0, None),       # no such type
           f(2, 4, 0, None, 4, P, -100, P, P, None, 0, None, 0, None),
           f(2, 4, 0, P, 4, None, -100, P, P, None, 0, None, 0, None),
           f(2, 4, 0, P + 2, 4, P, -100, P, P, None, 0, None, 0, None),
           f(4000, 4, 0, P, 4, P, -100, P, P, P, 4, None, 0, None)]       # no workspace
    assert bad == [_lib.VCB_ERR_INVALID] * len(bad), bad
    plain = _lib.lib().vcb_cross_entropy                                   # wants both
    assert plain(2, 4, 0, P, 4, P, -100, None, P, 4, None, 0, None) == _lib.VCB_ERR_INVALID
    assert plain(2, 4, 0, P, 4, P, -100, P, None, 4, None, 0, None) == _lib.VCB_ERR_INVALID
    assert f(0, 4, 0, None, 4, None, -100, None, None, None, 0, None, 0, None) == _lib.VCB_OK

"""What im_moe_route_ex and the router's score bias refuse, and the wait limit, without a GPU."""
from __future__ import annotations

from ironmule_b200 import _lib


def _status(name, *args):
    lib = _lib.load()
    return getattr(lib, name)(*args), lib.im_last_error().decode()


def route(scoring=0, bias=None, error=None, ptr=256, m=4):
    return _status("im_moe_route_ex", ptr, 0, m, 8, 8, bias, 2, scoring, 1, 1.0, ptr, ptr, ptr, ptr, ptr, 1 << 20, error,
                   None)


def test_route_ex_refusals():
    for scoring in (2, 3, 18, 32, -1):
        rc, msg = route(scoring=scoring, bias=256)
        assert rc == _lib.IM_INVALID and "scoring" in msg, scoring
    for scoring in (_lib.MOE_SOFTMAX, _lib.MOE_SIGMOID):
        rc, msg = route(scoring=scoring + _lib.MOE_BIAS_ON_SCORE)
        assert rc == _lib.IM_INVALID and "needs bias" in msg
    rc, msg = route(error=258)
    assert rc == _lib.IM_INVALID and "error word" in msg
    rc, msg = route(ptr=None)
    assert rc == _lib.IM_INVALID and "null" in msg


def test_wait_limit():
    lib = _lib.load()
    was = lib.im_set_wait_limit(5)
    try:
        assert was == 1_000_000_000
        assert lib.im_set_wait_limit(-1) == 5  # changes nothing
        assert lib.im_set_wait_limit(7) == 5
    finally:
        assert lib.im_set_wait_limit(was) == 7

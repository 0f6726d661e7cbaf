"""The mixture-of-experts entry points without a GPU: refusals with a status and a message, launching nothing, and the
sizes of plans and packed weights."""
from __future__ import annotations

from ironmule_b200 import _lib


def _status(name, *args):
    lib = _lib.load()
    return getattr(lib, name)(*args), lib.im_last_error().decode()


def route(m=4, e=8, ld=8, k=2, scoring=0, ptr=256, plan_bytes=1 << 20):
    return _status("im_moe_route", ptr, 0, m, e, ld, None, k, scoring, 1, 1.0, ptr, ptr, ptr, ptr, ptr,
                   plan_bytes, None)


def test_route_refusals():
    assert route(k=9)[0] == _lib.IM_INVALID
    assert route(k=0)[0] == _lib.IM_INVALID
    assert route(m=-1)[0] == _lib.IM_INVALID
    rc, msg = route(ld=7)
    assert rc == _lib.IM_INVALID and "stride" in msg
    rc, msg = route(e=600, ld=600)
    assert rc == _lib.IM_UNSUPPORTED and "512 experts" in msg
    rc, msg = route(e=64, ld=64, k=33)
    assert rc == _lib.IM_UNSUPPORTED and "places" in msg
    rc, msg = route(scoring=2)
    assert rc == _lib.IM_INVALID and "scoring" in msg
    rc, msg = route(ptr=None)
    assert rc == _lib.IM_INVALID and "null" in msg
    rc, msg = route(ptr=8)
    assert rc == _lib.IM_INVALID and "misaligned" in msg
    rc, msg = route(plan_bytes=4)
    assert rc == _lib.IM_INVALID and "plan of" in msg


def test_plan_sizes():
    lib = _lib.load()
    assert lib.im_moe_plan_bytes(0, 8, 2) >= 32
    assert lib.im_moe_plan_bytes(1, 600, 2) == 0 and lib.im_moe_plan_bytes(1, 8, 9) == 0
    # every expert can end in a part-filled item: one item per non-empty bucket and one per full item of 128
    for m, e, k in [(1, 128, 8), (5, 128, 8), (64, 8, 8), (65, 8, 2), (8192, 128, 8), (1 << 22, 512, 32)]:
        pairs = m * k
        items = 16 * (min(pairs, e + 1) + pairs // 128)
        assert 32 + items <= lib.im_moe_plan_bytes(m, e, k) <= 32 + items + 8 * pairs + 4 * 296 * (e + 1)
    assert lib.im_moe_packed_bytes(3, 33, 128) == 3 * (2 * 4608 + 512 + 8)  # 128-output blocks of 64-wide groups, maxima
    assert lib.im_moe_packed_bytes(3, 33, 100) == 0
    assert lib.im_moe_mlp_workspace_bytes(4, 8, 2, 128, 64) >= 8 * (128 + 64) * 2
    assert lib.im_moe_mlp_workspace_bytes(4, 8, 2, 100, 64) == 0
    assert lib.im_moe_grouped_workspace_bytes(4, 8, 2, 128) >= 8 * 128 * 2


def test_product_refusals():
    args = lambda m=4, n=32, k=64, x=256, plan=256, size=1 << 20, wsize=1 << 20: (  # noqa: E731
        "im_moe_grouped_qgemm", 256, x, 256, m, 8, 2, n, k, 0, 256, plan, size, 256, wsize, None)
    rc, msg = _status(*args(k=100))
    assert rc == _lib.IM_INVALID and "K=100" in msg
    rc, msg = _status(*args(x=None))
    assert rc == _lib.IM_INVALID and "null" in msg
    rc, msg = _status(*args(x=8))
    assert rc == _lib.IM_INVALID and "aligned" in msg
    rc, msg = _status(*args(plan=None))
    assert rc == _lib.IM_INVALID and "plan" in msg
    rc, msg = _status(*args(size=8))
    assert rc == _lib.IM_INVALID and "plan of" in msg
    rc, msg = _status(*args(wsize=8))
    assert rc == _lib.IM_INVALID and "workspace of" in msg
    assert _status(*args(m=0, x=None, plan=None))[0] == _lib.IM_OK
    mlp = lambda h=128, i=64, act=2, ws=256, size=1 << 20: (  # noqa: E731
        "im_moe_mlp", 256, 256, 256, 256, 4, 8, 2, h, i, act, 256, 256, 1 << 20, ws, size, None)
    assert _status(*mlp(h=100))[0] == _lib.IM_INVALID
    assert _status(*mlp(i=100))[0] == _lib.IM_INVALID
    rc, msg = _status(*mlp(act=1))
    assert rc == _lib.IM_INVALID and "activation" in msg
    rc, msg = _status(*mlp(size=8))
    assert rc == _lib.IM_INVALID and "workspace" in msg
    rc, msg = _status("im_moe_pack_w4g64", 256, 256, 256, 0, 32, 64, 256, None)
    assert rc == _lib.IM_INVALID


def test_block_refusals():
    def block(places=1, weights=None, h=256, m=4, hsz=128, col=0, z=256, nxt=256):
        return _status("im_block_residual", 256, weights, places, h, None, None, 0, col, 1.0, nxt, 1e-6, 0, m, hsz, 256,
                       z, None, None)

    rc, msg = block(places=2)
    assert rc == _lib.IM_INVALID and "weights" in msg
    assert block(places=33, weights=256)[0] == _lib.IM_UNSUPPORTED
    assert block(hsz=20000)[0] == _lib.IM_UNSUPPORTED
    assert block(hsz=0)[0] == _lib.IM_INVALID
    assert block(col=2)[0] == _lib.IM_INVALID
    rc, msg = block(h=None)
    assert rc == _lib.IM_INVALID and "null" in msg
    rc, msg = block(z=None)
    assert rc == _lib.IM_INVALID and "null" in msg
    assert block(m=0, h=None)[0] == _lib.IM_OK

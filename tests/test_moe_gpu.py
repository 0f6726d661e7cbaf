"""The mixture-of-experts operators against float64: routing (exact whole numbers), products by expert, the gated MLP,
and the block residual; at ragged sizes, with closed experts, empty experts, rows without any expert, and one to many
rows.

Tolerances, from the arithmetic. An output is rounded once to bf16: 2^-9 of it, taken as 2^-8. The products expand
4-bit codes exactly and accumulate in float32; s * sum((128 + q) x) and (b - 128 s) * sum(x) cancel, so their rounding
counts against A = sum |x| (143 s + |b|): 2^-21 A covers the accumulation at these lengths. Where weights are taken as
fp16 scale * q + bias, each is off by 2^-12 of itself at most: 2^-12 sum |x| |w|. The MLP's hidden activations add
their own rounding (2^-8) and the first products' errors times the activation's slope (at most 1.13)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from ironmule_b200 import _lib, kernels

pytestmark = pytest.mark.gpu


def quantised(gen, e, n, k, device):
    w = torch.randint(-2**31, 2**31, (e, n, k // 8), generator=gen, device=device, dtype=torch.int64).to(torch.int32)
    s = (0.005 * (0.5 + torch.rand((e, n, k // 64), generator=gen, device=device))).to(torch.bfloat16)
    b = (-7.0 * s.float() + 0.003 * torch.randn((e, n, k // 64), generator=gen, device=device)).to(torch.bfloat16)
    return w, s, b


def dense(q, e):
    """Expert e in float64, and the magnitudes 143 |s| + |b| that its accumulation runs through."""
    w, s, b = (t[e] for t in q)
    codes = torch.stack([(w >> (4 * i)) & 15 for i in range(8)], dim=2).flatten(1).double()
    s, b = (t.double().repeat_interleave(64, 1) for t in (s, b))
    return codes * s + b, 143.0 * s.abs() + b.abs()


def product(x, q, e):
    """x W^T in float64 and the bound on the error of its float32 value."""
    w, mag = dense(q, e)
    xd = x.double()
    return xd @ w.T, 2**-12 * (xd.abs() @ w.abs().T) + 2**-21 * (xd.abs() @ mag.T)


def route_reference(logits, top_k, scoring, normalise, scale, bias):
    v = logits.float().cpu().numpy()
    key = v if bias is None else v + bias.cpu().numpy()
    closed = np.isnan(v) | np.isneginf(v)
    key = np.where(closed, -np.inf, key)
    order = np.argsort(-key, axis=1, kind="stable")[:, :top_k]
    live = ~np.take_along_axis(closed, order, 1)
    ids = np.where(live, order, -1).astype(np.int32)
    v = np.where(closed, -np.inf, v).astype(np.float64)
    chosen = np.take_along_axis(v, order, 1)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        if scoring == "softmax":
            top = v.max(axis=1, keepdims=True)
            p = np.exp(chosen - top)
            total = np.where(live, p, 0).sum(axis=1, keepdims=True) if normalise else np.exp(v - top).sum(1, keepdims=True)
        else:
            p = 1.0 / (1.0 + np.exp(-chosen))
            total = np.where(live, p, 0).sum(axis=1, keepdims=True) if normalise else 1.0
        w = np.where(live, p / total * scale, 0.0)
    bucket = np.where(live, ids, logits.shape[1]).ravel()
    pairs = np.argsort(bucket, kind="stable").astype(np.int32)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(bucket, minlength=logits.shape[1] + 1))]).astype(np.int32)
    return ids, w, offsets, pairs


def check_route(logits, top_k, scoring="softmax", normalise=True, scale=1.0, bias=None):
    r = kernels.moe_route(logits, top_k, scoring=scoring, normalise=normalise, scale=scale, bias=bias)
    ids, w, offsets, pairs = route_reference(logits, top_k, scoring, normalise, scale, bias)
    assert np.array_equal(r.ids.cpu().numpy(), ids)
    assert np.array_equal(r.offsets.cpu().numpy(), offsets)
    assert np.array_equal(r.pairs.cpu().numpy(), pairs)
    # float32: an exponential of 2 ulps and a sum of up to 512 such terms in a tree, then a quotient
    np.testing.assert_allclose(r.weights.cpu().numpy(), w, rtol=4e-6, atol=1e-30)
    return r


@pytest.mark.parametrize("m,e,k", [(1, 1, 1), (1, 128, 8), (5, 60, 4), (64, 33, 3), (65, 128, 8), (333, 7, 7),
                                   (1000, 512, 32), (9000, 64, 6), (2400, 100, 1)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_route_is_exact(cuda, m, e, k, dtype):
    gen = torch.Generator(device=cuda).manual_seed(m + e)
    logits = torch.randn((m, e), generator=gen, device=cuda).to(dtype)  # bf16: many ties
    bias = torch.randn((e,), generator=gen, device=cuda)
    check_route(logits, k)
    check_route(logits, k, normalise=False, scale=2.5)
    check_route(logits, k, scoring="sigmoid", bias=bias, scale=2.5)
    check_route(logits, k, scoring="sigmoid", normalise=False)


@pytest.mark.parametrize("m", [1, 40, 500])
def test_route_closed_experts(cuda, m):
    gen = torch.Generator(device=cuda).manual_seed(m)
    logits = torch.randn((m, 24), generator=gen, device=cuda)
    logits[torch.rand((m, 24), generator=gen, device=cuda) < 0.7] = float("-inf")
    logits[0] = float("-inf")                       # a row without any expert
    logits[-1, 3] = float("nan")                    # NaN closes too
    for scoring in ("softmax", "sigmoid"):
        for normalise in (True, False):
            r = check_route(logits, 6, scoring=scoring, normalise=normalise)
            assert bool((r.ids[0] == -1).all()) and float(r.weights[0].abs().sum()) == 0.0


def test_route_extremes(cuda):
    lowest = torch.finfo(torch.bfloat16).min
    logits = torch.tensor([[lowest, lowest, 0.0, -0.0], [-200.0, -300.0, -250.0, float("-inf")],
                           [float("inf"), 1.0, float("inf"), 2.0], [0.0, -0.0, -0.0, 0.0]],
                          device=cuda, dtype=torch.bfloat16)
    r = kernels.moe_route(logits, 3)
    assert r.ids.tolist() == [[2, 3, 0], [0, 2, 1], [0, 2, 3], [0, 1, 2]]
    assert torch.isfinite(r.weights).all() and torch.allclose(r.weights.sum(1), torch.ones(4, device=cuda))
    r = kernels.moe_route(logits[:2], 3, scoring="sigmoid")  # far below: the scores underflow, their ratios do not
    assert torch.allclose(r.weights.sum(1), torch.ones(2, device=cuda))


def test_route_empty_batch(cuda):
    r = kernels.moe_route(torch.empty((0, 16), device=cuda), 2)
    assert r.offsets.tolist() == [0] * 18 and r.ids.shape == (0, 2)
    x = torch.empty((0, 64), dtype=torch.bfloat16, device=cuda)
    gen = torch.Generator(device=cuda).manual_seed(0)
    assert kernels.grouped_qgemm(x, kernels.Experts(*quantised(gen, 16, 32, 64, cuda)), r).shape == (0, 2, 32)


def check_grouped(cuda, m, e, k, n, kdim, by_pair=False, closed=0.0, skew=0.5, seed=0):
    gen = torch.Generator(device=cuda).manual_seed(seed)
    q = quantised(gen, e, n, kdim, cuda)
    logits = torch.randn((m, e), generator=gen, device=cuda) + skew * torch.randn((e,), generator=gen, device=cuda)
    logits[torch.rand((m, e), generator=gen, device=cuda) < closed] = float("-inf")
    x = torch.randn((m, k, kdim) if by_pair else (m, kdim), generator=gen, device=cuda).to(torch.bfloat16)
    r = kernels.moe_route(logits, k)
    y = kernels.grouped_qgemm(x, kernels.Experts(*q), r, out=torch.full((m, k, n), float("nan"), device=cuda,
                                                                        dtype=torch.bfloat16))
    ids = r.ids.long()
    assert r.status() == 0
    assert bool((y[ids < 0] == 0).all())
    for ex in range(e):
        row, place = torch.nonzero(ids == ex, as_tuple=True)
        if row.numel():
            want, err = product(x[row, place] if by_pair else x[row], q, ex)
            off = (y[row, place].double() - want).abs()
            assert bool((off <= 2**-8 * want.abs() + err).all()), (ex, float((off / (2**-8 * want.abs() + err)).max()))


@pytest.mark.parametrize("m,e,k,n,kdim", [(1, 8, 2, 32, 64), (1, 128, 8, 1536, 2048), (1, 4, 1, 1000, 9728),
                                          (5, 128, 8, 256, 768), (3, 2, 2, 31, 128), (12, 5, 3, 100, 320),
                                          (77, 60, 4, 1000, 576), (160, 16, 4, 512, 1024), (700, 8, 2, 320, 704),
                                          (300, 3, 3, 129, 64), (2000, 32, 4, 160, 256)])
def test_grouped_product(cuda, m, e, k, n, kdim):
    check_grouped(cuda, m, e, k, n, kdim)


@pytest.mark.parametrize("m,e,k", [(1, 8, 2), (30, 12, 4), (900, 6, 2)])
def test_grouped_product_by_pair_and_closed(cuda, m, e, k):
    check_grouped(cuda, m, e, k, 96, 448, by_pair=True, closed=0.3, skew=2.0, seed=m)
    check_grouped(cuda, m, e, k, 96, 448, closed=0.9, seed=m + 1)
    check_grouped(cuda, m, e, k, 40, 192, by_pair=True, closed=1.0, seed=m + 2)


def mlp_case(cuda, m, e, k, h, inter, seed, skew=0.5):
    gen = torch.Generator(device=cuda).manual_seed(seed)
    gate, up, down = quantised(gen, e, inter, h, cuda), quantised(gen, e, inter, h, cuda), quantised(gen, e, h, inter, cuda)
    x = torch.randn((m, h), generator=gen, device=cuda).to(torch.bfloat16)
    logits = torch.randn((m, e), generator=gen, device=cuda) + skew * torch.randn((e,), generator=gen, device=cuda)
    return gate, up, down, x, logits


@pytest.mark.parametrize("m,e,k,h,inter", [(1, 128, 8, 2048, 768), (5, 16, 4, 512, 192), (2, 4, 2, 64, 64),
                                           (33, 9, 3, 320, 448), (160, 128, 8, 256, 128), (1200, 8, 2, 384, 320)])
@pytest.mark.parametrize("act", ["swiglu", "geglu"])
def test_gated_mlp(cuda, m, e, k, h, inter, act):
    gate, up, down, x, logits = mlp_case(cuda, m, e, k, h, inter, m + h)
    logits[0] = float("-inf")
    if m > 1:
        logits[1, : e // 2] = float("-inf")
    r = kernels.moe_route(logits, k)
    y = kernels.moe_mlp(x, kernels.Experts.gate_up(gate, up), kernels.Experts(*down), r, activation=act)
    ids = r.ids.long()
    assert r.status() == 0
    assert bool((y[ids < 0] == 0).all()) and bool((ids[0] < 0).all())
    for ex in range(e):
        row, place = torch.nonzero(ids == ex, as_tuple=True)
        if not row.numel():
            continue
        g, dg = product(x[row], gate, ex)
        u, du = product(x[row], up, ex)
        if act == "swiglu":
            a = g * torch.sigmoid(g)
        else:
            a = 0.5 * g * (1.0 + torch.tanh(0.7978845608028654 * (g + 0.044715 * g**3)))
        hid = a * u
        dh = 1.13 * dg * (u.abs() + du) + a.abs() * du + 2**-8 * hid.abs()
        w, mag = dense(down, ex)
        want = hid @ w.T
        tol = 2**-8 * want.abs() + (dh + 2**-12 * hid.abs()) @ w.abs().T + 2**-21 * (hid.abs() @ mag.T)
        off = (y[row, place].double() - want).abs()
        assert bool((off <= tol).all()), (ex, float((off / tol).max()))


def test_rows_do_not_depend_on_the_batch(cuda):
    """A verification pass must give every row the bits that it gets alone (speculative decoding returns the tokens of
    plain decoding): batches of 1 to 160 rows over the same rows."""
    gate, up, down, x, logits = mlp_case(cuda, 160, 24, 4, 512, 320, 3)
    gu, dn = kernels.Experts.gate_up(gate, up), kernels.Experts(*down)
    whole = kernels.moe_mlp(x, gu, dn, kernels.moe_route(logits, 4))
    for r0, r1 in [(0, 1), (7, 8), (3, 8), (10, 26), (20, 90), (0, 159)]:
        part = kernels.moe_mlp(x[r0:r1].contiguous(), gu, dn, kernels.moe_route(logits[r0:r1].contiguous(), 4))
        assert torch.equal(part.view(torch.int16), whole[r0:r1].view(torch.int16)), (r0, r1)


def test_overlap_off_and_graph_replay_give_the_same_bits(cuda):
    gate, up, down, x, logits = mlp_case(cuda, 5, 32, 4, 256, 192, 5)
    gu, dn = kernels.Experts.gate_up(gate, up), kernels.Experts(*down)
    h = torch.randn((5, 256), device=cuda).to(torch.bfloat16)
    norm = torch.ones(256, dtype=torch.bfloat16, device=cuda)

    def block():
        r = kernels.moe_route(logits, 4)
        return kernels.block_residual(kernels.moe_mlp(x, gu, dn, r), h, 1e-6, weights=r.weights, next_norm=norm)

    want = [t.clone() for t in block()]
    was = kernels.set_launch_overlap(False)
    try:
        got = [t.clone() for t in block()]
    finally:
        kernels.set_launch_overlap(was)
    assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(got, want))
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(side):
        block()
    torch.cuda.current_stream(cuda).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(out, want))


def test_products_hold_the_range_of_bf16(cuda):
    """Rows of 2^-90, 1 and 2^90 and experts of very different weights: the powers of two that bring the operands into
    fp16 must leave every row as exact as one of ordinary size. Infinities and NaN stay in their row."""
    gate, up, down, x, logits = mlp_case(cuda, 24, 4, 2, 256, 128, 11)
    for q, f in ((gate, 2.0**-6), (up, 2.0**6), (down, 2.0**20)):
        q[1][1:] *= f
        q[2][1:] *= f
    gu, dn = kernels.Experts.gate_up(gate, up), kernels.Experts(*down)
    r = kernels.moe_route(logits, 2)
    y = kernels.grouped_qgemm(x, gu, r)
    for f in (2.0**-90, 2.0**90):
        # every value shifts by a power of two: the same bits apart from the exponent
        assert torch.equal(kernels.grouped_qgemm(x * f, gu, r).float(), y.float() * f)
    assert bool(torch.isfinite(kernels.moe_mlp(x * 2.0**40, gu, dn, r).float()).all())
    z = kernels.moe_mlp(x, gu, dn, r)
    x2 = x.clone()
    x2[3, 5], x2[7, 0] = float("inf"), float("nan")
    z2 = kernels.moe_mlp(x2, gu, dn, r)
    assert not bool(torch.isfinite(z2[3].float()).any()) and bool(torch.isnan(z2[7].float()).all())
    keep = [i for i in range(24) if i not in (3, 7)]
    assert torch.equal(z[keep], z2[keep]) and r.status() == 0


# ---- block residual -------------------------------------------------------------------------------------------
def block_reference(y, weights, h, post, gate, scale, nxt, gemma, eps):
    b = y.double() if weights is None else (weights.double()[:, :, None] * y.double()).sum(1)

    def norm(v, w):
        return v / torch.sqrt((v * v).mean(1, keepdim=True) + eps) * (w.double() + (1.0 if gemma else 0.0))

    if post is not None:
        b = norm(b, post)
    if gate is not None:
        b = b * gate.double()
    v = scale * h.double() + b
    return v, (norm(v, nxt) if nxt is not None else None)


@pytest.mark.parametrize("m,places,hsz", [(1, 8, 2048), (3, 1, 64), (17, 2, 4096), (5, 4, 8192), (2, 32, 16384),
                                          (9, 3, 1001), (4, 2, 7), (600, 8, 640), (2, 5, 2056)])
@pytest.mark.parametrize("gemma", [False, True])
def test_block_residual(cuda, m, places, hsz, gemma):
    gen = torch.Generator(device=cuda).manual_seed(m + hsz)
    rnd = lambda *s: torch.randn(s, generator=gen, device=cuda)  # noqa: E731
    y, h = rnd(m, places, hsz).to(torch.bfloat16), rnd(m, hsz).to(torch.bfloat16)
    w = torch.softmax(rnd(m, places), 1)
    post, nxt = (1 + 0.1 * rnd(hsz)).to(torch.bfloat16), (1 + 0.1 * rnd(hsz)).to(torch.bfloat16)
    gates = [None] + [(0.5 + 0.2 * rnd(*s)).to(torch.bfloat16) for s in ((hsz,), (m, 1), (m, hsz))]
    for gate in gates:
        for pn in (None, post):
            sq = torch.empty(m, device=cuda)
            out, z = kernels.block_residual(y, h, 1e-6, weights=w, post_norm=pn, gate=gate, residual_scale=0.75,
                                            next_norm=nxt, gemma=gemma, out_sq=sq)
            v, zz = block_reference(y, w, h, pn, gate, 0.75, nxt, gemma, 1e-6)
            # float32 throughout: 2^-18 of the terms' magnitudes (32 products, two means), then one rounding to bf16
            mag = v.abs() + h.double().abs() + (w.double()[:, :, None] * y.double().abs()).sum(1) * (4 if pn is not None else 1)
            assert bool(((out.double() - v).abs() <= 2**-8 * v.abs() + 2**-18 * mag).all())
            assert bool(((z.double() - zz).abs() <= 2**-8 * zz.abs() + 2**-15 * (zz.abs() + 1)).all())
            want = (out.double() ** 2).sum(1)
            assert bool(((sq.double() - want).abs() <= 2**-18 * want).all())


def test_block_residual_skips_closed_places_and_runs_in_place(cuda):
    gen = torch.Generator(device=cuda).manual_seed(1)
    y = torch.randn((4, 3, 256), generator=gen, device=cuda).to(torch.bfloat16)
    h = torch.randn((4, 256), generator=gen, device=cuda).to(torch.bfloat16)
    w = torch.rand((4, 3), generator=gen, device=cuda)
    w[0] = 0.0
    w[2, 1] = 0.0
    want, _ = kernels.block_residual(y, h, 1e-6, weights=w)
    y[0] = float("nan")
    y[2, 1] = float("inf")
    out, z = kernels.block_residual(y, h, 1e-6, weights=w, out=h)
    assert out is h and z is None and torch.equal(h, want) and bool(torch.isfinite(want.float()).all())


def test_block_residual_unaligned_rows_match_aligned_ones(cuda):
    gen = torch.Generator(device=cuda).manual_seed(2)
    y, h = (torch.randn((6, 520), generator=gen, device=cuda).to(torch.bfloat16) for _ in range(2))
    nxt = torch.ones(520, dtype=torch.bfloat16, device=cuda)
    want = kernels.block_residual(y, h, 1e-6, next_norm=nxt)
    buf = torch.empty(6 * 520 + 1, dtype=torch.bfloat16, device=cuda)
    odd = buf[1:].view(6, 520)
    odd.copy_(h)
    got = kernels.block_residual(y, odd, 1e-6, next_norm=nxt)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---- refusals ---------------------------------------------------------------------------------------------------
def test_refusals(cuda):
    gen = torch.Generator(device=cuda).manual_seed(0)
    logits = torch.randn((4, 8), device=cuda)
    r = kernels.moe_route(logits, 2)
    ex = kernels.Experts(*quantised(gen, 8, 64, 128, cuda))
    x = torch.zeros((4, 128), dtype=torch.bfloat16, device=cuda)
    with pytest.raises(ValueError, match="top_k"):
        kernels.moe_route(logits, 9)
    with pytest.raises(ValueError, match="scoring"):
        kernels.moe_route(logits, 2, scoring="tanh")
    with pytest.raises(TypeError):
        kernels.moe_route(logits.half(), 2)
    with pytest.raises(ValueError, match="contiguous"):
        kernels.moe_route(logits.T, 2)
    with pytest.raises(ValueError, match="bias"):
        kernels.moe_route(logits, 2, bias=torch.zeros(7, device=cuda))
    with pytest.raises(ValueError, match="CUDA"):
        kernels.moe_route(logits.cpu(), 2)
    with pytest.raises(_lib.KernelUnsupported, match="512 experts"):
        kernels.moe_route(torch.zeros((1, 600), device=cuda), 2)
    with pytest.raises(ValueError, match="routing"):
        kernels.grouped_qgemm(x[:3].contiguous(), ex, r)
    with pytest.raises(ValueError, match="K="):
        kernels.grouped_qgemm(x[:, :64].contiguous(), ex, r)
    with pytest.raises(TypeError):
        kernels.grouped_qgemm(x.float(), ex, r)
    with pytest.raises(ValueError, match="out must be"):
        kernels.grouped_qgemm(x, ex, r, out=torch.empty((4, 64), dtype=torch.bfloat16, device=cuda))
    with pytest.raises(ValueError, match="experts"):
        kernels.grouped_qgemm(x, kernels.Experts(*quantised(gen, 4, 64, 128, cuda)), r)
    with pytest.raises(ValueError, match="activation"):
        kernels.moe_mlp(x, ex, kernels.Experts(*quantised(gen, 8, 128, 64, cuda)), r, activation="relu")
    with pytest.raises(ValueError, match="down is"):
        kernels.moe_mlp(x, ex, ex, r)
    with pytest.raises(ValueError, match="shape mismatch"):
        w, s, b = quantised(gen, 2, 32, 128, cuda)
        kernels.Experts(w, s[:, :, :1].contiguous(), b)
    h = torch.zeros((4, 128), dtype=torch.bfloat16, device=cuda)
    with pytest.raises(ValueError, match="gate"):
        kernels.block_residual(x, h, 1e-6, gate=torch.zeros(64, dtype=torch.bfloat16, device=cuda))
    with pytest.raises(ValueError, match="without weights"):
        kernels.block_residual(torch.zeros((4, 2, 128), dtype=torch.bfloat16, device=cuda), h, 1e-6)
    with pytest.raises(ValueError, match="next_norm"):
        kernels.block_residual(x, h, 1e-6, next_norm=torch.zeros(64, dtype=torch.bfloat16, device=cuda))

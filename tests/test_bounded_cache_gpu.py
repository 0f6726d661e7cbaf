"""Decoding over a bounded cache on the GPU -- rotary positions, attention that adds up slot weights, eviction, and
verification from given random numbers -- against plain float64 forms, at the sizes and masks where they can go wrong."""
from __future__ import annotations

import math

import pytest
import torch

from ironmule_b200 import kernels

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
INF, NAN = float("inf"), float("nan")


def gen(cuda, seed):
    return torch.Generator(device=cuda).manual_seed(seed)


def page_table(g, seqs, slots, extra=0):
    per = -(-slots // 16)
    order = torch.randperm(seqs * per + extra, generator=g, device=g.device)[: seqs * per]
    return order.to(torch.int32).view(seqs, per).contiguous(), seqs * per + extra


def ints(values, cuda):
    return torch.tensor(values, dtype=torch.int32, device=cuda)


# ---- rotary positions -------------------------------------------------------------------------------------------
def turned(x, pos, freq, factor, layout, inverse=False):
    """(x turned, |a| + |b| of each value's pair) in float64."""
    x = x.double()
    t = pos.double()[:, None] * freq.double()
    c, s = factor * torch.cos(t)[:, None], factor * torch.sin(t)[:, None] * (-1 if inverse else 1)
    r = 2 * freq.numel()
    i = torch.arange(r // 2, device=x.device)
    ia, ib = (i, i + r // 2) if layout == "half" else (2 * i, 2 * i + 1)
    y, size = x.clone(), torch.zeros_like(x)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    size[..., ia] = size[..., ib] = a.abs() + b.abs()
    return y, size


def assert_turned(got, want, size, factor):
    # c and s: the angle's rest rounded to float32 (2^-25), sincospi (2^-24), factor and its product (2^-23 together); a
    # product and a sum more (2^-23): under 2^-21 of the pair's values; then the rounding to the type
    tol = HALF_STEP[got.dtype] * want.abs() * (1 + 2.0**-10) + 2.0**-21 * abs(factor) * size
    bad = (got.double() - want).abs() > tol
    assert not bool(bad.any()), f"{int(bad.sum())} values off, most {float((got.double() - want).abs().max())}"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("m,h,d,rotary", [(1, 1, 2, 2), (1, 32, 128, 128), (7, 3, 80, 32), (33, 5, 96, 96), (5, 2, 20, 6),
                                          (3, 9, 17, 16), (200, 8, 256, 64), (2, 4, 64, 0),
                                          (70, 6, 144, 72), (9, 4, 20, 8)])
def test_rope_turns_rows(cuda, dtype, layout, m, h, d, rotary):
    g = gen(cuda, m * d + rotary)
    x = torch.randn((m, h, d), generator=g, device=cuda).to(dtype)
    freq = torch.rand(rotary // 2, generator=g, device=cuda, dtype=torch.float64)
    for pos in (torch.randint(0, 5000, (m,), generator=g, device=cuda, dtype=torch.int32),
                torch.randint(-(2**40), 2**40, (m,), generator=g, device=cuda)):
        for inverse in (False, True):
            for table in (freq, freq.float()):
                got = kernels.rope(x, pos, table, layout=layout, factor=1.25, inverse=inverse)
                want, size = turned(x, pos, table, 1.25, layout, inverse)
                assert got.is_contiguous() and got.dtype == dtype
                if pos.dtype == torch.int64:  # 2^40 turns: the float64 angle itself is off by 2^-13, as the test's is
                    assert float((got.double() - want).abs().max()) <= 2.0**-10 * float(1 + size.max()) + HALF_STEP[
                        dtype] * float(want.abs().max())
                else:
                    assert_turned(got, want, size, 1.25)
                assert torch.equal(got[..., rotary:], x[..., rotary:])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rope_takes_strides_and_works_in_place(cuda, layout):
    g = gen(cuda, 3)
    pos = torch.randint(0, 70000, (19,), generator=g, device=cuda, dtype=torch.int32)
    freq, factor = kernels.rope_frequencies(48, 10000.0, scaling="linear", stretch=4.0, device=cuda)
    for width, offset in ((6 * 64, 64), (6 * 64 + 3, 5)):  # aligned rows, and rows at odd addresses
        packed = torch.randn((19, width), generator=g, device=cuda).to(torch.bfloat16)
        x = packed[:, offset:offset + 4 * 64].view(19, 4, 64)
        want, size = turned(x, pos, freq, factor, layout)
        assert_turned(kernels.rope(x, pos, freq, layout=layout), want, size, 1.0)
        by_head = x.transpose(0, 1).contiguous().transpose(0, 1)  # heads outermost
        out = torch.empty((4, 19, 64), dtype=torch.bfloat16, device=cuda).transpose(0, 1)
        assert_turned(kernels.rope(by_head, pos, freq, layout=layout, out=out), want, size, 1.0)
        rest = packed.clone()
        assert kernels.rope(x, pos, freq, layout=layout, out=x) is x
        assert_turned(x, want, size, 1.0)
        rest[:, offset:offset + 4 * 64] = x.reshape(19, -1)
        assert torch.equal(rest, packed)  # nothing beside x was written
    wide = x[:, :1].expand(19, 4, 64)  # one head read by four
    assert_turned(kernels.rope(wide, pos, freq, layout=layout), *turned(wide, pos, freq, 1.0, layout), 1.0)
    assert kernels.rope(x[:0], pos[:0], freq, layout=layout).shape == (0, 4, 64)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rope_inverse_is_the_gradient(cuda, layout):
    g = gen(cuda, 5)
    x, dy = (torch.randn((6, 2, 24), generator=g, device=cuda) for _ in range(2))
    pos = torch.randint(0, 1000, (6,), generator=g, device=cuda, dtype=torch.int32)
    freq = torch.rand(8, generator=g, device=cuda)
    got = kernels.rope(dy, pos, freq, layout=layout, factor=1.5, inverse=True).double()
    leaf = x.double().requires_grad_()
    t = pos.double()[:, None] * freq.double()
    c, s = 1.5 * torch.cos(t)[:, None], 1.5 * torch.sin(t)[:, None]
    a, b = (leaf[..., :8], leaf[..., 8:16]) if layout == "half" else (leaf[..., 0:16:2], leaf[..., 1:16:2])
    pairs = torch.stack([a * c - b * s, a * s + b * c])
    rest = leaf[..., 16:]
    y = torch.cat([pairs[0], pairs[1], rest], -1) if layout == "half" else torch.cat(
        [pairs.permute(1, 2, 3, 0).flatten(-2), rest], -1)
    (want,) = torch.autograd.grad(y, leaf, dy.double())
    size = dy.abs().double().sum(-1, keepdim=True)
    assert bool(((got - want).abs() <= 2.0**-21 * 1.5 * size + 2.0**-24 * want.abs()).all())
    # and against differences of the forward call: the map is linear, so a difference is exact but for roundings
    for at in ((0, 0, 0), (3, 1, 9), (5, 0, 20)):
        step = torch.zeros_like(x)
        step[at] = 1.0
        diff = (kernels.rope(step, pos, freq, layout=layout, factor=1.5).double() * dy.double()).sum()
        assert abs(float(diff - got[at])) <= 2.0**-20 * 1.5 * float(size.max())


def kv_case(cuda, seed, m, hq, hkv, d, dtype, seqs=3, slots=70):
    g = gen(cuda, seed)
    table, pages = page_table(g, seqs, slots, extra=2)
    qkv = torch.randn((m, (hq + 2 * hkv) * d), generator=g, device=cuda).to(dtype)
    at = torch.randperm(seqs * slots, generator=g, device=cuda)[:m]
    seq, slot = (at // slots).to(torch.int32), (at % slots).to(torch.int32)
    pos = torch.randint(0, 10**6, (m,), generator=g, device=cuda, dtype=torch.int32)
    k = torch.randn((pages, hkv, 16, d), generator=g, device=cuda).to(dtype)
    return g, table, qkv, seq, slot, pos, k, k.flip(0).contiguous()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,hq,hkv,d,rotary,layout", [(1, 32, 8, 128, 128, "half"), (5, 4, 4, 64, 32, "interleaved"), (60, 4, 2, 144, 72, "half"),
                                                      (40, 6, 2, 80, 80, "half"), (3, 2, 1, 18, 10, "half"),
                                                      (150, 8, 1, 256, 64, "interleaved")])
def test_rope_kv_turns_and_writes_the_cache(cuda, dtype, m, hq, hkv, d, rotary, layout):
    g, table, qkv, seq, slot, pos, k, v = kv_case(cuda, m + d, m, hq, hkv, d, dtype)
    if m > 4:  # rows without a slot, behind the table's end, of no sequence, on a page that is none
        slot[0], slot[1], seq[2] = -1, table.shape[1] * 16, 7
        gone = int(seq[3]), int(slot[3])
        table[gone[0], gone[1] // 16] = 999
    freq = torch.rand(rotary // 2, generator=g, device=cuda, dtype=torch.float64)
    slot_pos = torch.full((3, hkv, 75), -5, dtype=torch.int32, device=cuda)
    rows = qkv.view(m, hq + 2 * hkv, d)
    want, size = turned(rows[:, :hq + hkv], pos, freq, 1.1, layout)
    k_want, v_want, pos_want = k.double(), v.double(), slot_pos.clone()
    k_size = torch.zeros_like(k_want)
    for i in range(m):
        s, j = int(seq[i]), int(slot[i])
        if not (0 <= s < 3 and 0 <= j < table.shape[1] * 16) or not 0 <= int(table[s, j // 16]) < k.shape[0]:
            continue
        page = int(table[s, j // 16])
        k_want[page, :, j % 16], v_want[page, :, j % 16] = want[i, hq:], rows[i, hq + hkv:].double()
        k_size[page, :, j % 16] = size[i, hq:]
        pos_want[s, :, j] = pos[i]
    q = kernels.rope_kv(qkv, freq, pos, slot, seq, table, hq, hkv, d, k, v, layout=layout, factor=1.1, slot_pos=slot_pos)
    assert_turned(q, want[:, :hq], size[:, :hq], 1.1)
    assert_turned(k, k_want, k_size, 1.1)
    assert torch.equal(v.double(), v_want) and torch.equal(slot_pos, pos_want)


def test_rope_kv_leaves_rows_behind_the_last_alone(cuda):
    _, table, qkv, seq, slot, pos, k, v = kv_case(cuda, 8, 12, 4, 2, 64, torch.bfloat16)
    freq = torch.ones(32, device=cuda)
    q_out = torch.full((12, 4, 64), 3.0, dtype=torch.bfloat16, device=cuda)
    k2, v2 = k.clone(), v.clone()
    kernels.rope_kv(qkv, freq, pos, slot, seq, table, 4, 2, 64, k, v, q_out=q_out, rows=5)
    assert bool((q_out[5:] == 3.0).all())
    kernels.rope_kv(qkv[:5].contiguous(), freq, pos, slot, seq, table, 4, 2, 64, k2, v2)
    assert torch.equal(k, k2) and torch.equal(v, v2)


# ---- attention with slot weights ----------------------------------------------------------------------------------
def attend_plain(q, k, v, table, seq_rows, row_slot, weights, scale, window=0, max_kv=1 << 30, seq_slot=None):
    """(out, weights', tolerance of out, tolerance of weights') in float64."""
    m, hq, d = q.shape
    hkv = k.shape[1]
    group = hq // hkv
    out, after = torch.zeros((m, hq, d), dtype=torch.float64, device=q.device), weights.double()
    out_tol, w_tol = torch.zeros_like(out), torch.zeros_like(after)
    bounds, slots = seq_rows.tolist(), row_slot.tolist()
    for b in range(len(bounds) - 1):
        s = b if seq_slot is None else int(seq_slot[b])
        rows = range(bounds[b], bounds[b + 1])
        if not rows:
            continue
        n = min(max(slots[r] for r in rows) + 1, max_kv, table.shape[1] * 16)
        if n <= 0:
            continue
        first, cap = next(slots[r] for r in rows if slots[r] >= 0), after.shape[-1]
        kept = min(n, cap)
        after[s, :, max(0, min(first, kept)):kept] = 0
        pages = table[s, :-(-n // 16)].long()
        for h in range(hkv):
            ks, vs = (t[pages, h].flatten(0, 1)[:n].double() for t in (k, v))
            for r in rows:
                last = min(slots[r], n - 1)
                lo = max(0, slots[r] - window + 1) if window else 0
                if last < lo:
                    continue
                for qh in range(h * group, (h + 1) * group):
                    qv = q[r, qh].double()
                    kk, vv = ks[lo:last + 1], vs[lo:last + 1]
                    sc = scale * (kk @ qv)
                    p = torch.softmax(sc, 0)
                    out[r, qh] = p @ vv
                    end = min(last + 1, cap)
                    if end > lo:
                        after[s, h, lo:end] += p[:end - lo]
                    # scores: d products summed in float32 (2^-23 each step, whichever way they round), scaled; a score's
                    # error moves a weight by itself and the sum by as much; exponentials 2^-22; sums of n weights in
                    # runs of at most n / 8 + 64; weights that meet v are kept to 2^-16 of themselves
                    size = abs(scale) * (kk.abs() @ qv.abs())
                    err = 2 * float(size.max()) * (d * 2.0**-23 + 2.0**-21) + 2.0**-21 + (kk.shape[0] / 8 + 64) * 2.0**-24
                    out_tol[r, qh] = (err + 2.0**-16) * (p @ vv.abs()) + HALF_STEP[q.dtype] * out[r, qh].abs()
                    if end > lo:
                        w_tol[s, h, lo:end] += err * p[:end - lo] + 1e-30
    w_tol += 2.0**-22 * after.abs()
    return out, after, out_tol * (1 + 2.0**-7) + 1e-30, w_tol


def attend_case(cuda, seed, lengths, rows, hq, hkv, d, dtype, extra=1, spread=1.0):
    """Sequences of those lengths, the last `rows[b]` slots of each being its new rows; cache garbage is NaN and inf."""
    g = gen(cuda, seed)
    seqs, most = len(lengths), max(max(lengths), 1)
    table, pages = page_table(g, seqs, most + 20, extra)
    k = (spread * torch.randn((pages, hkv, 16, d), generator=g, device=cuda)).to(dtype)
    v = torch.randn((pages, hkv, 16, d), generator=g, device=cuda).to(dtype)
    slot, bounds = [], [0]
    for b, n in enumerate(lengths):
        for t, bad in ((k, NAN), (v, INF)):  # slots behind the end hold whatever was there
            for j in range(n, table.shape[1] * 16):
                t[int(table[b, j // 16]), :, j % 16] = bad
        slot += [n - rows[b] + i for i in range(rows[b])] if n else [-1] * rows[b]
        bounds.append(bounds[-1] + rows[b])
    q = torch.randn((bounds[-1], hq, d), generator=g, device=cuda).to(dtype)
    weights = 3 * torch.rand((seqs, hkv, table.shape[1] * 16), generator=g, device=cuda)
    return q, k, v, table, ints(bounds, cuda), ints(slot, cuda), weights


def attend_check(case, *, window=0, max_kv=None, keys_per_split=0, in_place=False, scale=None, seq_slot=None):
    q, k, v, table, bounds, slot, weights = case
    scale = q.shape[2] ** -0.5 if scale is None else scale
    counts = (bounds[1:] - bounds[:-1]).tolist()
    max_kv = table.shape[1] * 16 if max_kv is None else max_kv
    want, after, tol, w_tol = attend_plain(q, k, v, table, bounds, slot, weights, scale, window, max_kv, seq_slot)
    given = weights.clone()
    target = given if in_place else torch.full_like(weights, -7.0)
    out = kernels.attention_weights(q, k, v, table, bounds, slot, given, max_rows_per_seq=max(counts), max_kv_len=max_kv,
                                    scale=scale, window=window, keys_per_split=keys_per_split,
                                    weights_out=None if in_place else target, seq_slot=seq_slot)
    assert bool(((out.double() - want).abs() <= tol).all()), float(((out.double() - want).abs() / tol).max())
    seen = torch.zeros_like(weights, dtype=torch.bool)
    slots = slot.tolist()
    for b, c in enumerate(counts):
        s = b if seq_slot is None else int(seq_slot[b])
        rows = range(int(bounds[b]), int(bounds[b + 1]))
        n = min(max([slots[r] for r in rows], default=-1) + 1, max_kv, table.shape[1] * 16)
        seen[s, :, :max(0, n)] = True
    off = ((target.double() - after).abs() > w_tol) & seen
    assert not bool(off.any()), float(((target.double() - after).abs() / w_tol)[seen].max())
    assert torch.equal(target[~seen], (weights if in_place else torch.full_like(weights, -7.0))[~seen])
    if not in_place:
        assert torch.equal(given, weights)
    return out, target


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [16, 64, 80, 96, 112, 128, 192, 256])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (8, 2), (7, 1), (20, 1)])
def test_attention_weights_of_one_token(cuda, dtype, d, hq, hkv):
    attend_check(attend_case(cuda, d + hq, [1, 2, 15, 16, 17, 200, 0, 333], [1] * 8, hq, hkv, d, dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("window", [0, 1, 5, 40, 1000])
@pytest.mark.parametrize("rows", [[5, 5, 5], [1, 9, 0, 33], [64, 2]])
def test_attention_weights_of_verify_rows(cuda, dtype, window, rows):
    lengths = [[5, 64, 200], [130, 9, 50, 99], [64, 300]][len(rows) == 4 and 1 or len(rows) == 2 and 2 or 0]
    attend_check(attend_case(cuda, window + len(rows), lengths, rows, 8, 4, 128, dtype), window=window)


@pytest.mark.parametrize("kps", [64, 128, 192, 4096])
def test_attention_weights_splits(cuda, kps):
    case = attend_case(cuda, kps, [700, 64, 65, 1000, 128], [2, 1, 3, 1, 5], 8, 2, 64, torch.bfloat16)
    attend_check(case, keys_per_split=kps, in_place=True)
    attend_check(case, keys_per_split=kps, window=130)


@pytest.mark.parametrize("window", [1, 20, 100])
@pytest.mark.parametrize("kps", [0, 64])
def test_attention_weights_of_rows_far_apart(cuda, window, kps):
    """Rows of one sequence need not follow one another: with a window, slots between them are seen by none."""
    q, k, v, table, bounds, slot, weights = attend_case(cuda, 8, [2000, 900], [6, 3], 8, 2, 128, torch.bfloat16)
    slot[:] = ints([3, 1999, 700, 64, 1500, 90, 899, 0, 333], cuda)
    attend_check((q, k, v, table, bounds, slot, weights), window=window, keys_per_split=kps)
    attend_check((q, k, v, table, bounds, slot, weights), window=window, keys_per_split=kps, in_place=True)
    attend_check((q, k, v, table, bounds, slot, weights), keys_per_split=kps)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [16, 48, 64, 80, 96, 112, 128, 144, 192, 256])
@pytest.mark.parametrize("kps", [0, 64])
def test_attention_weights_of_blocks_with_several_splits(cuda, dtype, d, kps):
    """Rows of two windows side by side: a block takes a split of one and then a split of the other, and what the first leaves
    in shared memory reaches nothing, in heads that are narrower than the columns kept for them either."""
    for seed in range(3):
        q, k, v, table, bounds, slot, weights = attend_case(cuda, d + seed, [420, 420], [6, 3], 8, 2, d, dtype)
        slot[:] = ints([200, 201, 202, 392, 393, 394, 150, 342, 343], cuda)
        attend_check((q, k, v, table, bounds, slot, weights), window=100, keys_per_split=kps)


def test_attention_weights_bits_do_not_depend_on_the_launch(cuda):
    """With keys_per_split given, a row alone equals the same row in a batch, among other rows."""
    q, k, v, table, bounds, slot, weights = attend_case(cuda, 11, [700, 333, 64], [5, 3, 1], 8, 2, 128, torch.bfloat16)
    many = kernels.attention_weights(q, k, v, table, bounds, slot, weights.clone(), max_rows_per_seq=5, max_kv_len=720,
                                     scale=0.1, keys_per_split=128)
    for b in range(3):
        for r in range(int(bounds[b]), int(bounds[b + 1])):
            one = kernels.attention_weights(q[r:r + 1].contiguous(), k, v, table, ints([0, 1], cuda),
                                            slot[r:r + 1].contiguous(), weights.clone(), max_rows_per_seq=1,
                                            max_kv_len=int(slot[r]) + 1, scale=0.1, keys_per_split=128,
                                            seq_slot=ints([b], cuda))
            assert torch.equal(one[0], many[r])
    again = kernels.attention_weights(q, k, v, table, bounds, slot, weights.clone(), max_rows_per_seq=5, max_kv_len=720,
                                      scale=0.1, keys_per_split=128)
    assert torch.equal(again, many)


@pytest.mark.parametrize("window", [0, 700])
def test_attention_weights_bits_over_many_splits(cuda, window):
    """The same with more splits than one warp joins, and rows whose windows begin at different splits: neither the launch's
    max_kv_len nor the other rows' windows change a row's bits."""
    lengths, rows = [2500, 1300, 1999], [5, 1, 3]
    q, k, v, table, bounds, slot, weights = attend_case(cuda, 12, lengths, rows, 8, 2, 64, torch.float16)
    slot[0], slot[6] = 900, 1500  # rows of other splits beside rows at the end
    kw = {"scale": 0.125, "keys_per_split": 64, "window": window}
    many = kernels.attention_weights(q, k, v, table, bounds, slot, weights.clone(), max_rows_per_seq=5, max_kv_len=2520, **kw)
    for b in range(3):
        for r in range(int(bounds[b]), int(bounds[b + 1])):
            for most in (int(slot[r]) + 1, 2520):
                one = kernels.attention_weights(q[r:r + 1].contiguous(), k, v, table, ints([0, 1], cuda),
                                                slot[r:r + 1].contiguous(), weights.clone(), max_rows_per_seq=1,
                                                max_kv_len=most, seq_slot=ints([b], cuda), **kw)
                assert torch.equal(one[0], many[r])


def test_attention_weights_masks(cuda):
    # masked rows, a sequence without rows, table rows in another order, weights shorter than the cache, a short max_kv
    q, k, v, table, bounds, slot, weights = attend_case(cuda, 4, [90, 40, 77], [3, 0, 2], 4, 2, 64, torch.float16)
    slot[1] = -1
    attend_check((q, k, v, table, bounds, slot, weights))
    attend_check((q, k, v, table, bounds, slot, weights[:, :, :50].contiguous()))
    attend_check((q, k, v, table, bounds, slot, weights), max_kv=33)
    order = ints([2, 1, 0], cuda)
    swapped = table[order.long()].contiguous()
    attend_check((q, k, v, swapped, bounds, slot, weights), seq_slot=order)
    slot[2] = 10**6  # a slot behind the table sees what the table has
    attend_check((q, k.nan_to_num(0.5), v.nan_to_num(0.5, 0.5, 0.5), table, bounds, slot, weights), in_place=True,
                 max_kv=2 * 10**6)


@pytest.mark.parametrize("rows", [[1, 1, 1], [5, 3, 5]])
@pytest.mark.parametrize("window", [110, 150, 215])
@pytest.mark.parametrize("in_place", [False, True])
def test_attention_weights_of_half_a_window(cuda, rows, window, in_place):
    """Windows of half the slots and more, whose splits a call may take in one kernel: some splits are seen by no row, in
    some the first pages are not. A row's bits are those of a call over a longer table."""
    case = attend_case(cuda, window, [200, 64, 190], rows, 8, 4, 128, torch.bfloat16)
    out, after = attend_check(case, window=window, in_place=in_place, keys_per_split=64)
    attend_check(case, window=window, in_place=in_place)
    q, k, v, table, bounds, slot, weights = case
    wider = torch.cat([table, table.new_full((3, 60), -1)], dim=1)
    given = torch.full((3, 4, wider.shape[1] * 16), -7.0, device=cuda)
    given[:, :, :weights.shape[2]] = weights
    far = kernels.attention_weights(q, k, v, wider, bounds, slot, given, max_rows_per_seq=max(rows), max_kv_len=1100,
                                    scale=128 ** -0.5, window=window, keys_per_split=64)
    assert torch.equal(far, out)
    for b, n in enumerate((200, 64, 190)):
        torch.testing.assert_close(given[b, :, :n], after[b, :, :n], rtol=1e-5, atol=1e-7)


@pytest.mark.parametrize("lengths,rows", [([90, 40], [4, 3]), ([5000, 900], [4, 3]), ([300], [9])])
@pytest.mark.parametrize("in_place", [False, True])
def test_attention_weights_of_rows_padded_in_front(cuda, lengths, rows, in_place):
    """Rows without a slot before a sequence's own: what the earlier slots have gathered stays."""
    q, k, v, table, bounds, slot, weights = attend_case(cuda, 6, lengths, rows, 4, 2, 64, torch.bfloat16)
    for b in range(len(rows)):
        slot[int(bounds[b]):int(bounds[b]) + rows[b] // 2] = -1
    out, after = attend_check((q, k, v, table, bounds, slot, weights), in_place=in_place)
    lone = [int(bounds[b]) + i for b in range(len(rows)) for i in range(rows[b] // 2)]
    assert not bool(out[lone].any())
    for b, n in enumerate(lengths):
        assert bool((after[b, :, :n - rows[b]] >= weights[b, :, :n - rows[b]]).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths,rows,hq,hkv,d,window", [([300], [256], 8, 1, 64, 0), ([2100, 5], [2048, 5], 1, 1, 80, 0),
                                                          ([700, 300], [256, 100], 16, 2, 128, 0), ([600], [512], 4, 1, 256, 100)])
def test_attention_weights_of_prompt_pieces(cuda, dtype, lengths, rows, hq, hkv, d, window):
    """Up to 2048 vectors a kv head."""
    attend_check(attend_case(cuda, 36, lengths, rows, hq, hkv, d, dtype), window=window)


def test_attention_weights_over_its_own_queries(cuda):
    for length in (100, 5000):
        case = attend_case(cuda, 7, [length, 33], [3, 2], 8, 2, 128, torch.bfloat16)
        q, k, v, table, bounds, slot, weights = case
        kw = {"max_rows_per_seq": 3, "max_kv_len": length, "scale": 0.1}
        want = kernels.attention_weights(q, k, v, table, bounds, slot, weights.clone(), **kw)
        own = q.clone()
        assert kernels.attention_weights(own, k, v, table, bounds, slot, weights.clone(), out=own, **kw) is own
        assert torch.equal(own, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_weights_of_values_that_are_not_finite(cuda, dtype):
    """A later row's key and value do not reach an earlier row, whatever they are; a seen NaN does."""
    q, k, v, table, bounds, slot, weights = attend_case(cuda, 9, [37], [5], 4, 2, 64, dtype)
    for t in (k, v):
        for j, bad in ((34, NAN), (35, INF), (36, -INF)):
            t[int(table[0, j // 16]), :, j % 16] = bad
    out = kernels.attention_weights(q, k, v, table, bounds, slot, weights.clone(), max_rows_per_seq=5, max_kv_len=48,
                                    scale=0.125)
    want, _, tol, _ = attend_plain(q[:2], k, v, table, ints([0, 2], cuda), slot[:2], weights, 0.125)
    assert bool(((out[:2].double() - want).abs() <= tol).all())
    assert bool(out[2:].isnan().all())
    # scores of -inf alone leave a row empty; a single one of them leaves the others' weights
    k[int(table[0, 0]), :, 0] = 0.0
    q2, k2, v2, table2, bounds2, slot2, w2 = attend_case(cuda, 10, [3], [1], 2, 2, 64, dtype)
    q2[:] = q2.abs() + 0.5
    k2[int(table2[0, 0]), :, 1] = -INF
    w = w2.clone()
    out = kernels.attention_weights(q2, k2, v2, table2, bounds2, slot2, w, max_rows_per_seq=1, max_kv_len=3, scale=1.0)
    assert bool(out.isfinite().all()) and bool((w[0, :, 1] == w2[0, :, 1]).all())
    k2[int(table2[0, 0]), :, :3] = -INF
    out = kernels.attention_weights(q2, k2, v2, table2, bounds2, slot2, w, max_rows_per_seq=1, max_kv_len=3, scale=1.0)
    assert bool((out == 0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths,rows,d,window,kps", [([37], [1], 64, 0, 0), ([37, 20], [5, 3], 64, 0, 0), ([700], [1], 128, 0, 64),
                                                       ([700, 300], [5, 2], 80, 0, 0), ([5000], [1], 128, 0, 0),
                                                       ([3000, 200], [5, 2], 256, 0, 0), ([900], [33], 64, 0, 64),
                                                       ([3000], [5], 128, 300, 0), ([300], [3], 128, 200, 0)])
def test_attention_weights_of_a_query_that_is_nan(cuda, dtype, lengths, rows, d, window, kps):
    """Its row is NaN, and so are the weights of the slots that it sees; nothing else changes by a bit."""
    q, k, v, table, bounds, slot, weights = attend_case(cuda, 31, lengths, rows, 8, 2, d, dtype)
    kw = {"max_rows_per_seq": max(rows), "max_kv_len": table.shape[1] * 16, "scale": d ** -0.5, "window": window,
          "keys_per_split": kps}
    want, after = kernels.attention_weights(q, k, v, table, bounds, slot, was := weights.clone(), **kw), was
    for at, head in ((0, 1), (rows[0] // 2, 6), (int(bounds[-1]) - 1, 3)):
        bad = q.clone()
        bad[at, head, 5] = NAN
        got = weights.clone()
        out = kernels.attention_weights(bad, k, v, table, bounds, slot, got, **kw)
        assert bool(out[at, head].isnan().all())
        others = torch.ones_like(out, dtype=torch.bool)
        others[at, head] = False
        assert torch.equal(out[others], want[others])
        s = 0 if at < rows[0] else 1
        sees = torch.zeros_like(weights, dtype=torch.bool)
        last = int(slot[at])
        sees[s, head // 4, max(0, last - window + 1) if window else 0:last + 1] = True
        assert bool(got[sees].isnan().all())
        assert torch.equal(got[~sees], after[~sees])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths,rows,kps,bad", [([300], [1], 64, (64, 128)), ([300], [5], 64, (0, 64)), ([3000], [1], 64, (128, 192)),
                                                  ([3000, 500], [5, 1], 64, (0, 64)), ([300, 100], [4, 2], 0, (10, 11))])
def test_attention_weights_of_keys_that_are_nan(cuda, dtype, lengths, rows, kps, bad):
    """A split that has NaN scores alone is no split without a slot: every row that sees it is NaN."""
    q, k, v, table, bounds, slot, weights = attend_case(cuda, 32, lengths, rows, 8, 2, 128, dtype)
    for j in range(*bad):
        k[int(table[0, j // 16]), 1, j % 16] = NAN
    kw = {"max_rows_per_seq": max(rows), "max_kv_len": table.shape[1] * 16, "scale": 0.1, "keys_per_split": kps}
    out = kernels.attention_weights(q, k, v, table, bounds, slot, got := weights.clone(), **kw)
    want, after, tol, w_tol = attend_plain(q, k, v, table, bounds, slot, weights, 0.1)
    assert torch.equal(out.isnan(), want.isnan()) and bool(out[:rows[0], 4:].isnan().all())
    assert torch.equal(got.isnan(), after.isnan())
    fine = ~want.isnan()
    assert bool(((out.double() - want).abs() <= tol)[fine].all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths,rows,hq,d,window,kps", [([100], [1], 8, 64, 0, 0), ([100], [5], 8, 80, 0, 0), ([3000], [1], 8, 128, 0, 64),
                                                          ([3000, 200], [5, 1], 8, 256, 0, 0), ([700], [9], 14, 96, 0, 0),
                                                          ([2000], [3], 8, 128, 1990, 0), ([400], [2], 16, 192, 0, 0)])
def test_attention_weights_of_values_that_are_infinite(cuda, dtype, lengths, rows, hq, d, window, kps):
    """Under a positive weight they are infinite, with their sign; of both signs they are NaN; nothing else is."""
    q, k, v, table, bounds, slot, weights = attend_case(cuda, 35, lengths, rows, hq, 2, d, dtype)
    for j, at, bad in ((5 + 30, 3, INF), (20 + 30, 4, -INF), (21 + 30, 5, INF), (40 + 30, 5, -INF), (41 + 30, d - 1, NAN)):
        v[int(table[0, j // 16]), :, j % 16, at] = bad
    want, after, tol, w_tol = attend_plain(q, k, v, table, bounds, slot, weights, d ** -0.5, window)
    kw = {"max_rows_per_seq": max(rows), "max_kv_len": table.shape[1] * 16, "scale": d ** -0.5, "window": window,
          "keys_per_split": kps}
    out = kernels.attention_weights(q, k, v, table, bounds, slot, got := weights.clone(), **kw).double()
    fine = want.isfinite()
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out[want.isinf()], want[want.isinf()])
    assert not bool(fine.all()) and bool(((out - want).abs() <= tol)[fine].all())
    plain = torch.where(v.isfinite(), v, 0.0)
    kernels.attention_weights(q, k, plain, table, bounds, slot, same := weights.clone(), **kw)
    assert torch.equal(got, same)


def test_attention_weights_of_large_scores_and_equal_ones(cuda):
    case = attend_case(cuda, 21, [500, 64], [1, 4], 8, 2, 128, torch.bfloat16, spread=8.0)
    attend_check(case, scale=1.0)  # scores in the hundreds: one slot has nearly all the weight
    q, k, v, table, bounds, slot, weights = case
    q.zero_()  # every visible slot has the same weight
    out, after = attend_check(case)
    assert bool(((after[0, :, 10] - weights[0, :, 10]).double() - 4 / 500).abs().max() <= 2.0**-22 * 4)


def test_attention_weights_follow_from_call_to_call(cuda):
    """Token by token, in place: the weights are the sums of every call's, and a reused slot starts from zero."""
    q, k, v, table, bounds, slot, weights = attend_case(cuda, 33, [40], [8], 4, 2, 64, torch.bfloat16)
    total = weights.clone()
    total[0, :, 32:] = 1e6  # stale sums of slots that are new
    want = weights.double()
    want[0, :, 32:] = 0
    tol = torch.zeros_like(want)
    for i in range(8):
        one = (q[i:i + 1].contiguous(), k, v, table, ints([0, 1], cuda), slot[i:i + 1].contiguous())
        kernels.attention_weights(*one, total, max_rows_per_seq=1, max_kv_len=64, scale=0.125)
        _, now, _, w_tol = attend_plain(*one, torch.zeros_like(weights), 0.125)
        want += now
        tol += w_tol + 2.0**-22 * want
    assert bool(((total.double() - want).abs() <= tol)[0, :, :40].all())


# ---- eviction ---------------------------------------------------------------------------------------------------
def evict_plain(k, v, table, lengths, seen, weights, pos, budget, recent, sinks):
    """The same on lists; caches [L, pages, Hkv, 16, D]. Returns new copies."""
    k, v, weights_out, pos_out = k.clone(), v.clone(), weights.clone(), pos.clone()
    left = []
    for s in range(table.shape[0]):
        n = max(0, min(int(lengths[s]), weights.shape[-1], table.shape[1] * 16))
        keep = min(n, budget)
        left.append(keep)
        for layer in range(weights.shape[0]):
            for h in range(weights.shape[2]):
                w, p = weights[layer, s, h].tolist(), pos[layer, s, h].tolist()

                def rank(j):
                    safe = p[j] < sinks or p[j] >= int(seen[s]) - recent
                    if safe:  # whatever its weight
                        return (0, 0.0, 0, j)
                    return (1, math.inf, 1, j) if math.isnan(w[j]) else (1, -w[j], 0, j)

                kept = set(sorted(range(n), key=rank)[:keep])
                holes = [j for j in range(keep) if j not in kept]
                movers = [j for j in range(keep, n) if j in kept]
                assert len(holes) == len(movers)
                for to, at in zip(holes, movers):
                    weights_out[layer, s, h, to], pos_out[layer, s, h, to] = w[at], p[at]
                    there, here = (int(table[s, j // 16]) for j in (to, at))
                    for t in (k, v):
                        t[layer, there, h, to % 16] = t[layer, here, h, at % 16]
    return k, v, weights_out, pos_out, left


def same(a, b):
    return torch.equal(a.contiguous().view(torch.int32 if a.element_size() == 4 else torch.int16),
                       b.contiguous().view(torch.int32 if b.element_size() == 4 else torch.int16))


def evict_case(cuda, seed, lengths, layers, hkv, d, dtype, cap=None, kind="heavy"):
    g = gen(cuda, seed)
    seqs, most = len(lengths), max(max(lengths), 1)
    table, pages = page_table(g, seqs, most, extra=3)
    cap = cap or table.shape[1] * 16
    k = torch.randn((layers, pages, hkv, 16, d), generator=g, device=cuda).to(dtype)
    v = torch.randn((layers, pages, hkv, 16, d), generator=g, device=cuda).to(dtype)
    weights = torch.randn((layers, seqs, hkv, cap), generator=g, device=cuda).exp()
    if kind == "ties":
        weights = (4 * torch.rand((layers, seqs, hkv, cap), generator=g, device=cuda)).floor() - 1.0
        weights = torch.where(weights == 0, torch.where(torch.rand_like(weights) < 0.5, -0.0, 0.0), weights)
    elif kind == "odd":
        pick = torch.randint(0, 6, weights.shape, generator=g, device=cuda)
        for i, x in enumerate((NAN, INF, -INF, 1e-42)):
            weights[pick == i] = x
    seen = ints([2 * n for n in lengths], cuda)
    pos = torch.stack([torch.randperm(2 * max(most, cap), generator=g, device=cuda)[:cap]
                       for _ in range(layers * seqs * hkv)]).to(torch.int32).view(layers, seqs, hkv, cap)
    return k, v, table, ints(lengths, cuda), seen, weights.contiguous(), pos.contiguous()


def evict_check(case, budget, recent=0, sinks=0, in_place=True):
    k, v, table, lengths, seen, weights, pos = (t.clone() for t in case)
    wk, wv, ww, wp, left = evict_plain(k, v, table, lengths, seen, weights, pos, budget, recent, sinks)
    wo = weights if in_place else torch.full_like(weights, -3.0)
    po = pos if in_place else torch.full_like(pos, -3)
    got = kernels.cache_evict(k, v, table, lengths, seen, weights, pos, budget=budget, recent=recent, sinks=sinks,
                              weights_out=None if in_place else wo, pos_out=None if in_place else po)
    assert got.tolist() == left
    assert same(k, wk) and same(v, wv)
    if not in_place:  # nothing is written behind the new ends
        behind = torch.arange(wo.shape[-1], device=wo.device) >= got[None, :, None, None]
        ww, wp = torch.where(behind, -3.0, ww), torch.where(behind, -3, wp)
        assert same(weights, case[5]) and torch.equal(pos, case[6])
    assert same(wo, ww) and torch.equal(po, wp)


@pytest.mark.parametrize("kind", ["heavy", "ties", "odd"])
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("lengths,budget,recent,sinks", [([1], 1, 0, 0), ([1, 2, 3], 1, 0, 0), ([17, 0, 100, 40], 40, 5, 3),
                                                         ([333, 1000], 999, 0, 0), ([333, 1000], 31, 31, 0),
                                                         ([64, 700], 300, 100, 200), ([50, 20], 0, 0, 0)])
def test_evict(cuda, kind, in_place, lengths, budget, recent, sinks):
    case = evict_case(cuda, budget + len(lengths), lengths, 2, 3, 32, torch.bfloat16, kind=kind)
    evict_check(case, budget, recent, sinks, in_place)


@pytest.mark.parametrize("dtype,d", [(torch.float16, 64), (torch.float32, 5), (torch.bfloat16, 3), (torch.bfloat16, 256),
                                     (torch.float16, 72)])
def test_evict_moves_any_type_and_head_size(cuda, dtype, d):
    evict_check(evict_case(cuda, d, [90, 33], 1, 2, d, dtype), 40, 10, 2)


@pytest.mark.parametrize("length,budget", [(5000, 1250), (20000, 19990), (40000, 7), (70001, 30000), (9000, 4500),
                                           (262144, 100000)])
def test_evict_long_rows(cuda, length, budget):
    evict_check(evict_case(cuda, budget, [length, 100], 1, 1, 8, torch.bfloat16), budget, min(7, budget), 0)
    evict_check(evict_case(cuda, budget, [length], 1, 1, 8, torch.bfloat16, kind="ties"), budget, min(7, budget), 0, False)


def test_evict_lengths_beyond_the_tables(cuda):
    """A length past the weights or the page table is cut to them, a negative one is zero; a page that is none is skipped."""
    k, v, table, lengths, seen, weights, pos = evict_case(cuda, 2, [100, 90, 80], 1, 2, 32, torch.bfloat16, cap=70)
    lengths = ints([1000, -4, 60], cuda)
    evict_check((k, v, table, lengths, seen, weights, pos), 20, 4, 0)
    table2 = table.clone()
    table2[0, 3] = -1
    table2[2, 0] = 10**6
    got = kernels.cache_evict(k, v, table2, lengths, seen, weights, pos, budget=20)
    assert got.tolist() == [20, 0, 20]


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("length,budget", [(100, 40), (3000, 1000), (3000, 2990)])
def test_evict_over_pages_that_are_none(cuda, in_place, length, budget):
    """A slot whose page lies outside the cache neither moves nor is moved to: every slot of the cache holds the token that
    slot_pos names, with its weight."""
    g = gen(cuda, 3)
    table, pages = page_table(g, 2, length)
    cap = table.shape[1] * 16
    pos = torch.stack([torch.randperm(cap, generator=g, device=cuda) for _ in range(4)]).to(torch.int32).view(2, 2, cap)
    k = torch.zeros((pages, 2, 16, 8), device=cuda)
    for s in range(2):
        rows = pos[s].view(2, -1, 16).transpose(0, 1).float()
        k[table[s].long()] = rows[..., None].expand(-1, -1, -1, 8)
    v = k + 0.5
    heavy = torch.rand((2, 2, cap), generator=g, device=cuda)  # a token's weight, by head
    weights = torch.gather(heavy, 2, pos.long())
    bad = table.clone()
    for s, page in ((0, 1), (0, table.shape[1] - 1), (1, 0), (1, table.shape[1] - 2)):
        bad[s, page] = -1 if page else 10**6
    wo = weights if in_place else torch.full_like(weights, -3.0)
    po = pos if in_place else torch.full_like(pos, -3)
    was = pos.clone()
    left = kernels.cache_evict(k, v, bad, ints([length, length], cuda), ints([cap, cap], cuda), weights, pos, budget=budget,
                               weights_out=None if in_place else wo, pos_out=None if in_place else po)
    assert left.tolist() == [budget] * 2
    now = po[:, :, :budget]
    assert torch.equal(wo[:, :, :budget], torch.gather(heavy, 2, now.long()))
    moved = 0
    for s in range(2):
        held = k[table[s].long()].transpose(0, 1).flatten(1, 2)[:, :budget]
        on = ((bad[s] >= 0) & (bad[s] < pages)).repeat_interleave(16)[:budget]
        assert torch.equal(held[:, on], now[s][:, on, None].float().expand(-1, -1, 8))
        assert torch.equal(now[s][:, ~on], was[s][:, :budget][:, ~on])
        moved += int((now[s] != was[s][:, :budget]).sum())
    assert moved > 0 and torch.equal(v, k + 0.5)


def test_evict_protects_more_than_the_budget_has_room_for(cuda):
    """Positions that repeat (no program's) protect more slots than stay: the lower slots win."""
    k, v, table, lengths, seen, weights, pos = evict_case(cuda, 6, [60], 1, 1, 32, torch.bfloat16)
    pos.zero_()
    evict_check((k, v, table, lengths, seen, weights, pos), 20, 0, 1)
    assert kernels.cache_evict(k, v, table, lengths, seen, weights, pos, budget=20, sinks=1).tolist() == [20]


def test_evict_of_one_layer(cuda):
    k, v, table, lengths, seen, weights, pos = evict_case(cuda, 12, [60, 100], 1, 2, 64, torch.bfloat16)
    wk, wv, ww, wp, left = evict_plain(k, v, table, lengths, seen, weights, pos, 50, 8, 1)
    got = kernels.cache_evict(k[0], v[0], table, lengths, seen, weights[0], pos[0], budget=50, recent=8, sinks=1,
                              lengths_out=lengths)
    assert got is lengths and got.tolist() == left
    assert same(k, wk) and same(v, wv) and same(weights, ww) and torch.equal(pos, wp)


# ---- verification from given random numbers -----------------------------------------------------------------------
def verify_plain(p, q, drafts, u, n_drafts=None):
    """Float64 on the host, straight from the definition."""
    import numpy as np

    p, u, drafts = p.double().cpu().numpy(), u.double().cpu().numpy(), drafts.cpu().numpy()
    q = None if q is None else q.double().cpu().numpy()
    fix = lambda a: np.where(np.isfinite(a) & (a > 0), a, 0.0)  # noqa: E731
    tokens, counts = np.full((p.shape[0], p.shape[1]), -1, np.int64), []
    for b in range(p.shape[0]):
        n = p.shape[1] - 1 if n_drafts is None else min(max(int(n_drafts[b]), 0), p.shape[1] - 1)
        kept = 0
        while kept < n:
            d = drafts[b, kept]
            if not 0 <= d < p.shape[2]:
                break
            offered = 1.0 if q is None else fix(q[b, kept, d])
            if not u[b, kept] * offered < fix(p[b, kept, d]):
                break
            tokens[b, kept] = d
            kept += 1
        w = fix(p[b, kept])
        if kept < n:
            if q is not None:
                r = np.maximum(w - fix(q[b, kept]), 0.0)
            else:
                r = w.copy()
                if 0 <= drafts[b, kept] < p.shape[2]:
                    r[drafts[b, kept]] = 0.0
            w = r if r.sum() > 0 else w
        total = np.cumsum(w)
        over = np.nonzero(total > u[b, -1] * total[-1])[0]
        tokens[b, kept] = over[0] if over.size else 0
        counts.append(kept + 1)
    return tokens, counts


def verify_case(cuda, seed, b, k, v, dtype, near=0.5, sharp=2.0):
    g = gen(cuda, seed)
    logits = sharp * torch.randn((b, k + 1, v), generator=g, device=cuda)
    p = torch.softmax(logits, -1)
    q = torch.softmax(logits[:, :k] + near * torch.randn((b, k, v), generator=g, device=cuda), -1)
    p = torch.where(p > 1e-3 * p.amax(-1, keepdim=True), p, 0.0)
    drafts = torch.multinomial(q.reshape(b * k, v), 1, generator=g).view(b, k) if k else torch.zeros((b, 0), device=cuda)
    return p.to(dtype), q.to(dtype), drafts.to(torch.int32), torch.rand((b, k + 1), generator=g, device=cuda)


def verify_check(p, q, drafts, u, n_drafts=None):
    tokens, count = kernels.verify_sampled(p, q, drafts, u, n_drafts=n_drafts)
    want, counts = verify_plain(p, q, drafts, u, n_drafts)
    assert count.tolist() == counts
    assert tokens.tolist() == want.tolist()
    return counts


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dist", [True, False])
@pytest.mark.parametrize("b,k,v", [(1, 0, 1), (1, 1, 2), (3, 4, 5), (64, 3, 31), (16, 8, 33), (5, 2, 1000), (7, 5, 4099),
                                   (2, 4, 151936), (300, 2, 70)])
def test_verify_sampled(cuda, dtype, dist, b, k, v):
    p, q, drafts, u = verify_case(cuda, b + v, b, k, v, dtype)
    counts = verify_check(p, q if dist else None, drafts, u)
    if b >= 64:
        assert len(set(counts)) > 1  # some kept, some refused
    g = gen(cuda, 1)
    verify_check(p, q if dist else None, drafts, u, torch.randint(-1, k + 2, (b,), generator=g, device=cuda,
                                                                  dtype=torch.int32))


def test_verify_sampled_many_drafts(cuda):
    p, q, drafts, u = verify_case(cuda, 3, 4, 40, 50, torch.float32, near=0.0)
    counts = verify_check(q[:, :1].expand(4, 41, 50).contiguous(), q[:, :1].expand(4, 40, 50).contiguous(),
                          drafts % 50, u)
    p = torch.cat([q, q[:, :1]], 1)
    assert verify_check(p.contiguous(), q, drafts, u) == [41] * 4  # p = q keeps everything drawn from it
    assert all(c >= 1 for c in counts)


@pytest.mark.parametrize("b", [1, 2, 9, 150])
@pytest.mark.parametrize("v", [2, 4096, 32768])
def test_verify_sampled_with_little_between_start_and_meeting(cuda, b, v):
    """No drafts and few tokens a block: blocks of a cluster tell each other their sums right after their start."""
    p, _, drafts, u = verify_case(cuda, b + v, b, 0, v, torch.float32)
    verify_check(p, None, drafts, u)
    tokens, count = kernels.verify_sampled(p, None, drafts, u)
    for _ in range(200):
        got = kernels.verify_sampled(p, None, drafts, u)
        assert torch.equal(got[0], tokens) and torch.equal(got[1], count)


def test_verify_sampled_borders(cuda):
    p = torch.tensor([[0.25, 0.0, 0.25, 0.5], [0.5, 0.25, 0.0, 0.25]], device=cuda)[None]
    q = torch.tensor([[0.5, 0.0, 0.25, 0.25]], device=cuda)[None]
    for u0 in (0.0, 0.25, 0.49999997, 0.5, 0.75, 0.99999994):
        for u1 in (0.0, 0.25, 0.5, 0.74999994, 0.75, 0.99999994):
            for d in (0, 1, 2, 3, -1, 4, 2**31 - 1, -(2**31)):
                args = (p, q, ints([[d]], cuda), torch.tensor([[u0, u1]], device=cuda))
                verify_check(*args)
                verify_check(p, None, *args[2:])


def test_verify_sampled_of_what_is_no_distribution(cuda):
    u = torch.tensor([[0.3, 0.6]], device=cuda)
    one = lambda *rows: torch.tensor([rows], device=cuda)  # noqa: E731
    d = ints([[1]], cuda)
    # q covers p everywhere: nothing is left, the token comes from p; a draft without any chance leaves its own q out
    verify_check(one((0.2, 0.1, 0.2), (1.0, 0.0, 0.0)), one((0.4, 0.9, 0.4)), d, u)
    verify_check(one((0.0, 1.0, 0.0), (1.0, 0.0, 0.0)), None, d, torch.tensor([[1.0, 0.5]], device=cuda))
    verify_check(one((0.0, 0.0, 0.0), (0.0, 0.0, 0.0)), one((0.5, 0.5, 0.0)), d, u)  # nothing at all: token 0
    verify_check(one((0.0, 0.0, 0.0), (0.0, 0.0, 0.0)), None, d, u, ints([0], cuda))
    verify_check(one((NAN, -1.0, 0.5), (INF, 0.1, NAN)), one((0.1, NAN, 0.2)), d, u)
    verify_check(one((NAN, 0.5, 0.5), (INF, 0.1, 0.3)), one((0.1, INF, 0.2)), d, u)


def test_verify_sampled_outputs_over_inputs(cuda):
    """A sequence's count may take the place of its n_drafts, and its tokens that of its random numbers; one sequence's
    drafts may lie in the buffer that takes its tokens. What another sequence still reads is refused."""
    p, q, drafts, u = verify_case(cuda, 15, 40, 3, 5000, torch.float32)
    n = torch.randint(0, 4, (40,), generator=gen(cuda, 2), device=cuda, dtype=torch.int32)
    tokens, count = kernels.verify_sampled(p, q, drafts, u, n_drafts=n)
    own, over = n.clone(), u.clone()
    got = kernels.verify_sampled(p, q, drafts, over, n_drafts=own, tokens=over.view(torch.int32), count=own)
    assert torch.equal(got[0], tokens) and torch.equal(got[1], count) and got[1] is own
    for b in range(3):
        buffer = torch.cat([drafts[b, :1], drafts[b]]).view(1, 4)
        got = kernels.verify_sampled(p[b:b + 1], q[b:b + 1], buffer[:, 1:], u[b:b + 1], n_drafts=n[b:b + 1], tokens=buffer)
        assert torch.equal(got[0], tokens[b:b + 1]) and torch.equal(got[1], count[b:b + 1])
    flat = torch.zeros(400, dtype=torch.int32, device=cuda)
    held = flat[:120].view(40, 3).copy_(drafts)
    for kw, word in (({"tokens": flat[:160].view(40, 4)}, "drafts"), ({"count": flat[100:140]}, "drafts"),
                     ({"tokens": flat[200:360].view(40, 4), "count": flat[350:390]}, "count"),
                     ({"tokens": flat[200:360].view(40, 4), "n_drafts": flat[359:399].copy_(n)}, "n_drafts")):
        with pytest.raises(ValueError, match=word):
            kernels.verify_sampled(p, q, held, u, **{"n_drafts": n, **kw})
    with pytest.raises(ValueError, match="drafts"):  # upwards within one sequence
        kernels.verify_sampled(p[:1], q[:1], flat[:3].view(1, 3), u[:1], tokens=flat[1:5].view(1, 4))
    assert torch.equal(held, drafts)


def test_verify_sampled_takes_wider_rows(cuda):
    p, q, drafts, u = verify_case(cuda, 5, 3, 2, 100, torch.float32)
    wide = torch.full((9, 133), NAN, device=cuda)
    wide[:, 1:101] = p.view(9, 100)
    view = wide[:, 1:101].unflatten(0, (3, 3))
    tokens, count = kernels.verify_sampled(view, q, drafts, u)
    want, counts = verify_plain(p, q, drafts, u)
    assert tokens.tolist() == want.tolist() and count.tolist() == counts


def test_verify_sampled_draws_the_target(cuda):
    """The first token of many verifications has the target's distribution (chi-square, 9 degrees, p > 1e-4)."""
    g = gen(cuda, 77)
    p = torch.softmax(torch.randn((1, 2, 10), generator=g, device=cuda), -1)
    q = torch.softmax(torch.randn((1, 1, 10), generator=g, device=cuda), -1)
    n = 60000
    drafts = torch.multinomial(q[0, 0].expand(n, 10), 1, generator=g).to(torch.int32)
    u = torch.rand((n, 2), generator=g, device=cuda)
    tokens, _ = kernels.verify_sampled(p.expand(n, 2, 10).contiguous(), q.expand(n, 1, 10).contiguous(), drafts, u)
    seen = torch.bincount(tokens[:, 0].long(), minlength=10).double()
    want = n * p[0, 0].double() / p[0, 0].double().sum()
    assert float(((seen - want) ** 2 / want).sum()) < 33.7


# ---- together ---------------------------------------------------------------------------------------------------
def test_decoding_over_a_bounded_cache(cuda):
    """Tokens are turned and written, attended with their weights, and the cache is cut whenever it is full: what stays is
    what a float64 program of the same rules keeps, and the outputs are its outputs."""
    g = gen(cuda, 42)
    hq, hkv, d, budget, block = 4, 2, 64, 48, 16
    freq, factor = kernels.rope_frequencies(d, 10000.0, scaling="yarn", stretch=4.0, trained=64, device=cuda)
    table, pages = page_table(g, 2, budget + block)
    k = torch.zeros((pages, hkv, 16, d), dtype=torch.bfloat16, device=cuda)
    v = torch.zeros_like(k)
    weights = torch.zeros((2, hkv, budget + block), device=cuda)
    slot_pos = torch.full((2, hkv, budget + block), -1, dtype=torch.int32, device=cuda)
    lengths, seen = ints([0, 0], cuda), ints([0, 0], cuda)
    kept = [[[] for _ in range(hkv)] for _ in range(2)]  # per head: [position, k, v, weight] in slot order
    for step in range(150):
        qkv = torch.randn((2, (hq + 2 * hkv) * d), generator=g, device=cuda).to(torch.bfloat16)
        q = kernels.rope_kv(qkv, freq, seen, lengths, ints([0, 1], cuda), table, hq, hkv, d, k, v, factor=factor,
                            slot_pos=slot_pos)
        out = kernels.attention_weights(q, k, v, table, ints([0, 1, 2], cuda), lengths, weights, max_rows_per_seq=1,
                                        max_kv_len=budget + block, scale=d ** -0.5)
        turned_k = q.new_empty((2, hkv, d))
        for b in range(2):  # the turned keys as the cache holds them
            page = table[b, int(lengths[b]) // 16].long()
            turned_k[b] = k[page, :, int(lengths[b]) % 16]
            for h in range(hkv):
                heads = kept[b][h]
                heads.append([int(seen[b]), turned_k[b, h].double(), qkv[b, (hq + hkv + h) * d:][:d].double(), 0.0])
                keys, values = (torch.stack([e[i] for e in heads]) for i in (1, 2))
                for qh in range(2 * h, 2 * h + 2):
                    p = torch.softmax(d ** -0.5 * (keys @ q[b, qh].double()), 0)
                    torch.testing.assert_close(out[b, qh].double(), p @ values, rtol=2.0**-8, atol=2.0**-12)
                    for e, x in zip(heads, p.tolist()):
                        e[3] += x
        lengths += 1
        seen += 1
        if int(lengths[0]) == budget + block:
            kernels.cache_evict(k, v, table, lengths, seen, weights, slot_pos, budget=budget, recent=8, sinks=2,
                                lengths_out=lengths)
            assert lengths.tolist() == [budget, budget]
            for b in range(2):
                for h in range(hkv):
                    heads = kept[b][h]
                    order = sorted(range(len(heads)), key=lambda j: (
                        not (heads[j][0] < 2 or heads[j][0] >= int(seen[b]) - 8), -heads[j][3]))
                    chosen = order[:budget]
                    # a near-tie at the border could go either way in float32
                    assert heads[order[budget - 1]][3] - heads[order[budget]][3] > 1e-5 or order[budget - 1] in range(
                        len(heads) - 8, len(heads))
                    holes = [j for j in range(budget) if j not in chosen]
                    movers = [j for j in range(budget, len(heads)) if j in chosen]
                    for to, at in zip(holes, movers):
                        heads[to] = heads[at]
                    del heads[budget:]
                    assert slot_pos[b, h, :budget].tolist() == [e[0] for e in heads]
                    got = weights[b, h, :budget].double()
                    want = torch.tensor([e[3] for e in heads], dtype=torch.float64, device=cuda)
                    assert float((got - want).abs().max()) < 1e-4


def test_a_captured_step_is_replayed(cuda):
    """The four calls in one CUDA graph, twice, on inputs that change between replays; two graphs do not share scratch."""
    g = gen(cuda, 43)
    hq, hkv, d = 8, 2, 64
    freq, _ = kernels.rope_frequencies(d, 10000.0, device=cuda)
    table, pages = page_table(g, 3, 400)

    def state(seed):
        h = gen(cuda, seed)
        k = torch.randn((pages, hkv, 16, d), generator=h, device=cuda).to(torch.bfloat16)
        return {"qkv": torch.randn((3, (hq + 2 * hkv) * d), generator=h, device=cuda).to(torch.bfloat16), "k": k,
                "v": k.flip(0).contiguous(), "w": torch.rand((3, hkv, 400), generator=h, device=cuda),
                "pos": torch.arange(400, device=cuda, dtype=torch.int32).expand(3, hkv, 400).contiguous(),
                "n": ints([399, 200, 17], cuda), "p": torch.softmax(torch.randn((3, 3, 999), generator=h, device=cuda), -1),
                "q": torch.softmax(torch.randn((3, 2, 999), generator=h, device=cuda), -1),
                "d": torch.randint(0, 999, (3, 2), generator=h, device=cuda, dtype=torch.int32),
                "u": torch.rand((3, 3), generator=h, device=cuda)}

    def step(s):
        q = kernels.rope_kv(s["qkv"], freq, s["n"], s["n"], ints_012, table, hq, hkv, d, s["k"], s["v"], slot_pos=s["pos"])
        out = kernels.attention_weights(q, s["k"], s["v"], table, ints_0123, s["n"], s["w"], max_rows_per_seq=1,
                                        max_kv_len=400, scale=0.125)
        left = kernels.cache_evict(s["k"], s["v"], table, s["n"], s["n"], s["w"], s["pos"], budget=150, recent=20)
        return (out, left, *kernels.verify_sampled(s["p"], s["q"], s["d"], s["u"]))

    ints_012, ints_0123 = ints([0, 1, 2], cuda), ints([0, 1, 2, 3], cuda)
    step(state(0))
    graphs = []
    for seed in (1, 2):
        s = state(seed)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(s)
        graphs.append((graph, s, outs))
    for fresh in (3, 4):
        for i, (graph, s, outs) in enumerate(graphs):
            for name, t in state(fresh + 10 * i).items():
                s[name].copy_(t)
            graph.replay()
        for i, (graph, s, outs) in enumerate(graphs):
            want = state(fresh + 10 * i)
            for got, x in zip(outs, step(want)):
                assert torch.equal(got, x)
            for name in ("k", "v", "w", "pos"):
                assert torch.equal(s[name], want[name])


def test_calls_on_two_streams_at_once(cuda):
    case = attend_case(cuda, 3, [300, 77], [2, 1], 8, 2, 64, torch.bfloat16)
    p, q, drafts, u = verify_case(cuda, 9, 8, 3, 5000, torch.float32)
    ev = evict_case(cuda, 14, [900, 333], 2, 2, 64, torch.bfloat16)

    def work():
        w, e = case[6].clone(), [t.clone() for t in ev]
        out = kernels.attention_weights(*case[:6], w, max_rows_per_seq=2, max_kv_len=320, scale=0.1)
        left = kernels.cache_evict(*e, budget=100, recent=3)
        return (out, w, left, e[0], e[5], *kernels.verify_sampled(p, q, drafts, u))

    want = work()
    streams = [torch.cuda.Stream(cuda) for _ in range(2)]
    got = []
    for _ in range(3):
        for st in streams:
            st.wait_stream(torch.cuda.current_stream(cuda))
            with torch.cuda.stream(st):
                got.append(work())
    torch.cuda.synchronize()
    for outs in got:
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


def test_caches_whose_offsets_pass_32_bits(cuda):
    """Pages far behind 2^31 values of a cache: the bits of the same pages in a small one."""
    far, hq, hkv, d = 140000, 8, 8, 128
    g = gen(cuda, 50)
    small = [torch.randn((40, hkv, 16, d), generator=g, device=cuda).to(torch.bfloat16) for _ in range(2)]
    large = [torch.empty((far, hkv, 16, d), dtype=torch.bfloat16, device=cuda) for _ in range(2)]
    for a, b in zip(small, large):
        b[far - 40:] = a
    table = torch.randperm(40, generator=g, device=cuda).to(torch.int32).view(2, 20).contiguous()
    qkv = torch.randn((2, (hq + 2 * hkv) * d), generator=g, device=cuda).to(torch.bfloat16)
    freq, _ = kernels.rope_frequencies(d, 10000.0, device=cuda)
    outs = []
    for (k, v), pages in ((small, table), (large, table + (far - 40))):
        n, w = ints([311, 250], cuda), torch.rand((2, hkv, 320), generator=gen(cuda, 51), device=cuda)
        pos = torch.arange(320, device=cuda, dtype=torch.int32).expand(2, hkv, 320).contiguous()
        q = kernels.rope_kv(qkv, freq, n, n, ints([0, 1], cuda), pages, hq, hkv, d, k, v, slot_pos=pos)
        out = kernels.attention_weights(q, k, v, pages, ints([0, 1, 2], cuda), n, w, max_rows_per_seq=1, max_kv_len=320,
                                        scale=0.1)
        left = kernels.cache_evict(k, v, pages, n, n, w, pos, budget=100, recent=10)
        outs.append((q, out, left, w, pos, k[-40:], v[-40:]))
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_layers_whose_offsets_pass_32_bits(cuda):
    k = torch.empty((3, 50000, 8, 16, 128), dtype=torch.bfloat16, device=cuda)  # 2.4 * 10^9 values
    v = torch.empty_like(k)
    g = gen(cuda, 52)
    table = ints([[49990, 3, 49999, 17]], cuda)
    for t in (k, v):
        t[:, table[0].long()] = torch.randn((3, 4, 8, 16, 128), generator=g, device=cuda).to(torch.bfloat16)
    w = torch.rand((3, 1, 8, 64), generator=g, device=cuda)
    pos = torch.arange(64, device=cuda, dtype=torch.int32).expand(3, 1, 8, 64).contiguous()
    near = [t[:, table[0].long()].clone() for t in (k, v)]
    args = (ints([[0, 1, 2, 3]], cuda), ints([60], cuda), ints([60], cuda), w.clone(), pos.clone())
    kernels.cache_evict(*near, *args, budget=20, recent=3)
    kernels.cache_evict(k, v, table, *args[1:3], w, pos, budget=20, recent=3)
    assert torch.equal(k[:, table[0].long()], near[0]) and torch.equal(v[:, table[0].long()], near[1])
    assert torch.equal(w, args[3]) and torch.equal(pos, args[4])


FIRST_CALL_CAPTURED = """
import sys
import torch
sys.path.insert(0, sys.argv[1])
from ironmule_b200 import kernels
dev = torch.device("cuda:0")
g = torch.Generator(device=dev).manual_seed(1)
k = torch.randn((4, 2, 16, 64), generator=g, device=dev).to(torch.bfloat16)
v = k.flip(0).contiguous()
n = torch.tensor([40], dtype=torch.int32, device=dev)
i01 = torch.tensor([0, 1], dtype=torch.int32, device=dev)
table = torch.arange(4, dtype=torch.int32, device=dev).view(1, 4)
w = torch.rand((1, 2, 64), generator=g, device=dev)
pos = torch.arange(64, dtype=torch.int32, device=dev).expand(1, 2, 64).contiguous()
p = torch.softmax(torch.randn((1, 2, 9999), generator=g, device=dev), -1)
u = torch.tensor([[0.9, 0.3]], device=dev)
qkv = torch.randn((1, 8 * 64), generator=g, device=dev).to(torch.bfloat16)
freq, _ = kernels.rope_frequencies(64, 10000.0, device=dev)
kept = [t.clone() for t in (k, v, w, pos)]
def step(k, v, w, pos):
    q = kernels.rope_kv(qkv, freq, n, n, i01[:1], table, 4, 2, 64, k, v, slot_pos=pos)
    out = kernels.attention_weights(q, k, v, table, i01, n, w, max_rows_per_seq=1, max_kv_len=64, scale=0.1)
    left = kernels.cache_evict(k, v, table, n, n, w, pos, budget=20)
    return out, left, *kernels.verify_sampled(p, p[:, :1].contiguous(), i01[:1].view(1, 1), u)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    outs = step(k, v, w, pos)
graph.replay()
for a, b in zip(outs, step(*kept)):
    assert torch.equal(a, b)
for a, b in zip((k, v, w, pos), kept):
    assert torch.equal(a, b)
print("ok")
"""


def test_the_first_calls_of_a_process_may_be_captured(cuda):
    import subprocess
    import sys
    from pathlib import Path

    root = Path(__file__).resolve().parents[1]
    run = subprocess.run([sys.executable, "-c", FIRST_CALL_CAPTURED, str(root)], capture_output=True, text=True,
                         timeout=300, cwd=root)
    assert run.returncode == 0 and run.stdout.strip().endswith("ok"), run.stdout + run.stderr


# ---- refusals ---------------------------------------------------------------------------------------------------
def refuses(fn, *args, error=ValueError, match=None, **kw):
    with pytest.raises(error, match=match):
        fn(*args, **kw)


def test_refusals_of_the_wrappers(cuda):
    x = torch.zeros((4, 2, 16), device=cuda)
    pos, freq = ints([0, 1, 2, 3], cuda), torch.ones(8, device=cuda)
    refuses(kernels.rope, x.cpu(), pos, freq, error=TypeError)
    refuses(kernels.rope, x.double(), pos, freq, error=TypeError)
    refuses(kernels.rope, x[0], pos, freq, match="M, H, D")
    refuses(kernels.rope, x.transpose(1, 2), pos, freq, match="contiguous heads")
    refuses(kernels.rope, x, pos[:3], freq, match="positions")
    refuses(kernels.rope, x, pos.float(), freq, error=TypeError)
    refuses(kernels.rope, x, pos, torch.ones(9, device=cuda), match="turns 18")
    refuses(kernels.rope, x, pos, freq, layout="other", match="layout")
    refuses(kernels.rope, x, pos, freq, out=x[:, :1].expand(4, 2, 16), match="apart")
    flat = torch.zeros(200, device=cuda)
    refuses(kernels.rope, flat[:128].view(4, 2, 16), pos, freq, out=flat[8:136].view(4, 2, 16), match="overlaps")
    q, k, v, table, bounds, slot, weights = attend_case(cuda, 3, [30, 40], [1, 1], 4, 2, 64, torch.bfloat16)
    kw = {"max_rows_per_seq": 1, "max_kv_len": 40, "scale": 1.0}
    refuses(kernels.attention_weights, q.float(), k, v, table, bounds, slot, weights, error=TypeError, **kw)
    refuses(kernels.attention_weights, q, k.half(), v, table, bounds, slot, weights, error=TypeError, **kw)
    refuses(kernels.attention_weights, q, k, v[:-1].contiguous(), table, bounds, slot, weights, match="caches", **kw)
    refuses(kernels.attention_weights, q[:, :3].contiguous(), k, v, table, bounds, slot, weights, match="heads", **kw)
    refuses(kernels.attention_weights, q, k, v, table, bounds, slot[:1], weights, match="row_slot", **kw)
    refuses(kernels.attention_weights, q, k, v, table[:1].contiguous(), bounds, slot, weights, match="sequences", **kw)
    refuses(kernels.attention_weights, q, k, v, table, bounds, slot, weights[:, :1].contiguous(), match="weights", **kw)
    refuses(kernels.attention_weights, q, k, v, table, bounds, slot, weights, weights_out=weights[:1], match="weights_out",
            **kw)
    twice = torch.zeros(3 * 4 * 64, dtype=torch.bfloat16, device=cuda)
    refuses(kernels.attention_weights, twice[:512].view(2, 4, 64), k, v, table, bounds, slot, weights, match="overlaps",
            out=twice[256:].view(2, 4, 64), **kw)
    none = torch.zeros((2, 2, 0), device=cuda)  # no slot's weight is kept
    out = kernels.attention_weights(q, k, v, table, bounds, slot, none, **kw)
    assert torch.equal(out, kernels.attention_weights(q, k, v, table, bounds, slot, weights.clone(), **kw))
    from ironmule_b200 import _lib

    refuses(kernels.attention_weights, q, k, v, table, bounds, slot, weights, keys_per_split=65, error=_lib.KernelError,
            **kw)
    odd = attend_case(cuda, 3, [30], [1], 2, 2, 24, torch.bfloat16)
    refuses(kernels.attention_weights, *odd, error=_lib.KernelUnsupported, match="head_dim", **kw)
    k5, v5, table, lengths, seen, weights, spos = evict_case(cuda, 12, [60, 100], 2, 2, 64, torch.bfloat16)
    refuses(kernels.cache_evict, k5, v5, table, lengths, seen, weights, spos, budget=10, recent=8, sinks=3, match="budget")
    refuses(kernels.cache_evict, k5, v5, table, lengths, seen, weights[0], spos, budget=10, match="weights")
    refuses(kernels.cache_evict, k5, v5, table, lengths[:1], seen, weights, spos, budget=10, match="lengths")
    refuses(kernels.cache_evict, k5, v5, table, lengths, seen, weights, spos[..., :50].contiguous(), budget=10,
            match="slot_pos")
    both = torch.zeros(4, dtype=torch.int32, device=cuda)
    for out, what in ((seen, "seen"), (both[1:3], "seen"), (both[:2], "lengths")):
        refuses(kernels.cache_evict, k5, v5, table, lengths if what == "seen" else both[1:3],
                seen if out is seen else both[2:], weights, spos, budget=10, lengths_out=out, match=what)
    refuses(kernels.cache_evict, k5, v5, table, lengths, seen, weights, spos, budget=2**70, match="64-bit")
    refuses(kernels.cache_evict, k5, v5.half(), table, lengths, seen, weights, spos, budget=10, error=TypeError)
    p, q, drafts, u = verify_case(cuda, 9, 2, 3, 50, torch.float32)
    refuses(kernels.verify_sampled, p[:, :3], q, drafts, u, match="target_probs")
    refuses(kernels.verify_sampled, p, q[:, :, :49], drafts, u, match="draft_probs")
    refuses(kernels.verify_sampled, p, q.half(), drafts, u, error=TypeError)
    refuses(kernels.verify_sampled, p, q, drafts.long(), u, error=TypeError)
    refuses(kernels.verify_sampled, p, q, drafts, u[:, :3], match="uniforms")
    refuses(kernels.verify_sampled, p.transpose(1, 2).contiguous().transpose(1, 2), q, drafts, u, match="spaced")
    refuses(kernels.verify_sampled, p, q, drafts, u, n_drafts=ints([1], cuda), match="n_drafts")

"""Decoding over a bounded cache without a GPU: frequency tables, and what the C entry points refuse."""
from __future__ import annotations

import math
import re
from pathlib import Path

import pytest
import torch

from ironmule_b200 import _lib, kernels


def _status(name, *args):
    lib = _lib.load()
    return getattr(lib, name)(*args), lib.im_last_error().decode()


def table(rotary, base, **kw):
    freq, factor = kernels.rope_frequencies(rotary, base, device="cpu", **kw)
    assert freq.dtype == torch.float64 and freq.shape == (rotary // 2,)
    return freq.tolist(), factor


def test_frequencies():
    plain, factor = table(8, 10000.0)
    assert factor == 1.0 and plain == pytest.approx([1.0, 0.1, 0.01, 0.001], rel=1e-14)
    linear, factor = table(8, 10000.0, scaling="linear", stretch=4.0)
    assert factor == 1.0 and linear == pytest.approx([x / 4 for x in plain], rel=1e-14)
    ntk, factor = table(8, 10000.0, scaling="ntk", stretch=4.0)
    assert factor == 1.0 and ntk[0] == 1.0 and ntk[-1] == pytest.approx(plain[-1] / 4, rel=1e-13)
    yarn, factor = table(64, 10000.0, scaling="yarn", stretch=8.0, trained=4096)
    plain, _ = table(64, 10000.0)
    assert factor == pytest.approx(0.1 * math.log(8.0) + 1.0, rel=1e-15)
    turns = [4096 * f / (2 * math.pi) for f in plain]
    for f, y, t in zip(plain, yarn, turns):
        assert f / 8 * (1 - 1e-14) <= y <= f * (1 + 1e-14)
        if t > 40.0:
            assert y == pytest.approx(f, rel=1e-14)
        if t < 0.75:
            assert y == pytest.approx(f / 8, rel=1e-14)
    assert all(a >= b for a, b in zip(yarn, yarn[1:]))
    assert table(64, 10000.0, scaling="yarn", stretch=1.0, trained=4096) == (pytest.approx(plain, rel=1e-14), 1.0)


@pytest.mark.parametrize("args,kw", [((0, 1e4), {}), ((7, 1e4), {}), ((8, 1.0), {}), ((8, math.inf), {}),
                                     ((8, 1e4), {"scaling": "other"}), ((8, 1e4), {"scaling": "linear", "stretch": 0.5}),
                                     ((2, 1e4), {"scaling": "ntk", "stretch": 2.0}),
                                     ((8, 1e4), {"scaling": "yarn", "stretch": 2.0}),
                                     ((8, 1e4), {"scaling": "yarn", "stretch": 2.0, "trained": 9, "fast": 1.0, "slow": 2.0})])
def test_frequencies_refused(args, kw):
    with pytest.raises(ValueError):
        kernels.rope_frequencies(*args, device="cpu", **kw)


def rope(x=256, row=32, head=16, pos=256, freq=256, rotary=8, layout=0, m=2, h=2, d=16, dtype=0, out=256):
    return _status("im_rope", x, row, head, pos, 0, freq, 0, rotary, 1.0, layout, 0, m, h, d, dtype, out, row, head, None)


def test_rope_refusals():
    assert rope(m=0)[0] == _lib.IM_OK and rope(h=0)[0] == _lib.IM_OK
    for kw, word in (({"m": -1}, "sizes"), ({"d": 0}, "sizes"), ({"layout": 2}, "layout"), ({"dtype": 3}, "type"),
                     ({"rotary": 7}, "turn"), ({"rotary": 18}, "turn"), ({"x": None}, "null"), ({"freq": None}, "null"),
                     ({"out": None}, "null"), ({"x": 257}, "misaligned"), ({"pos": 258}, "misaligned")):
        rc, msg = rope(**kw)
        assert rc == _lib.IM_INVALID and word in msg, (kw, msg)
    assert rope(h=1 << 17)[0] == _lib.IM_UNSUPPORTED and rope(m=1 << 31)[0] == _lib.IM_UNSUPPORTED


def rope_kv(m=2, hq=4, hkv=2, d=16, dtype=0, rotary=16, layout=0, ptr=256, slot_pos=None, cap=0):
    return _status("im_rope_kv", ptr, 256, 0, rotary, 1.0, layout, ptr, ptr, ptr, ptr, 1, 1, 1, m, hq, hkv, d, dtype, ptr,
                   ptr, ptr, slot_pos, cap, None)


def test_rope_kv_refusals():
    assert rope_kv(m=0)[0] == _lib.IM_OK
    for kw, word in (({"hq": 3}, "sizes"), ({"m": -2}, "sizes"), ({"cap": -1}, "sizes"), ({"layout": -1}, "layout"),
                     ({"dtype": -1}, "type"), ({"rotary": 32}, "turn"), ({"ptr": None}, "null"),
                     ({"slot_pos": 258}, "misaligned")):
        rc, msg = rope_kv(**kw)
        assert rc == _lib.IM_INVALID and word in msg, (kw, msg)
    assert rope_kv(d=8192)[0] == _lib.IM_UNSUPPORTED


def attend(b=2, rows=1, hq=4, hkv=2, d=64, kv=100, kps=0, window=0, dtype=0, ptr=256, ws=256, size=1 << 40, m=2, cap=100):
    return _status("im_attention_weights", ptr, ptr, ptr, dtype, ptr, 2, 7, 14, ptr, None, ptr, m, b, rows, hq, hkv, d, kv,
                   kps, window, 1.0, ptr, ptr, cap, ptr, ws, size, None)


def test_attention_weights_refusals():
    assert attend(b=0)[0] == attend(rows=0)[0] == attend(m=0)[0] == _lib.IM_OK
    for kw, word in (({"hq": 3}, "sizes"), ({"b": -1}, "sizes"), ({"window": -1}, "sizes"), ({"cap": -1}, "sizes"),
                     ({"kps": 65}, "multiple of 64"), ({"kps": -64}, "multiple of 64"), ({"ptr": None}, "null"),
                     ({"ptr": 264}, "aligned"), ({"ws": None, "window": 9}, "workspace"),
                     ({"ws": 128, "window": 9}, "workspace"), ({"size": 64, "window": 9}, "workspace")):
        rc, msg = attend(**kw)
        assert rc == _lib.IM_INVALID and word in msg, (kw, msg)
    for kw, word in (({"dtype": 2}, "type"), ({"d": 8}, "head_dim"), ({"d": 72}, "head_dim"), ({"d": 272}, "head_dim"),
                     ({"b": 70000}, "large"), ({"kv": 1 << 31}, "large")):
        rc, msg = attend(**kw)
        assert rc == _lib.IM_UNSUPPORTED and word in msg, (kw, msg)
    lib = _lib.load()
    need = lib.im_attention_weights_workspace_bytes(2, 1, 4, 2, 64, 100, 0, 9)
    assert need > 0 and attend(size=need - 1, window=9)[0] == _lib.IM_INVALID
    assert lib.im_attention_weights_workspace_bytes(2, 1, 4, 2, 64, 100, 0, 0) == 0  # one kernel, nothing to hold
    assert lib.im_attention_weights_workspace_bytes(2, 1, 4, 2, 64, 10000, 0, 0) > 0
    assert lib.im_attention_weights_workspace_bytes(0, 1, 4, 2, 64, 100, 0, 0) == 0
    assert lib.im_attention_weights_workspace_bytes(1, 1, 3, 2, 64, 100, 0, 0) == 0


def evict(layers=1, s=2, hkv=2, cap=100, row=128, budget=50, recent=0, sinks=0, ptr=256, ws=256, size=1 << 40):
    return _status("im_cache_evict", ptr, ptr, layers, 1 << 20, 14, ptr, 7, ptr, ptr, ptr, ptr, ptr, ptr, ptr, s, hkv, cap,
                   row, budget, recent, sinks, ws, size, None)


def test_evict_refusals():
    assert evict(layers=0)[0] == evict(s=0)[0] == _lib.IM_OK
    for kw, word in (({"hkv": 0}, "sizes"), ({"cap": 0}, "sizes"), ({"budget": -1}, "sizes"), ({"sinks": -1}, "sizes"),
                     ({"recent": 40, "sinks": 11}, "budget"), ({"recent": 51}, "budget"), ({"ptr": None}, "null"),
                     ({"ws": None, "cap": 900, "budget": 400}, "workspace"),
                     ({"ws": 8, "cap": 20000}, "workspace"), ({"size": 16, "cap": 20000}, "workspace")):
        rc, msg = evict(**kw)
        assert rc == _lib.IM_INVALID and word in msg, (kw, msg)
    assert evict(cap=262145)[0] == _lib.IM_UNSUPPORTED and evict(layers=1 << 30)[0] == _lib.IM_UNSUPPORTED
    lib = _lib.load()
    assert lib.im_cache_evict_workspace_bytes(1, 2, 2, 100, 50) == 0  # a row's own block moves its slots
    assert lib.im_cache_evict_workspace_bytes(1, 2, 2, 900, 400) > 0
    rc, msg = evict(recent=2**62, sinks=2**62, budget=2**62 + 2**61)  # a sum past 64 bits
    assert rc == _lib.IM_INVALID and "budget" in msg


def verify(b=2, k=3, v=50, ld=50, dtype=2, ptr=256, q=256, n=None):
    return _status("im_verify_sampled", ptr, ld, q, ld, dtype, ptr, k, n, ptr, k + 1, b, k, v, ptr, ptr, None)


def test_verify_refusals():
    assert verify(b=0)[0] == _lib.IM_OK
    for kw, word in (({"b": -1}, "sizes"), ({"v": 0}, "sizes"), ({"ld": 49}, "sizes"), ({"k": -1}, "sizes"),
                     ({"dtype": 5}, "type"), ({"ptr": None}, "null"), ({"q": 258}, "misaligned"), ({"n": 2}, "misaligned")):
        rc, msg = verify(**kw)
        assert rc == _lib.IM_INVALID and word in msg, (kw, msg)
    assert verify(b=1 << 16)[0] == _lib.IM_UNSUPPORTED and verify(k=5000)[0] == _lib.IM_UNSUPPORTED


def test_wrappers_need_cuda_tensors():
    x = torch.zeros((1, 1, 4))
    i = torch.zeros((1,), dtype=torch.int32)
    with pytest.raises(TypeError):
        kernels.rope(x, i, torch.ones(2))
    with pytest.raises(ValueError):
        kernels.rope_kv(torch.zeros((1, 12)), torch.ones(2), i, i, i, i.view(1, 1), 1, 1, 4, x, x)
    with pytest.raises(ValueError):
        kernels.cache_evict(torch.zeros((1, 1, 16, 4)), torch.zeros((1, 1, 16, 4)), i.view(1, 1), i, i,
                            torch.zeros((1, 1, 16)), torch.zeros((1, 1, 16), dtype=torch.int32), budget=4)
    with pytest.raises(TypeError):
        kernels.verify_sampled(torch.zeros((1, 1, 4)), None, torch.zeros((1, 0), dtype=torch.int32), torch.zeros((1, 1)))


@pytest.mark.parametrize("name", sorted(kernels._WORDS))
def test_calls_in_one_array_answer_as_the_entries_do(name):
    """Every argument arrives at its place: small pointers and sizes, one of them wrong at a time, are refused alike."""
    lib = _lib.load()
    entry, pack = kernels._WORDS[name]
    kinds = [t.__name__ for t in _lib.SIGNATURES[name][1]]
    good = {"im_rope": (256, 16, 16, 256, 0, 256, 0, 4, 1.0, 0, 0, 1, 1, 16, 0, 256, 16, 16, 0),
            "im_rope_kv": (256, 256, 0, 4, 1.0, 0, 256, 256, 256, 256, 1, 1, 1, 1, 4, 2, 16, 0, 256, 256, 256, 256, 16, 0),
            "im_attention_weights": (256, 256, 256, 0, 256, 1, 1, 1, 256, 256, 256, 1, 1, 1, 4, 2, 16, 16, 0, 0, 1.0, 256,
                                     256, 16, 256, 256, 1 << 30, 0),
            "im_cache_evict": (256, 256, 1, 512, 1, 256, 1, 256, 512, 256, 256, 256, 256, 256, 1, 2, 16, 32, 8, 2, 2, 256,
                               1 << 30, 0),
            "im_verify_sampled": (256, 64, 256, 64, 0, 256, 2, 256, 256, 3, 1, 2, 64, 256, 256, 0)}[name]
    assert len(good) == len(kinds)
    refused = 0
    for at, kind in enumerate(kinds[:-1]):
        for bad in (257, 0, -1, 1 << 20, 1 << 40) if kind not in ("c_double", "c_float") else (0.5,):
            args = [*good]
            args[at] = bad
            # a second fault, so that nothing is ever launched: a type that is none, more recent slots than any budget
            if name == "im_cache_evict":
                args[19] = 1 << 41
            else:
                args[[i for i, k in enumerate(kinds) if k == "c_int"][-1]] = 9
            if kind == "c_int" and bad == 1 << 40:
                continue  # not an int
            want = getattr(lib, name)(*args), lib.im_last_error()
            words = pack(entry, *args)
            assert (lib.im_bounded_call(words, len(words)), lib.im_last_error()) == want, (at, bad)
            refused += want[0] != _lib.IM_OK
    assert refused > len(kinds)


def test_calls_in_one_array_refusals():
    lib = _lib.load()
    words = kernels._WORDS["im_verify_sampled"][1](*[0] * 17)
    for given, size in ((None, 136), (words, 0), (words, 7), (words, 136), (words, 128), (words, 1 << 20)):
        assert lib.im_bounded_call(given, size) == _lib.IM_INVALID and b"im_bounded_call" in lib.im_last_error()
    for entry in (-1, 5, 1 << 40):
        words = kernels._WORDS["im_verify_sampled"][1](entry, *[0] * 16)
        assert lib.im_bounded_call(words, 136) == _lib.IM_INVALID


def test_blocks_of_a_cluster_meet_before_they_reach_into_each_other():
    """A block's shared memory may be read or written by others once it is known to run: in every kernel's text a meeting
    of the cluster stands before the first remote address."""
    seen = 0
    for path in sorted((Path(kernels.__file__).parent / "csrc").glob("*.cu*")):
        text = re.sub(r"//[^\n]*", "", path.read_text())
        for body in text.split("__global__")[1:]:
            remote = body.find("map_shared_rank")
            if remote < 0:
                continue
            seen += 1
            met = re.search(r"\.(sync|barrier_wait)\(", body)
            assert met and met.start() < remote, f"{path.name}: remote shared memory before a meeting"
    assert seen >= 3

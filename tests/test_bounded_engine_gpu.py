"""BoundedDecoder on the GPU: plain decoding until the cache is cut, and a cut cache that holds what it says."""
from __future__ import annotations

import pytest
import torch

from ironmule_b200 import engine

pytestmark = pytest.mark.gpu


def model(cuda, ctx, name="tiny-target", **kw):
    return engine.QuantModel(engine.PRESETS[name], cuda, seed=5, sigma=0.08, max_ctx=ctx, max_rows=64, **kw)


def tokens(cuda, n, seed=0):
    gen = torch.Generator(device=cuda).manual_seed(seed)
    return torch.randint(0, 1000, (n,), generator=gen, device=cuda, dtype=torch.int32)


def test_until_the_first_cut_it_is_plain_decoding(cuda):
    bounded, plain = model(cuda, 256, max_seqs=2), model(cuda, 256)
    dec = engine.BoundedDecoder(bounded, 200)
    text = tokens(cuda, 150)
    for at in (0, 90, 149):  # one token's logits behind a prefix in chunks, then token by token
        got = dec.feed(text[dec._seen[1]:at + 1], seq=1, logits=True).float()
        plain.prefill(text[:at])
        want = plain.logits_for(text[at:at + 1], at).float()
        assert float((got - want).abs().max()) <= 2e-2 * float(want.abs().max())
    assert dec.cuts == 0 and dec.lengths.tolist() == [0, 150] and dec.seen.tolist() == [0, 150]
    # every row spreads a weight of one: per kv head its query heads' share, in all of them the number of rows
    c = bounded.cfg
    total = dec.weights[:, 1].double().sum(dim=(1, 2))
    assert float((total / (150 * c.heads) - 1).abs().max()) < 1e-4
    assert dec.slot_pos[:, 1, :, :150].eq(torch.arange(150, device=cuda)).all()


def test_a_cut_cache_holds_the_keys_of_the_tokens_it_names(cuda):
    """Layer 0's keys and values follow from token and position alone, so a slot must hold the bits that an uncut cache has
    at its token's place; the first and last tokens stay in every layer and head."""
    bounded, full = model(cuda, 128), model(cuda, 512)
    dec = engine.BoundedDecoder(bounded, 64, recent=16, sinks=4)
    text = tokens(cuda, 400, seed=3)
    full.prefill(text)
    for end in (100, 180, 181, 182, 330, 400):
        dec.feed(text[dec._seen[0]:end])
        held = dec._held[0]
        assert dec.lengths.tolist() == [held] and held <= 128 and dec.seen.tolist() == [end]
        pos = dec.slot_pos[:, 0, :, :held].long()
        ordered = pos.sort(dim=-1).values
        assert bool((ordered[..., 1:] > ordered[..., :-1]).all()) and int(pos.min()) == 0 and int(pos.max()) == end - 1
        must = torch.cat([torch.arange(4, device=cuda), torch.arange(end - 16, end, device=cuda)])
        assert bool((pos[..., None] == must).any(dim=-2).all())
        for small, large in ((bounded.k_cache, full.k_cache), (bounded.v_cache, full.v_cache)):
            rows = small[0, bounded.page_table[0].long()].transpose(0, 1).flatten(1, 2)[:, :held]
            every = large[0, full.page_table[0].long()].transpose(0, 1).flatten(1, 2)
            assert torch.equal(rows, torch.gather(every, 1, pos[0, :, :, None].expand(-1, -1, every.shape[-1])))
    assert dec.cuts >= 4


def test_a_cut_is_its_sequences(cuda):
    """A sequence's tokens stay when another's cache is cut, over the budget or not, and its logits keep their bits."""
    text, other = tokens(cuda, 130, seed=5), tokens(cuda, 300, seed=6)
    kw = {"recent": 16, "sinks": 4}
    both, alone = (engine.BoundedDecoder(model(cuda, 128, max_seqs=3), 64, **kw) for _ in range(2))
    for dec in (both, alone):
        dec.feed(text[:100], seq=1)
        dec.feed(text[:20], seq=2)
    both.feed(other, seq=0)
    assert both.cuts >= 3 and both.lengths.tolist() == [both._held[0], 100, 20] and both._held[1:] == [100, 20]
    for seq, done in ((1, 100), (2, 20)):
        for dec in (both, alone):
            assert dec._held[seq] == done
        for t in ("weights", "slot_pos"):
            assert torch.equal(getattr(both, t)[:, seq, :, :done], getattr(alone, t)[:, seq, :, :done])
        assert torch.equal(both.feed(text[done:done + 9], seq, logits=True), alone.feed(text[done:done + 9], seq, logits=True))
    both.feed(text[109:], seq=1)  # and its own cut does come
    alone.feed(text[109:], seq=1)
    assert both._held[1] == alone._held[1] < 128 and torch.equal(both.slot_pos[:, 1], alone.slot_pos[:, 1])
    assert alone.cuts == 1 and both.seen.tolist() == [300, 130, 29]
    both.cut()
    assert both._held == both.lengths.tolist() == [64, 64, 29]


def test_a_sequence_has_its_pages_to_itself(cuda):
    m = model(cuda, 96, max_seqs=2)
    dec = engine.BoundedDecoder(m, 32)
    dec.feed(tokens(cuda, 5))
    m.page_table[1, 2] = m.page_table[0, 1]
    for seq in (0, 1):
        dec.start(seq)
        with pytest.raises(ValueError, match="pages to itself"):
            dec.feed(tokens(cuda, 5), seq=seq)
    m.page_table[1, 2] = m.page_table[1, 3]
    dec.feed(tokens(cuda, 5))
    with pytest.raises(ValueError, match="pages to itself"):
        dec.generate(tokens(cuda, 5), 2, seq=1)


def test_generate_runs_past_the_cache_and_starts_afresh(cuda):
    m = model(cuda, 96)
    dec = engine.BoundedDecoder(m, 48, recent=12, sinks=2)
    prompt = tokens(cuda, 200, seed=9)
    first = dec.generate(prompt, 60)
    assert len(first) == 60 and dec.cuts >= 3 and dec._seen[0] == 259 and dec._held[0] <= 96
    assert dec.generate(prompt, 60) == first
    short = prompt[:20]
    fresh = engine.BoundedDecoder(model(cuda, 96), 48, recent=12, sinks=2)
    assert dec.generate(short, 10) == fresh.generate(short, 10)


def test_models_with_experts(cuda):
    dec = engine.BoundedDecoder(model(cuda, 96, "tiny-moe"), 32, recent=8, sinks=2)
    assert len(dec.generate(tokens(cuda, 120, seed=2), 5)) == 5 and dec.cuts >= 1


def test_refusals(cuda):
    m = model(cuda, 96)
    for budget, kw in ((0, {}), (96, {}), (200, {}), (32, {"recent": 30, "sinks": 3}), (32, {"recent": -1})):
        with pytest.raises(ValueError):
            engine.BoundedDecoder(m, budget, **kw)
    dec = engine.BoundedDecoder(m, 32)
    assert dec.feed(tokens(cuda, 0)) is None
    with pytest.raises(ValueError, match="no token"):
        dec.generate(tokens(cuda, 0), 3)
    for seq in (-1, 1):
        with pytest.raises(ValueError, match="sequence"):
            dec.generate(tokens(cuda, 5), 3, seq=seq)
        with pytest.raises(ValueError, match="sequence"):
            dec.feed(tokens(cuda, 5), seq=seq)
    with pytest.raises(ValueError, match="sliding window"):
        engine.BoundedDecoder(model(cuda, 96, "tiny-gemma"), 32)

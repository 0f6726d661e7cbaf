"""Models with experts in the speculative engine: every layer's mixture-of-experts block against float64 on the device's
own residual rows, and the engine's invariant that speculation changes no answer (a verify row has the bits of a one-row
decode)."""
from __future__ import annotations

import pytest
import torch

from ironmule_b200 import checkpoint, engine, kernels
from ironmule_b200.engine import PRESETS

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def keep_raw_experts(monkeypatch):
    """Experts hold packed weights only; the reference needs the stacked tensors they were packed from."""
    pack = kernels.Experts.__init__

    def keeping(self, w, scales, biases):
        pack(self, w, scales, biases)
        self.raw = (w, scales, biases)

    monkeypatch.setattr(kernels.Experts, "__init__", keeping)


def dense(w, s, b):
    codes = torch.stack([(w >> (4 * i)) & 15 for i in range(8)], dim=-1).flatten(-2).double()
    return codes * s.double().repeat_interleave(64, -1) + b.double().repeat_interleave(64, -1)


def rms(v, w, eps, gemma):
    return v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps) * (w.double() + (1.0 if gemma else 0.0))


def block_reference(cfg, layer, h):
    """The block's output rows in float64, and the gap between the last chosen and the first refused router score."""
    gemma = cfg.family == "gemma3"
    x = rms(h, layer.post_norm, cfg.eps, gemma)
    scores = x @ dense(layer.router.w, layer.router.s, layer.router.b).T
    top = torch.sort(scores, dim=1, descending=True)
    k = cfg.experts_per_token
    weights = torch.softmax(top.values[:, :k], dim=1)
    gu, down = dense(*layer.gate_up.raw), dense(*layer.down.raw)
    out = torch.zeros_like(h)
    for m in range(h.shape[0]):
        for j in range(k):
            e = int(top.indices[m, j])
            both = (gu[e] @ x[m]).view(-1, 2, 16)
            g, u = both[:, 0].reshape(-1), both[:, 1].reshape(-1)
            if gemma:
                a = 0.5 * g * (1.0 + torch.tanh(0.7978845608028654 * (g + 0.044715 * g**3)))
            else:
                a = g * torch.sigmoid(g)
            out[m] += weights[m, j] * (down[e] @ (a * u))
    if gemma:
        out = rms(out, layer.post_ff_norm, cfg.eps, True)
    return h + out, top.values[:, k - 1] - top.values[:, k]


@pytest.mark.parametrize("name", ["tiny-moe", "tiny-gemma-moe"])
@pytest.mark.parametrize("rows", [1, 7, 32])
def test_blocks_match_float64(cuda, name, rows):
    cfg = PRESETS[name]
    model = engine.QuantModel(cfg, cuda, seed=3, sigma=0.05, max_rows=32, max_ctx=64)
    tokens = torch.arange(rows, dtype=torch.int32, device=cuda) * 29 % cfg.vocab
    trace: list = []
    model.forward(model._meta(tokens, list(range(rows)), 0), max_kv_len=model.max_ctx, trace=trace)
    checked = 0
    for li, layer in enumerate(model.layers):
        h = trace[li]["h_mid"].double()
        want, gap = block_reference(cfg, layer, h)
        got = trace[li + 1]["h_in"].double()
        # Router logits are bf16: scores closer than their rounding may go either way, so those rows are left out.
        clear = gap > 2**-7 * 4
        # x, the scores, the experts' outputs and h' are rounded to bf16 (2^-9 each), the weights follow the scores
        scale = (want - h).abs().amax(dim=1, keepdim=True) + h.abs()
        off = (got - want).abs() / scale
        assert bool((off[clear] <= 0.03).all()), (li, float(off[clear].max()))
        checked += int(clear.sum())
    assert checked >= rows  # at least half of the rows of two layers


@pytest.mark.parametrize("name", ["tiny-moe", "tiny-gemma-moe"])
def test_speculation_changes_no_answer(cuda, name):
    prompts = [[5, 9, 100, 7, 3], [11, 12, 13], [1, 2, 3, 4, 5, 6, 7, 8, 9]]
    target = engine.QuantModel(PRESETS[name], cuda, seed=1, sigma=0.05, max_seqs=3, max_rows=32, max_logit_rows=32,
                               max_ctx=128)
    draft = engine.QuantModel(PRESETS["tiny-draft"], cuda, seed=2, max_seqs=3, max_ctx=128)
    plain = []
    for prompt in prompts:
        history = list(prompt)
        model = engine.QuantModel(PRESETS[name], cuda, seed=1, sigma=0.05, max_rows=32, max_ctx=128)
        logits = None
        for pos, tok in enumerate(history):
            logits = model.logits_for(torch.tensor([tok], dtype=torch.int32, device=cuda), pos)
        out = []
        while len(out) < 24:
            nxt = int(logits[0].float().argmax())
            out.append(nxt)
            logits = model.logits_for(torch.tensor([nxt], dtype=torch.int32, device=cuda), len(history) + len(out) - 1)
        plain.append(out)
    dec = engine.SpecDecoder(target, draft, k=4, batch=3)
    got = dec.generate(prompts, 24)
    assert [list(map(int, g))[:24] for g in got] == plain
    dec.capture()  # the round as one CUDA graph
    assert [list(map(int, g))[:24] for g in dec.generate(prompts, 24)] == plain


def test_every_draft_of_the_same_model_is_accepted(cuda):
    cfg = PRESETS["tiny-moe"]
    target, draft = (engine.QuantModel(cfg, cuda, seed=7, sigma=0.05, max_rows=32, max_logit_rows=32, max_ctx=128)
                     for _ in range(2))
    a = torch.tensor([3, 1, 4, 1, 5, 9], dtype=torch.int32, device=cuda)
    whole = target.logits_for(a, 0).clone()
    for i in range(a.numel()):
        assert torch.equal(draft.logits_for(a[i:i + 1], i)[0], whole[i])


def test_refusals(cuda, tmp_path):
    import dataclasses

    cfg = PRESETS["tiny-moe"]
    with pytest.raises(ValueError, match="one GPU"):
        engine.QuantModel(cfg, cuda, tp=2)
    with pytest.raises(ValueError, match="experts a token"):
        engine.QuantModel(dataclasses.replace(cfg, experts_per_token=9), cuda)
    with pytest.raises(checkpoint.CheckpointError, match="experts"):
        checkpoint.save_mlx_4bit(engine.QuantModel(cfg, cuda, max_ctx=32), tmp_path)

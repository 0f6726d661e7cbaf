"""The mixture-of-experts operators where they can go wrong at the edges of their ranges, against float64."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from ironmule_b200 import _lib, engine, kernels
from tests.test_moe_gpu import dense, mlp_case, quantised

pytestmark = pytest.mark.gpu


# ---- router ---------------------------------------------------------------------------------------------------
def softmax_over_chosen(logits, bias, top_k):
    """ids and weights in float64, the maximum taken over the chosen experts."""
    v = logits.float().cpu().numpy()
    order = np.argsort(-(v + bias.cpu().numpy()), axis=1, kind="stable")[:, :top_k]
    chosen = np.take_along_axis(v, order, 1).astype(np.float64)
    p = np.exp(chosen - chosen.max(axis=1, keepdims=True))
    return order, p / p.sum(axis=1, keepdims=True)


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_softmax_with_a_bias_that_passes_over_the_largest_logits(cuda, rows):
    """The chosen experts' logits lie 200 and more below the largest one: float32 exponentials taken relative to that
    one are all zero, relative to the largest chosen one they are not."""
    gen = torch.Generator(device=cuda).manual_seed(rows)
    logits = torch.randn((rows, 24), generator=gen, device=cuda)
    bias = torch.zeros(24, device=cuda)
    logits[:, :6] += 200.0 + 100.0 * torch.rand((rows, 1), generator=gen, device=cuda)
    bias[:6] = -10000.0
    r = kernels.moe_route(logits, 4, bias=bias)
    ids, want = softmax_over_chosen(logits, bias, 4)
    assert np.array_equal(r.ids.cpu().numpy(), ids)
    # float32: exponentials of 2 ulps, a sum of four, a quotient
    np.testing.assert_allclose(r.weights.cpu().numpy(), want, rtol=4e-6, atol=1e-30)
    one = kernels.moe_route(torch.tensor([[0.0, -200.0, -300.0]], device=cuda), 1,
                            bias=torch.tensor([-10000.0, 0.0, 0.0], device=cuda))
    assert one.ids.tolist() == [[1]] and one.weights.tolist() == [[1.0]]


@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
@pytest.mark.parametrize("rows,experts,top_k", [(1, 8, 2), (40, 60, 4), (300, 256, 8), (70, 500, 32)])
def test_a_bias_on_the_scores_chooses_by_score_plus_bias(cuda, scoring, rows, experts, top_k):
    gen = torch.Generator(device=cuda).manual_seed(rows + experts)
    logits = 2.0 * torch.randn((rows, experts), generator=gen, device=cuda)
    logits[torch.rand((rows, experts), generator=gen, device=cuda) < 0.1] = float("-inf")
    bias = (0.2 if scoring == "sigmoid" else 2.0 / experts) * torch.randn((experts,), generator=gen, device=cuda)
    for dtype in (torch.float32, torch.bfloat16):
        given = logits.to(dtype)
        r = kernels.moe_route(given, top_k, scoring=scoring, normalise=True, scale=2.5, bias=bias, bias_on="score")
        v = given.double()
        score = torch.sigmoid(v) if scoring == "sigmoid" else torch.softmax(v, 1)
        key = torch.where(v > float("-inf"), score + bias.double(), float("-inf"))
        order = torch.sort(key, dim=1, descending=True, stable=True)
        # float32 scores are off by some 2^-22 of themselves: rows with keys closer than that may go either way
        gap = (order.values[:, :top_k] - order.values[:, 1:top_k + 1]).amin(1)
        clear = gap > 2.0**-20
        assert int(clear.sum()) * 2 >= rows
        ids = order.indices[:, :top_k]
        assert torch.equal(r.ids[clear].long(), ids[clear])
        picked = torch.gather(score, 1, ids)
        want = 2.5 * picked / picked.sum(1, keepdim=True)
        assert bool(((r.weights.double() - want).abs()[clear] <= 4e-6 * want[clear]).all())
        flat = r.ids.flatten()
        assert torch.equal(r.pairs.long(), torch.sort(torch.where(flat < 0, experts, flat), stable=True).indices)


def test_where_the_bias_goes_decides(cuda):
    logits, bias = torch.tensor([[6.0, 5.0, 0.0]], device=cuda), torch.tensor([0.0, 0.1, 0.0], device=cuda)
    for dtype in (torch.float32, torch.bfloat16):
        on = lambda where: kernels.moe_route(logits.to(dtype), 1, scoring="sigmoid", normalise=False, bias=bias,  # noqa: E731
                                             bias_on=where)
        assert on("logit").ids.tolist() == [[0]] and on("score").ids.tolist() == [[1]]
        assert on("score").weights[0, 0].item() == pytest.approx(0.9933071490757153, rel=4e-6)
    closing = torch.tensor([0.0, float("-inf"), float("nan")], device=cuda)
    for scoring in ("sigmoid", "softmax"):
        r = kernels.moe_route(logits, 2, scoring=scoring, bias=closing, bias_on="score")
        assert r.ids.tolist() == [[0, -1]] and r.weights.tolist() == [[1.0, 0.0]]
    with pytest.raises(ValueError, match="bias_on"):
        kernels.moe_route(logits, 1, bias=bias, bias_on="probability")


# ---- status ---------------------------------------------------------------------------------------------------
def test_status_waits_for_the_products_stream(cuda):
    """On a stream of torch's pool, which the legacy default stream does not wait for: the error words are read after
    the work that is queued there (here a write of the word behind a delay)."""
    r = kernels.moe_route(torch.randn((4, 8), device=cuda), 2)
    ws = kernels.workspace(1 << 20, cuda)
    torch.cuda.synchronize()
    side = torch.cuda.Stream(cuda)
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)  # tens of milliseconds
        r.buf[r._plan_at + 1] = 1
        assert r.status() == 1
        torch.cuda._sleep(100_000_000)
        ws.fill_(1)
        assert kernels.qgemm_packed_status(ws) == 0x01010101


# ---- gated MLP -------------------------------------------------------------------------------------------------
def mlp_reference(x, gate, up, down, ex, act):
    """float64 outputs of one expert, and the bound on the kernel's error: weights as fp16 (2^-11 of each, and 2^-18 of
    its row's largest where a group is far below it), products and activations rounded to fp16 (2^-11), the gate's
    exponential, float32 sums, one rounding to bf16 (2^-8)."""
    def bound(q, xa):
        w, _ = dense(q, ex)
        return 2**-11 * (xa @ w.abs().T) + 2**-18 * xa.sum(1, keepdim=True) * w.abs().amax(1)

    xd = x.double()
    g, u = xd @ dense(gate, ex)[0].T, xd @ dense(up, ex)[0].T
    dg, du = bound(gate, xd.abs()), bound(up, xd.abs())
    a = g * torch.sigmoid(g) if act == "swiglu" else \
        0.5 * g * (1.0 + torch.tanh(0.7978845608028654 * (g + 0.044715 * g**3)))
    hid = a * u
    dh = 1.13 * dg * (u.abs() + du) + a.abs() * du + 2**-10 * hid.abs()
    w = dense(down, ex)[0]
    want = hid @ w.T
    return want, 2**-8 * want.abs() + dh @ w.abs().T + bound(down, hid.abs())


def check_mlp(x, gate, up, down, r, act="swiglu"):
    y = kernels.moe_mlp(x, kernels.Experts.gate_up(gate, up), kernels.Experts(*down), r, activation=act)
    ids = r.ids.long()
    for ex in range(gate[0].shape[0]):
        row, place = torch.nonzero(ids == ex, as_tuple=True)
        if row.numel():
            want, tol = mlp_reference(x[row], gate, up, down, ex, act)
            off = (y[row, place].double() - want).abs()
            assert bool((off <= tol).all()), (ex, float((off / tol).max()))
    return y


@pytest.mark.parametrize("act", ["swiglu", "geglu"])
@pytest.mark.parametrize("which", ["gate", "up"])
def test_an_expert_whose_gate_or_up_matrix_is_zero_gives_zeros(cuda, which, act):
    gate, up, down, x, logits = mlp_case(cuda, 40, 3, 2, 256, 128, 21)
    for t in (gate if which == "gate" else up)[1:]:
        t[0] = 0
    r = kernels.moe_route(logits, 2)
    for f in (1.0, 2.0**30, 2.0**-60):
        y = kernels.moe_mlp(x * f, kernels.Experts.gate_up(gate, up), kernels.Experts(*down), r, activation=act)
        assert bool((y[r.ids == 0] == 0).all()), f
        assert bool(torch.isfinite(y.float()).all())


@pytest.mark.parametrize("act", ["swiglu", "geglu"])
def test_tiny_gates_beside_large_up_projections(cuda, act):
    """g of about 2^-127, u of 2^48: their product is an ordinary number, u times its inverse is not."""
    gate, up, down, x, logits = mlp_case(cuda, 24, 4, 2, 256, 128, 22)
    for q, f in ((gate, 2.0**-115), (up, 2.0**60)):
        q[1].mul_(f)
        q[2].mul_(f)
    check_mlp(x * 2.0**-10, gate, up, down, kernels.moe_route(logits, 2), act)


def test_gate_up_of_an_odd_number_of_rows_is_refused(cuda):
    """Half of 129 rows is 64 too, but the packed matrices of 129 lie two blocks apart, not one."""
    gen = torch.Generator(device=cuda).manual_seed(0)
    r = kernels.moe_route(torch.randn((4, 8), device=cuda), 2)
    x = torch.zeros((4, 128), dtype=torch.bfloat16, device=cuda)
    with pytest.raises(ValueError, match="129 rows"):
        kernels.moe_mlp(x, kernels.Experts(*quantised(gen, 8, 129, 128, cuda)),
                        kernels.Experts(*quantised(gen, 8, 128, 64, cuda)), r)


def test_activations_keep_their_precision_beside_outliers(cuda):
    """A group of x a thousand times the others, which the weights leave out, and one large weight in the gate and the
    up matrix: neither may push the other rows' activations below fp16's range."""
    gate, up, down, x, logits = mlp_case(cuda, 40, 3, 2, 512, 128, 23)
    x[:, :64] *= 2.0**10
    for q in (gate, up):
        w, s, b = q
        s[:, :, 0], b[:, :, 0] = 0, 0
        w[:, 7, 8:16] = 0x88888888 - 2**32  # row 7, group 1: code 8 everywhere, worth zero
        w[:, 7, 8] = 0x8888888F - 2**32     # but 15 at one place, worth 7 scales
        s[:, 7, 1], b[:, 7, 1] = 0.25, -2.0
    check_mlp(x, gate, up, down, kernels.moe_route(logits, 2))


@pytest.mark.parametrize("f", [2.0**-40, 2.0**-6, 2.0**20])
def test_gated_mlp_of_small_and_large_rows(cuda, f):
    gate, up, down, x, logits = mlp_case(cuda, 24, 4, 2, 256, 128, 25)
    check_mlp(x * f, gate, up, down, kernels.moe_route(logits, 2))


@pytest.mark.parametrize("spread", [4, 10, 16])
def test_weight_rows_whose_groups_differ_widely(cuda, spread):
    """Scales of a row's groups spread over 2^spread: what a group far below the row's largest loses stays within 2^-18
    of that largest weight."""
    gate, up, down, x, logits = mlp_case(cuda, 24, 4, 2, 256, 128, 27)
    gen = torch.Generator(device=cuda).manual_seed(spread)
    for q in (gate, up, down):
        f = torch.exp2(-spread * torch.rand(q[1].shape, generator=gen, device=cuda)).to(torch.bfloat16)
        q[1].mul_(f)
        q[2].mul_(f)
    check_mlp(x, gate, up, down, kernels.moe_route(logits, 2))


@pytest.mark.parametrize("h,inter", [(64, 64), (2048, 192), (512, 1000 // 64 * 64)])
def test_gated_mlp_at_the_edge_of_its_bound(cuda, h, inter):
    """Every row of x, and every row of G and U, the same vector: g and u reach the bound that scales the activations,
    and must not overflow fp16 (with the largest value at the top of a power of two)."""
    v = 1.9375 * torch.ones((2, h), device=cuda).to(torch.bfloat16)
    ones = lambda n, k: (torch.full((2, n, k // 8), -1, dtype=torch.int32, device=cuda),  # noqa: E731
                         torch.full((2, n, k // 64), 0.125, dtype=torch.bfloat16, device=cuda),
                         torch.zeros((2, n, k // 64), dtype=torch.bfloat16, device=cuda))
    gate, up, down = ones(inter, h), ones(inter, h), ones(h, inter)
    check_mlp(v, gate, up, down, kernels.moe_route(torch.zeros((2, 2), device=cuda), 2))


# ---- bounded waits ----------------------------------------------------------------------------------------------
def test_a_wait_that_runs_out_sets_the_status_and_leaves_the_gpu_usable(cuda):
    """With no time beyond the first attempts, the one tile of a product over 2^20 inputs (milliseconds) outlasts its
    waits: the routing says so, the kernel ends, and the next product is right."""
    gen = torch.Generator(device=cuda).manual_seed(5)
    experts = kernels.Experts(*quantised(gen, 1, 64, 1 << 20, cuda))
    x = torch.randn((3, 1 << 20), generator=gen, device=cuda).to(torch.bfloat16)
    logits = torch.zeros((3, 1), device=cuda)
    r = kernels.moe_route(logits, 1)
    want = kernels.grouped_qgemm(x, experts, r)
    assert r.status() == 0
    was = kernels.set_wait_limit(0)
    try:
        assert was == 1_000_000_000 and kernels.set_wait_limit(-1) == 0
        kernels.grouped_qgemm(x, experts, r)
        assert r.status() == 1
    finally:
        kernels.set_wait_limit(was)
    again = kernels.moe_route(logits, 1)
    got = kernels.grouped_qgemm(x, experts, again)
    assert again.status() == 0 and torch.equal(got.view(torch.int16), want.view(torch.int16))
    gate, up, down, xs, scores = mlp_case(cuda, 160, 24, 4, 512, 320, 3)
    check_mlp(xs, gate, up, down, kernels.moe_route(scores, 4))


def test_a_callers_error_word_outlives_the_routing(cuda):
    gen = torch.Generator(device=cuda).manual_seed(6)
    experts = kernels.Experts(*quantised(gen, 1, 64, 1 << 20, cuda))
    x = torch.randn((1, 1 << 20), generator=gen, device=cuda).to(torch.bfloat16)
    logits, word = torch.zeros((1, 1), device=cuda), torch.zeros(1, dtype=torch.int32, device=cuda)
    kernels.grouped_qgemm(x, experts, kernels.moe_route(logits, 1, error=word))
    assert word.item() == 0
    was = kernels.set_wait_limit(0)
    try:
        kernels.grouped_qgemm(x, experts, kernels.moe_route(logits, 1, error=word))
    finally:
        kernels.set_wait_limit(was)
    r = kernels.moe_route(torch.zeros((100, 1), device=cuda), 1, error=word)
    assert r.status() == 0 and word.item() == 1
    with pytest.raises(ValueError, match="one element"):
        kernels.moe_route(logits, 1, error=torch.zeros(2, dtype=torch.int32, device=cuda))
    with pytest.raises(TypeError):
        kernels.moe_route(logits, 1, error=torch.zeros(1, device=cuda))


def test_the_engine_passes_its_error_word_and_raises_when_it_is_set(cuda, monkeypatch):
    cfg = engine.PRESETS["tiny-moe"]
    target = engine.QuantModel(cfg, cuda, seed=1, sigma=0.05, max_rows=32, max_logit_rows=32, max_ctx=128)
    draft = engine.QuantModel(engine.PRESETS["tiny-draft"], cuda, seed=2, max_ctx=128)
    words, mlp = [], kernels.moe_mlp

    def watched(x, gate_up, down, routing, **kw):
        words.append(routing.error)
        return mlp(x, gate_up, down, routing, **kw)

    monkeypatch.setattr(kernels, "moe_mlp", watched)
    dec = engine.SpecDecoder(target, draft, k=4, batch=1)
    prompt = [5, 9, 100, 7, 3]
    first = dec.generate([prompt], 8)
    assert len(words) >= cfg.layers and all(w is target.moe_error for w in words)
    dec.capture()
    assert dec.generate([prompt], 8) == first
    target.moe_error.fill_(1)  # what a product does whose wait runs out
    tokens = torch.tensor(prompt, dtype=torch.int32, device=cuda)
    engine_rows = [(t, i, 0, True) for i, t in enumerate(prompt)]
    for read in (lambda: dec.generate([prompt], 8), dec.done, dec.read_stats, lambda: dec.generated(0, 5),
                 lambda: engine.greedy_decode(target, tokens, 4),
                 lambda: engine.DeviceDraftEngine(target)._decode_conf(engine_rows)):
        with pytest.raises(_lib.KernelError, match="wait"):
            read()
    target.moe_error.zero_()
    assert dec.generate([prompt], 8) == first


@pytest.mark.parametrize("target,draft", [("tiny-moe", "tiny-draft"), ("tiny-gemma-moe", "tiny-moe"),
                                          ("tiny-target", "tiny-draft")])
@pytest.mark.parametrize("batch", [1, 14])
def test_launches_of_a_round_are_counted_with_experts(cuda, monkeypatch, target, draft, batch):
    models = [engine.QuantModel(engine.PRESETS[name], cuda, seed=i, sigma=0.05, max_seqs=batch, max_rows=80,
                                max_logit_rows=80, max_ctx=64) for i, name in enumerate((target, draft))]
    dec = engine.SpecDecoder(*models, k=4, batch=batch)
    seen, call = [], _lib.call

    def counted(name, *args):
        # products: the rows' layout and two products; a routing of more than 64 rows (argument 2): two launches
        seen.append(3 if name == "im_moe_mlp" else 2 if name == "im_moe_route_ex" and args[2] > 64 else 1)
        return call(name, *args)

    monkeypatch.setattr(_lib, "call", counted)
    dec.round()
    assert sum(seen) == dec.launches_per_round()

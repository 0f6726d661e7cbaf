"""The mixture-of-experts operators where they can go wrong at the edges of their ranges, against float64."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from ironmule_b200 import kernels

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

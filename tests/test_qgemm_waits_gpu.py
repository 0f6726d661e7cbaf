"""The packed qGEMM's tensor-core kernel when a bounded wait runs out."""
from __future__ import annotations

import pytest
import torch

from ironmule_b200 import kernels
from tests.test_moe_gpu import quantised

pytestmark = pytest.mark.gpu


def test_a_wait_that_runs_out_sets_the_status_and_leaves_the_gpu_usable(cuda):
    """With no time beyond the first attempts, the waits for the rows that a long layout kernel (2^20 inputs, 320 rows)
    still writes run out: the workspace says so, the kernel ends, and a product over a fresh workspace is right."""
    gen = torch.Generator(device=cuda).manual_seed(7)
    m, n, k = 320, 128, 1 << 20
    p = kernels.Packed(*(t[0] for t in quantised(gen, 1, n, k, cuda)))
    x = torch.randn((m, k), generator=gen, device=cuda).to(torch.bfloat16)
    kernels.qgemm_packed_path(2)
    try:
        need = kernels.qgemm_packed_workspace_bytes(m, n, k)
        ws = kernels.workspace(need, cuda)
        want = kernels.qgemm_packed(x, p, ws=ws)
        assert kernels.qgemm_packed_status(ws) == 0
        was = kernels.set_wait_limit(0)
        try:
            kernels.qgemm_packed(x, p, ws=ws)
            assert kernels.qgemm_packed_status(ws) == 1
        finally:
            kernels.set_wait_limit(was)
        ws.zero_()
        got = kernels.qgemm_packed(x, p, ws=ws)
        assert kernels.qgemm_packed_status(ws) == 0
        assert torch.equal(got.view(torch.int16), want.view(torch.int16))
    finally:
        kernels.qgemm_packed_path(0)

"""Calls from a host thread that has used no CUDA yet (as an autograd worker's first backward is)."""

from __future__ import annotations

import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_first_cuda_call_of_a_thread_may_be_a_tensor_map_kernel() -> None:
    from lsso_b200.ball.projection import weight_gradient
    from tests.gpu_util import require_native

    require_native()
    g = torch.randn(512, 64, device="cuda", dtype=torch.bfloat16)
    x = torch.randn(512, 72, device="cuda", dtype=torch.bfloat16)
    out = torch.empty(64, 72, device="cuda")
    want = weight_gradient(g, x, None)  # (also leaves the workspace in the allocator's cache)
    seen = []

    def call() -> None:
        try:
            seen.append(weight_gradient(g, x, None, out=out))
        except RuntimeError as error:
            seen.append(error)

    torch.cuda.synchronize()
    thread = threading.Thread(target=call)
    thread.start()
    thread.join()
    assert isinstance(seen[0], torch.Tensor), seen[0]
    torch.cuda.synchronize()
    assert torch.equal(seen[0], want)

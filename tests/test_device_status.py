"""The device status word: the gravest report since the last check stays."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _run_out_of_waiting() -> None:
    """Tensor-core kernels whose waits run out at once (status 1)."""
    from lsso_b200.ball import _native
    from lsso_b200.ball.feedforward import gated_feed_forward

    x = torch.randn(100, 256, device="cuda").bfloat16()
    w_in, w_out = torch.randn(512, 256, device="cuda").bfloat16(), torch.randn(256, 256, device="cuda").bfloat16()
    torch.cuda.synchronize()
    _native.set_wait_limit_ns(1)
    try:
        gated_feed_forward(x, w_in, w_out)
        torch.cuda.synchronize()
    finally:
        _native.set_wait_limit_ns(0)


def _look_up_outside(tokens: int, train: bool) -> None:
    """A lookup (and gradient) with an id outside the table (status 3)."""
    from lsso_b200.ball.embedding import token_embedding

    table = torch.randn(10, 16, device="cuda", requires_grad=train)
    ids = torch.zeros(tokens, dtype=torch.int64, device="cuda")
    ids[tokens // 2] = 10
    y = token_embedding(ids, table)
    if train:
        torch.autograd.grad(y.sum(), table)


@pytest.mark.parametrize("tokens", [5, 9000])  # sorted by one block, by several
@pytest.mark.parametrize("train", [False, True])
def test_an_id_outside_the_table_does_not_hide_undefined_outputs(tokens, train) -> None:
    from lsso_b200.ball import cuda
    from tests.gpu_util import require_native

    require_native()
    cuda.device_status(reset=True)
    _look_up_outside(tokens, train)
    assert cuda.device_status(reset=False) == 3
    _run_out_of_waiting()
    assert cuda.device_status(reset=False) == 1  # undefined outputs replace a zero row
    _look_up_outside(tokens, train)
    assert cuda.device_status(reset=False) == 1
    with pytest.raises(RuntimeError, match="gave up waiting"):
        cuda.check_device_status()
    assert cuda.device_status(reset=True) == 0

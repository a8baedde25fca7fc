"""Gradients of the causal mixer on the CUDA path, at inputs whose head outputs stay away from zero.

Behind a head output near zero the heads' norm multiplies every rounding, and two paths that round alike differ by their
draw alone.  Here query and key biases of one give every token a score of |q| |k| with itself, so that no head output is
below an eighth of the median.  The reference path under autocast rounds x, the projection, the rotary pairs, the heads, the norm and
the output, and their gradients: 12 roundings of u / sqrt 3 each.  The kernels add the decay attention's operands, 1.2 u
in place of u / sqrt 3 for y, dq, dk and dv: an error of at most ((12 / 3 + 4 (1.2^2 - 1 / 3)) / (12 / 3))^(1/2) = 1.5
times as large.  Twice the reference path's error is asked, at every seed.
"""

from __future__ import annotations

import pytest
import torch

from lsso import LSSOConfig
from lsso_b200.ball.causal import CausalMixer
from lsso_b200.ball.decay import decay_attention_reference
from lsso_b200.ball.rotary import rotary_reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize(("dim", "heads", "rank"), [(128, 4, 32), (256, 8, 32), (192, 3, 48)])
def test_errors_are_those_of_the_roundings(dim, heads, rank, dtype, seed) -> None:
    from tests.gpu_util import relative_l2, require_native

    require_native()
    torch.manual_seed(seed)
    mixer = CausalMixer(LSSOConfig(dim, heads, rank, bias=True)).cuda()
    with torch.no_grad():
        mixer.w_qkv.bias[:2 * heads * rank] = 1.0
    x = torch.randn(3, 300, dim, device="cuda").to(dtype)
    mask = torch.ones(3, 300, dtype=torch.bool, device="cuda")
    mask[1, 200:] = False
    mask[2, 100:150] = False
    up = torch.randn(3, 300, dim, device="cuda").to(dtype)

    def run(implementation, module, x, amp):
        x = x.clone().requires_grad_()
        with torch.autocast("cuda", dtype=amp or torch.bfloat16, enabled=amp is not None):
            y = module(x, mask, implementation=implementation)
        names, parameters = zip(*module.named_parameters())
        grads = torch.autograd.grad(y, (x, *parameters), up.to(y.dtype))
        return dict(zip(("y", "x", *names), (y.detach().double(), *(g.double() for g in grads))))

    got = run("cuda", mixer, x, dtype)
    # (the CUDA path's projections have BF16 multiplicands and outputs under FP16 autocast too)
    rounded = run("reference", mixer, x.bfloat16(), torch.bfloat16)
    exact = CausalMixer(mixer.config).cuda().double()
    exact.load_state_dict(mixer.state_dict())
    want = run("reference", exact, x.double(), None)
    with torch.no_grad():
        q, k, v = exact._split(exact.w_qkv(x.double()), rotary_reference, exact._positions(x, mask, None, None))
        sizes = decay_attention_reference(q, k, v, exact.log_decay, valid_mask=mask).square().mean(-1).sqrt()[mask]
    assert sizes.min() >= 0.125 * sizes.median()
    for name in want:
        assert relative_l2(got[name], want[name]) <= 2 * relative_l2(rounded[name], want[name]), name

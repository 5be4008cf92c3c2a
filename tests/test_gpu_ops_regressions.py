"""Faults that the operators once had: each test here failed before its fault was mended."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")


@pytest.mark.parametrize("how", ["plain", "int32 tokens", "transposed logits", "a slice of positions"])
def test_results_can_be_changed_in_place(how):
    """Log probabilities masked in place, as a loss over some positions does, whichever way the call
    takes; the entropy, saved for the backward pass, keeps its own storage and version."""
    _need_gpu()
    from luminamoon_amd import ops

    g = torch.Generator().manual_seed(0)
    z = torch.randn(3, 5, 40, generator=g).cuda()
    if how == "transposed logits":
        z = z.transpose(0, 1)
    elif how == "a slice of positions":
        z = z[:, :-1]
    tokens = torch.randint(0, 40, z.shape[:-1], generator=g).cuda()
    if how == "int32 tokens":
        tokens = tokens.int()
    mask = (torch.rand(z.shape[:-1], generator=g) < 0.5).float().cuda()
    z = z.detach().requires_grad_()
    scores = ops.token_log_probs(z, tokens)
    assert scores.log_probs._base is None and scores.entropy._base is None
    scores.log_probs.mul_(mask)
    (scores.log_probs - 0.1 * scores.entropy).sum().backward()
    got, z.grad = z.grad, None
    scores = ops.token_log_probs(z, tokens)
    (scores.log_probs * mask - 0.1 * scores.entropy).sum().backward()
    assert torch.equal(got, z.grad)

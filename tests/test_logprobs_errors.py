"""What token_logprobs says to logits that a program would train through; no GPU."""
import pytest
import torch

from tyloquant_amd import runtime as R


def test_gradients_are_refused():
    """scores have no backward pass: logits that a gradient is wanted of are refused, not detached without a word"""
    z, tokens = torch.zeros(3, 100, requires_grad=True), torch.zeros(3, dtype=torch.int64)
    for logits in (z, z * 2):
        with pytest.raises(RuntimeError, match="no backward pass"):
            R.token_logprobs(logits, tokens)
        with pytest.raises(ValueError, match="current GPU"):       # the next thing asked
            R.token_logprobs(logits.detach(), tokens)
    with torch.no_grad(), pytest.raises(ValueError, match="current GPU"):
        R.token_logprobs(z, tokens)
    with torch.inference_mode(), pytest.raises(ValueError, match="current GPU"):
        R.token_logprobs(z * 2, tokens)

"""FusedQwen2.score refuses a text longer than its cache, whose later tokens would be scored on a cut context (on the CPU: before
any GPU call)."""
import pytest
import torch

from lowbit import decode, fused


def test_score_refuses_a_text_longer_than_the_cache():
    model = fused.FusedQwen2(decode.random_model("tiny", device="cpu"), 8, "fp16")
    with pytest.raises(ValueError, match="9-token text does not fit a 8-token cache"):
        model.score(torch.zeros(9, dtype=torch.long))

"""verify_trees takes the greedy picks from the library's kernel: the first of equal logits, and no reduction of torch's."""
import pytest
import torch

from lowbit import decode, fused

pytestmark = pytest.mark.gpu


def test_picks_are_the_first_of_the_largest(cuda, monkeypatch):
    model = fused.FusedQwen2(decode.random_model("tiny", seed=15), 64, "fp16")
    # three rows of the head alike, so that their logits are: of the one that wins somewhere, of a later one and an earlier one
    i32 = dict(dtype=torch.int32, device="cuda")
    tokens = torch.tensor([5, 9, 700], device="cuda")
    run = lambda: model.verify_trees(tokens, torch.tensor([-1, 0, 1], **i32), torch.full((1, 2), -1, **i32),   # noqa: E731
                                     torch.zeros(1, **i32), torch.full((1,), 3, **i32), model.paged_caches(3, 16), 3, 32, 3)
    pick = int(run()[0][0, 0])
    assert 0 < pick < model.head.shape[0] - 1
    head = model.head.clone()
    head[pick - 1] = head[pick + 1] = head[pick]
    monkeypatch.setattr(model, "head", head)

    def other(*args, **kwargs):
        raise AssertionError("a reduction of torch's")

    for name in ("argmax", "max", "topk", "sort"):
        monkeypatch.setattr(torch.Tensor, name, other)
    accepted, counts, lens, missing = run()
    assert int(accepted[0, 0]) == pick - 1 and int(missing) == 0

"""Steps without tokens or without sequences, which forward_paged and the attention serve, through the plan and the acceptance too."""
import pytest
import torch

from lowbit import decode, fused, ops

pytestmark = pytest.mark.gpu

I32, I64 = dict(dtype=torch.int32, device="cuda"), dict(dtype=torch.int64, device="cuda")


@pytest.mark.parametrize("parents", [False, True])
@pytest.mark.parametrize("tokens", [0, 5])
def test_plan_of_no_sequences(cuda, tokens, parents):
    above = torch.zeros(tokens, **I32) if parents else None
    for table, rows in ((torch.zeros((0, 4), **I32), None), (torch.zeros((3, 4), **I32), torch.zeros(0, **I32))):
        step = ops.ext().plan_paged(table, torch.zeros(table.shape[0], **I32), torch.zeros(0, **I32), tokens, 9, 16, rows=rows,
                                    parents=above, words=2)
        assert step.page_table.shape == (0, 4) and step.kv_lens.shape == (0,) and step.copies.shape == (0, 2)
        assert step.q_starts.tolist() == [0] and step.missing.tolist() == [0]
        assert step.positions.tolist() == [0] * tokens and step.slots.tolist() == [-1] * tokens
        assert step.masks.tolist() == [[0, 0]] * tokens if parents else step.masks is None
        for got, dt in zip(step, (torch.int32,) * 3 + (torch.int64,) * 3 + (torch.int32,) * 2):
            assert got is None or (got.dtype is dt and got.is_cuda)
    with pytest.raises(RuntimeError, match="a row for every"):          # (rows of the table that nothing says of who keeps them)
        ops.ext().plan_paged(torch.zeros((3, 4), **I32), torch.zeros(3, **I32), torch.zeros(0, **I32), tokens, 9, 16)


def test_acceptance_of_no_drafts(cuda):
    for tokens, keys in ((0, [7, 0, 33]), (0, []), (4, [])):
        t, kv, starts = torch.zeros(tokens, **I64), torch.tensor(keys, **I32), torch.zeros(len(keys) + 1, **I32)
        for slots in (None, torch.zeros(tokens, **I64)):
            path, counts, accepted, lens = ops.ext().accept_drafts(t, t, None, starts, kv, torch.zeros((len(keys), 3), **I32), None, 5,
                                                                   slots=slots)
            assert path.tolist() == accepted.tolist() == [[-1] * 5] * len(keys)
            assert path.shape == accepted.shape == (len(keys), 5) and path.dtype is torch.int32 and accepted.dtype is torch.int64
            assert counts.tolist() == [0] * len(keys) and lens.tolist() == keys
            assert counts.dtype is lens.dtype is torch.int32 and lens.data_ptr() != kv.data_ptr() or not keys


def test_verify_trees_of_nothing(cuda):
    """No tokens beside two sequences, which keep what they have; padded tokens alone."""
    model = fused.FusedQwen2(decode.random_model("tiny", seed=13), 64, "fp16")
    caches = model.paged_caches(6, 16)
    for tokens, keys in ((0, [20, 3]), (3, [])):
        table = torch.arange(2 * len(keys), **I32).view(len(keys), 2)
        want = table.clone()
        accepted, counts, lens, missing = model.verify_trees(
            torch.zeros(tokens, **I64), torch.zeros(tokens, **I32), table, torch.tensor(keys, **I32), torch.zeros(len(keys), **I32),
            caches, 8, 32, 4)
        assert accepted.tolist() == [[-1] * 4] * len(keys) and counts.tolist() == [0] * len(keys)
        assert lens.tolist() == keys and int(missing) == 0 and torch.equal(table, want)
    assert not caches[0].any() and not caches[1].any()

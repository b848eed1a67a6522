"""accept_drafts of nodes that have no slot in the cache, or a negative token, against the sequential restatement."""
import random

import pytest
import torch

from lowbit import ops

from test_gpu_accept_drafts import i32, i64, make, oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("by_slots", [True, False])
@pytest.mark.parametrize("chain", [False, True])
def test_nodes_without_a_place_are_not_confirmed(cuda, by_slots, chain):
    rng = random.Random(7)
    for sizes in ([1], [26], [5, 0, 70, 1, 33], [300, 129]):
        for share in (0.02, 0.3, 1.0):
            print(sizes, share, flush=True)
            ps, longest, layers = 16, 40, 2
            pasts = [rng.randrange(60) for _ in sizes]
            tokens, picks, parents, table, pages = make(rng, sizes, pasts, ps, chain=chain, vocab=2)
            gone = [rng.random() < share for _ in tokens]
            starts = [sum(sizes[:b]) for b in range(len(sizes) + 1)]
            none = [n > 0 and gone[starts[b]] for b, n in enumerate(sizes)]
            # (a sequence without node 0 as one whose drafts are all gone, less its node 0)
            for b, n in enumerate(sizes):
                if none[b]:
                    gone[starts[b]:starts[b + 1]] = [True] * n
            left = [-1 if g else t for g, t in zip(gone, tokens)]
            caches = tuple(torch.randn(layers, pages, 2, ps, 64, device="cuda").half() for _ in range(2))
            path, counts, accepted, lens, moved = oracle(left, picks, parents, sizes, pasts, table, ps, caches, longest, pages)
            for b in range(len(sizes)):
                if none[b]:
                    path[b], accepted[b] = -1, -1
                    counts[b] -= 1
                    lens[b] -= 1
            slots = [-1 if g else rng.randrange(pages * ps) for g in gone]
            given = i64(tokens if by_slots else left)
            got = ops.ext().accept_drafts(given, i64(picks), None if chain else i32(parents), i32(starts),
                                          i32([p + n for p, n in zip(pasts, sizes)]), i32(table), caches, longest,
                                          slots=i64(slots) if by_slots else None)
            for a, b in zip(got, (path, counts, accepted, lens)):
                assert torch.equal(a, b)
            assert torch.equal(caches[0], moved[0]) and torch.equal(caches[1], moved[1])
            if by_slots:
                assert given.tolist() == tokens


def test_picks_below_zero_confirm_nothing(cuda):
    """A negative pick is no token, so a draft with the same negative number does not follow it."""
    got = ops.ext().accept_drafts(i64([3, -1, 4]), i64([-1, 4, 9]), None, i32([0, 3]), i32([8]), i32([[0]]), None, 3)
    assert [g.tolist() for g in got] == [[[0, -1, -1]], [1], [[-1, -1, -1]], [6]]


def test_slots_that_do_not_fit_are_refused(cuda):
    args = (i64([3, 1]), i64([1, 4]), None, i32([0, 2]), i32([2]), i32([[0]]), None, 3)
    for slots in (i64([0]), i32([0, 1]), torch.zeros(2, dtype=torch.int64)):
        with pytest.raises(RuntimeError, match="slots"):
            ops.ext().accept_drafts(*args, slots=slots)

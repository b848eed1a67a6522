"""plan_paged where more than 1024 sequences, whose state lies in the workspace, share pages that several of them would write: against
the sequential restatement of its rules, so every value has to be equal."""
import random

import pytest

from test_gpu_plan_paged import check

pytestmark = pytest.mark.gpu


def shared(rng, count, groups, ps):
    """`count` sequences, most of them in `groups` spread over all numbers, each on one partly filled page: at lengths that many
    of the group have, among them sequences that pause, with a page before it or none."""
    table, past, new, at = [None] * count, [0] * count, [0] * count, 0
    order = list(range(count))
    rng.shuffle(order)
    step = count // (groups + 1)
    for g in range(groups + 1):
        mine = order[g * step:(g + 1) * step] if g < groups else order[groups * step:]
        before, page = at, at + 1
        at += 2
        for b in mine:
            if g == groups:                                  # pages of their own, or no keys
                past[b] = rng.choice([0, rng.randrange(1, ps), ps])
                page, at = at, at + 1
            else:
                past[b] = (ps if g % 2 else 0) + rng.randrange(1, ps)
            new[b] = rng.choice([0, 1, 1, 3, ps + 2])
            table[b] = ([before, page] if past[b] > ps else [page, -5]) + [-5, -5]
            if past[b] == 0:
                table[b][0] = -5
    pages = at + sum(n // ps + 3 for n in new)
    names = list(range(pages))
    rng.shuffle(names)
    return [[names[p] if p >= 0 else p for p in r] for r in table], past, new, pages


@pytest.mark.parametrize("count,groups", [(1025, 1), (1400, 3), (2300, 7)])
def test_one_page_of_many_sequences(cuda, count, groups):
    """Of the hundreds on a page, the one with the most keys, or of several the first that writes, keeps it, whichever workgroup's
    waves come first: again and again the same tables."""
    rng = random.Random(count)
    table, past, new, pages = shared(rng, count, groups, 16)
    print(count, groups, sum(new), pages, flush=True)
    for _ in range(3):
        check(table, past, new, sum(new) + 3, pages, 16, wide=False)

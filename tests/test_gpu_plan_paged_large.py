"""plan_paged beyond 8192 tokens, whose tables and tokens are a launch of their own, and beyond 1024 sequences, whose hash of shared pages
lies in the workspace: rows, trees of several words, copies and replayed graphs, against the sequential restatement of its rules."""
import random

import pytest
import torch

from lowbit import ops

from test_gpu_plan_paged import NAMES, check, i32, make, oracle
from test_gpu_plan_paged_shared import shared

pytestmark = pytest.mark.gpu


def trees(rng, sizes):
    return [rng.choice([i - 1, rng.randrange(max(i, 1)), -1 if i % 7 == 0 else i - 1]) for n in sizes for i in range(n)]


@pytest.mark.parametrize("count,held,most_new", [(300, 80, 60), (1100, 300, 12), (1500, 1500, 3)])
def test_rows(cuda, count, held, most_new):
    """Sequences that go on from rows, many from the same one and some from none."""
    rng = random.Random(count)
    table, past, _, _ = make(rng, 1, 90, 16, rows=held)
    new = [rng.randrange(most_new + 1) for _ in range(count)]
    new[0] += max(0, 8200 - sum(new)) if count == 300 else 0
    width = len(table[0]) + new[0] // 16 + 1
    table = [r + [-3] * (width - len(r)) for r in table]
    rows = [rng.choice([rng.randrange(held), rng.randrange(held // 4), -1, held]) for _ in range(count)]
    pages = max(max(r) for r in table) + 1 + 2 * count + sum(new) // 16
    print(count, held, sum(new), flush=True)
    check(table, past, new, sum(new) + 5, pages, 16, rows=rows, wide=False)
    check(table, past, new, sum(new) + 5, pages, 16, rows=rows, parents=trees(rng, new) + [0] * 5, words=2, wide=False)


@pytest.mark.parametrize("count,words,most", [(100, 3, 180), (1100, 1, 14), (1030, 5, 320)])
def test_trees(cuda, count, words, most):
    rng = random.Random(count)
    table, past, _, pages = make(rng, count, 60, 16, share=0.3)
    sizes = [rng.choice([0, 1, 1, 2, 5]) for _ in range(count)]
    for b in rng.sample(range(count), min(count, 40) if most > 20 else count):
        sizes[b] = rng.randrange(most + 1)
    sizes[3] = most
    if count == 100:                                         # (a launch of their own for the tokens)
        sizes[7:20] = [600] * 13
    width = max(-(-(p + n) // 16) for p, n in zip(past, sizes)) + 1
    table = [r[:width] + [-3] * (width - len(r)) for r in table]
    print(count, sum(sizes), flush=True)
    assert count > 1024 or sum(sizes) > 8192
    check(table, past, sizes, sum(sizes) + 2, pages + sum(sizes) // 16 + count, 16, parents=trees(rng, sizes) + [0, 0], words=words,
          wide=False)


def test_copies(cuda):
    """More than 1024 sequences, most of them on pages that others would write: the filled rows reach the copies in every layer."""
    rng = random.Random(4)
    table, past, new, pages = shared(rng, 1200, 5, 16)
    caches = tuple(torch.randn(3, pages, 2, 16, 8, device="cuda").half() for _ in range(2))
    want, res = tuple(c.clone() for c in caches), oracle(table, past, list(new), sum(new), pages, 16)
    for b, (src, dst) in enumerate(res[6].tolist()):
        if dst >= 0:
            for c in want:
                c[:, dst, :, :past[b] % 16] = c[:, src, :, :past[b] % 16]
    got = ops.ext().plan_paged(i32(table), i32(past), i32(new), sum(new), pages, 16, caches=caches)
    for name, a, b in zip(NAMES, got, res):
        assert (a is None and b is None) or torch.equal(a, b), name
    assert torch.equal(caches[0], want[0]) and torch.equal(caches[1], want[1])


@pytest.mark.parametrize("count,most_new,by_rows", [(60, 300, False), (60, 300, True), (1100, 6, False), (1100, 6, True)])
def test_replayed(cuda, count, most_new, by_rows):
    """Captured once, replayed with other lengths, rows and trees between eager calls."""
    rng = random.Random(count + by_rows)
    held, words, batches = 50 if by_rows else count, 5, []
    for _ in range(3):
        table, past, _, pages = make(rng, count, 200, 16, share=0.4, rows=held if by_rows else None)
        new = [rng.randrange(most_new + 1) for _ in range(count)]
        rows = [rng.randrange(-1, held) for _ in range(count)] if by_rows else None
        batches.append((table, past, new, rows, trees(rng, new), pages + 2 * count + sum(new) // 16))
    tokens, pages = max(max(sum(b[2]) for b in batches) + 7, 8200), max(b[5] for b in batches)
    width = max(len(b[0][0]) for b in batches) + most_new // 16 + 2
    table, past = torch.full((held, width), -1, dtype=torch.int32, device="cuda"), i32([0] * held)
    new, parents = i32([0] * count), i32([-1] * tokens)
    rows = i32([-1] * count) if by_rows else None
    run = lambda: ops.ext().plan_paged(table, past, new, tokens, pages, 16, rows=rows, parents=parents, words=words)   # noqa: E731

    def load(i):
        t, p, n, r, above, _ = batches[i]
        above, t = above + [-1] * (tokens - len(above)), [x + [-1] * (width - len(x)) for x in t]
        table.copy_(i32(t))
        past.copy_(i32(p))
        new.copy_(i32(n))
        parents.copy_(i32(above))
        if by_rows:
            rows.copy_(i32(r))
        return oracle(t, p, list(n), tokens, pages, 16, r, above, words)

    load(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step = run()
    for i in (1, 2, 0, 1):
        want = load(i)
        graph.replay()
        eager = run()
        torch.cuda.synchronize()
        for name, a, b, c in zip(NAMES, step, eager, want):
            assert torch.equal(a, c) and torch.equal(b, c), (name, i)

"""accept_drafts on the GPU against a sequential restatement: paths, counts and tokens are whole numbers and the moved rows copies, so
everything has to be equal."""
import random

import pytest
import torch

from lowbit import ops

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def i64(x):
    return torch.tensor(x, dtype=torch.int64, device="cuda")


def make(rng, sizes, pasts, ps, pages_spare=2, chain=False, vocab=3):
    """Trees over a small vocabulary (so that siblings share tokens and picks hit often) on pages in no order."""
    tokens, picks, parents = [], [], []
    for n in sizes:
        for i in range(n):
            parents.append(i - 1 if chain or i == 0 else rng.choice([i - 1, rng.randrange(i)]))
            tokens.append(rng.randrange(vocab))
            picks.append(rng.randrange(vocab))
    need = [-(-(p + n) // ps) for p, n in zip(pasts, sizes)]
    order = list(range(sum(need) + pages_spare))
    rng.shuffle(order)
    width, at, table = max(need) + 1, 0, []
    for k in need:
        table.append(order[at:at + k] + [-1] * (width - k))
        at += k
    return tokens, picks, parents, table, len(order)


def oracle(tokens, picks, parents, sizes, pasts, table, ps, caches, longest, pages):
    paths, counts, accepted, lens, first = [], [], [], [], 0
    want = tuple(c.clone() for c in caches)
    for b, n in enumerate(sizes):
        path = [0] if n else []
        while path and len(path) < longest:
            below = [c for c in range(path[-1] + 1, n) if parents[first + c] == path[-1] and tokens[first + c] == picks[first + path[-1]]]
            if not below:
                break
            path.append(below[0])

        def place(key):
            ok = 0 <= key < len(table[b]) * ps and 0 <= table[b][key // ps] < pages
            return (table[b][key // ps], key % ps) if ok else None

        moves = [(place(pasts[b] + c), place(pasts[b] + d)) for d, c in enumerate(path) if c != d]
        for c, w in zip(caches, want):
            for src, dst in moves:
                if src and dst:
                    w[:, dst[0], :, dst[1]] = c[:, src[0], :, src[1]]   # (from the caches as they were)
        said = [picks[first + c] for c in path]
        pad = [-1] * (longest - len(path))
        paths.append(path + pad)
        accepted.append(said + pad)
        counts.append(len(path))
        lens.append(pasts[b] + len(path))
        first += n
    return i32(paths), i32(counts), i64(accepted), i32(lens), want


def check(rng, sizes, pasts, ps, hkv, d, layers, dt, longest, chain=False, vocab=3, spoil=None):
    tokens, picks, parents, table, pages = make(rng, sizes, pasts, ps, chain=chain, vocab=vocab)
    if spoil:
        spoil(table, parents)
    caches = tuple(torch.randn(layers, pages, hkv, ps, d, device="cuda").to(dt) for _ in range(2))
    starts = [0]
    for n in sizes:
        starts.append(starts[-1] + n)
    want = oracle(tokens, picks, parents, sizes, pasts, table, ps, caches, longest, pages)
    args = (i64(tokens), i64(picks), None if chain else i32(parents), i32(starts), i32([p + n for p, n in zip(pasts, sizes)]), i32(table))
    loose = ops.ext().accept_drafts(*args, None, longest)
    got = ops.ext().accept_drafts(*args, caches, longest)
    for a, b, c in zip(got, loose, want):
        assert a.shape == c.shape and a.dtype == c.dtype and torch.equal(a, c) and torch.equal(b, c)
    assert torch.equal(caches[0], want[4][0]) and torch.equal(caches[1], want[4][1])
    return want


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hkv,d,ps", [(2, 128, 64), (8, 64, 16), (1, 128, 16), (32, 128, 16), (3, 8, 32)])
def test_trees(cuda, hkv, d, ps, dt):
    rng = random.Random(hkv * d + ps)
    for sizes in ([1], [26], [2, 0, 64, 63], [5, 17, 40, 1, 33, 9, 64]):
        pasts = [rng.choice([0, 1, ps - 1, ps, rng.randrange(200)]) for _ in sizes]
        for longest in (1, 3, 9, 64):
            print(sizes, longest, flush=True)
            check(rng, sizes, pasts, ps, hkv, d, 2, dt, longest, vocab=rng.choice([1, 2, 3]))


def test_large_trees_and_long_paths(cuda):
    """More nodes than a wave has lanes, paths of more rows than a workgroup holds at once: a vocabulary of one token confirms the
    first child everywhere."""
    rng = random.Random(3)
    for sizes in ([65], [300, 129], [1024]):
        for vocab in (1, 2):
            check(rng, sizes, [rng.randrange(60) for _ in sizes], 16, 2, 128, 1, torch.float16, 1024, vocab=vocab)
    # a long path that skips every other node, so that every row moves
    n = 1000
    tokens, picks = [7] * n, [7] * n
    parents = [-1] + [i - 2 if i % 2 == 0 else 0 for i in range(1, n)]
    tokens = [7 if i % 2 == 0 else 8 for i in range(n)]
    past, ps, pages = 21, 16, 70
    table = list(range(pages))
    rng.shuffle(table)
    caches = tuple(torch.randn(2, pages, 3, ps, 128, device="cuda").half() for _ in range(2))
    want = oracle(tokens, picks, parents, [n], [past], [table], ps, caches, 1024, pages)
    got = ops.ext().accept_drafts(i64(tokens), i64(picks), i32(parents), i32([0, n]), i32([past + n]), i32([table]), caches, 1024)
    assert int(got[1]) == 500
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert torch.equal(caches[0], want[4][0]) and torch.equal(caches[1], want[4][1])


def test_chains(cuda):
    rng = random.Random(5)
    for sizes in ([1], [5], [4, 0, 9], [70, 2]):
        check(rng, sizes, [rng.randrange(50) for _ in sizes], 16, 2, 64, 2, torch.float16, 80, chain=True, vocab=2)


def test_what_the_caller_gets_wrong(cuda):
    """Pages outside the cache (their rows stay), parents that are no earlier nodes, fewer keys than new tokens."""
    rng = random.Random(6)

    def pages(table, parents):
        for r in table:
            r[1] = rng.choice([-1, 1 << 30, -(1 << 31)])

    def loops(table, parents):
        for i in range(1, len(parents), 4):
            parents[i] = rng.choice([i, 1 << 30, -(1 << 31), 63])

    for spoil in (pages, loops):
        check(rng, [40, 33], [10, 3], 16, 2, 128, 2, torch.float16, 20, vocab=2, spoil=spoil)
    check(rng, [30], [-12], 16, 2, 128, 2, torch.float16, 20, vocab=1)   # (kv_lens below the new tokens: keys below 0 are nowhere)


def test_captured(cuda):
    rng = random.Random(9)
    ps, layers, sizes = 16, 3, [20, 33]
    batches = []
    for i in range(3):
        pasts = [rng.randrange(100) for _ in sizes]
        batches.append((pasts,) + make(rng, sizes, pasts, ps))
    width, pages = max(len(b[4][0]) for b in batches), max(b[5] for b in batches)
    t, p, q = i64([0] * 53), i64([0] * 53), i32([0] * 53)
    starts, kv = i32([0, 20, 53]), i32([0, 0])
    table = torch.full((2, width), -1, dtype=torch.int32, device="cuda")
    caches = tuple(torch.zeros(layers, pages, 2, ps, 128, dtype=torch.float16, device="cuda") for _ in range(2))
    run = lambda: ops.ext().accept_drafts(t, p, q, starts, kv, table, caches, 12)          # noqa: E731

    def load(i):
        pasts, tokens, picks, parents, rows, _ = batches[i]
        t.copy_(i64(tokens))
        p.copy_(i64(picks))
        q.copy_(i32(parents))
        kv.copy_(i32([a + n for a, n in zip(pasts, sizes)]))
        table.fill_(-1)
        table[:, :len(rows[0])] = i32(rows)
        for c in caches:
            c.normal_()
        full = [r + [-1] * (width - len(r)) for r in rows]
        return oracle(tokens, picks, parents, sizes, pasts, full, ps, caches, 12, pages)

    load(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = run()
    for i in (1, 2, 0, 1):
        want = load(i)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        assert torch.equal(caches[0], want[4][0]) and torch.equal(caches[1], want[4][1])


def test_nodes_past_the_masks_are_not_confirmed(cuda):
    """A child that is the 1024th node or an earlier one is, a later one, which no mask has room for, is not."""
    n, past = 1200, 3
    for child, count in ((1023, 2), (1024, 1), (1199, 1)):
        tokens, parents = [5] * n, [-1] * n
        tokens[child], parents[child] = 6, 0
        path, counts, accepted, lens = ops.ext().accept_drafts(
            i64(tokens), i64([6] * n), i32(parents), i32([0, n]), i32([past + n]), i32([list(range(80))]), None, 4)
        assert counts.tolist() == [count] and lens.tolist() == [past + count]
        assert path.tolist() == [([0, child] if count == 2 else [0]) + [-1] * (4 - count)]
        assert accepted.tolist() == [[6] * count + [-1] * (4 - count)]

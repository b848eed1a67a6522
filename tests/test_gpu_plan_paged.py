"""plan_paged on the GPU against a sequential restatement of its rules: tables, starts, positions, slots, masks and copies are whole
numbers, so every value has to be equal. Each case runs as given and as a call too large for one workgroup (a wide table)."""
import random

import pytest
import torch

from lowbit import ops

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def oracle(table, past, new, tokens, pages, ps, rows=None, parents=None, words=1, in_place=False):
    """The rules, one sequence after another, on lists."""
    width, count = len(table[0]), len(new)
    own_rows = rows is not None
    rows = list(range(count)) if rows is None else rows
    past = [min(max(past[r], 0), width * ps) if 0 <= r < len(table) else 0 for r in rows]
    new, left, starts = [min(max(n, 0), tokens) for n in new], tokens, [0]
    for b in range(count):
        new[b] = min(new[b], left)
        left -= new[b]
        starts.append(starts[-1] + new[b])
    kept = [table[r][:-(-past[b] // ps)] if past[b] else [] for b, r in enumerate(rows)]
    used = {p for k in kept for p in k if 0 <= p < pages}
    whole = {p for b, k in enumerate(kept) for p in k[:past[b] // ps]}
    free = [p for p in range(pages) if p not in used]
    handed, missing, copies, out = 0, 0, [], []

    def take():
        nonlocal handed, missing
        handed += 1
        if handed <= len(free):
            return free[handed - 1]
        missing += 1
        return -1

    for b in range(count):
        k, pair = list(kept[b]), [-1, -1]
        if past[b] % ps and new[b] and 0 <= k[-1] < pages:
            better = [c for c in range(count) if c != b and past[c] % ps and kept[c][-1] == k[-1]
                      and (past[c] > past[b] or (past[c] == past[b] and c < b and new[c]))]
            if k[-1] in whole or better:
                pair = [k[-1], take()]
                k[-1] = pair[1]
        copies.append(pair)
        need = -(-(past[b] + new[b]) // ps)
        while len(k) < min(need, width):
            k.append(take())
        missing += max(0, need - max(width, len(kept[b])))
        behind = table[rows[b]][len(k):] if in_place else [-1] * (width - len(k))
        out.append(k + behind)
    positions, slots, masks = [], [], []
    for b in range(count):
        bits, depth = [], []
        for i in range(new[b]):
            key = past[b] + i
            page = out[b][key // ps] if key // ps < width else -1
            slots.append(page * ps + key % ps if 0 <= page < pages else -1)
            if parents is None:
                positions.append(key)
                continue
            p = parents[starts[b] + i]
            up = 0 <= p < i
            bits.append((1 << i if i < 64 * words else 0) | (bits[p] if up else 0))
            depth.append(depth[p] + 1 if up else 0)
            positions.append(past[b] + depth[i])
        masks += bits
    pad = tokens - len(slots)
    result = [i32(out), i32(starts), i32([p + n for p, n in zip(past, new)]),
              torch.tensor(positions + [0] * pad, dtype=torch.int64, device="cuda"),
              torch.tensor(slots + [-1] * pad, dtype=torch.int64, device="cuda"), None, i32(copies).view(-1, 2), i32([missing])]
    if parents is not None:
        split = [[(m >> 64 * w) & (2 ** 64 - 1) for w in range(words)] for m in masks] + [[0] * words] * pad
        result[5] = torch.tensor([[x - 2 ** 64 if x >> 63 else x for x in r] for r in split], dtype=torch.int64,
                                 device="cuda").view(tokens, words)
    return result


NAMES = ("page_table", "q_starts", "kv_lens", "positions", "slots", "masks", "copies", "missing")


def check(table, past, new, tokens, pages, ps, rows=None, parents=None, words=1, wide=True):
    for width in (len(table[0]), (1 << 16) + 3) if wide else (len(table[0]),):      # (the second: four launches)
        t = [r + [-7] * (width - len(table[0])) for r in table]
        want = oracle(t, past, list(new), tokens, pages, ps, rows, parents, words)
        args = (i32(t), i32(past), i32(new), tokens, pages, ps)
        more = dict(rows=None if rows is None else i32(rows), parents=None if parents is None else i32(parents), words=words)
        got = ops.ext().plan_paged(*args, **more)
        for name, a, b in zip(NAMES, got, want):
            if b is None:
                assert a is None
                continue
            assert a.shape == b.shape and a.dtype == b.dtype, (name, a.shape, b.shape)
            assert torch.equal(a, b), (name, width, (a != b).nonzero()[:4].tolist(), a[a != b][:4].tolist(), b[a != b][:4].tolist())
        if rows is None:                                     # into the table itself
            want = oracle(t, past, list(new), tokens, pages, ps, rows, parents, words, in_place=True)
            given = args[0]
            got = ops.ext().plan_paged(*args, **more, out=given)
            assert got.page_table.data_ptr() == given.data_ptr()
            for name, a, b in zip(NAMES, got, want):
                assert (a is None and b is None) or torch.equal(a, b), (name, width, "in place")


def make(rng, count, most, ps, spare=3, share=0.0, rows=None):
    """A table of `rows` (or count) rows on up to `most` keys, some of them sharing pages of earlier rows; new tokens."""
    held = rows or count
    past = [rng.choice([0, 1, ps - 1, ps, ps + 1, rng.randrange(most + 1), rng.randrange(most + 1)]) for _ in range(held)]
    past = [min(p, most) for p in past]
    new = [rng.choice([0, 1, 1, 2, rng.randrange(3 * ps)]) for _ in range(count)]
    width = max(-(-(p + max(new)) // ps) for p in past) + rng.randrange(3)
    width = max(width, 1)
    at, table = 0, []
    for b in range(held):
        k = -(-past[b] // ps)
        row = []
        if b and rng.random() < share:
            other = rng.randrange(b)
            row = table[other][:min(k, -(-past[other] // ps), rng.randrange(width + 1))]
        while len(row) < k:
            row.append(at)
            at += 1
        table.append(row + [-9] * (width - len(row)))
    pages = at + -(-sum(new) // ps) + 2 * count + spare
    order = list(range(pages))
    rng.shuffle(order)
    return [[order[p] if p >= 0 else p for p in r] for r in table], past, new, pages


@pytest.mark.parametrize("ps", [16, 64, 1024])
def test_lengths(cuda, ps):
    rng = random.Random(ps)
    for count, most in ((1, 0), (1, 5 * ps), (2, 3 * ps), (7, 4 * ps), (33, 9 * ps), (65, 2 * ps), (200, 6 * ps)):
        table, past, new, pages = make(rng, count, most, ps)
        print(count, most, flush=True)
        check(table, past, new, sum(new) + rng.choice([0, 1, 70]), pages, ps, wide=count < 40)


@pytest.mark.parametrize("share", [0.3, 0.9])
def test_shared_pages(cuda, share):
    """Rows that go on with pages of other rows, at the same and at other lengths."""
    rng = random.Random(int(100 * share))
    for count, most in ((2, 20), (3, 60), (9, 100), (40, 64), (130, 200)):
        for _ in range(3):
            table, past, new, pages = make(rng, count, most, 16, share=share)
            print(count, most, flush=True)
            check(table, past, new, sum(new), pages, 16, wide=count < 10)


def test_rows(cuda):
    """Sequences that go on from rows of the table, some from the same one, some from none."""
    rng = random.Random(8)
    for count, held in ((1, 1), (4, 1), (8, 8), (16, 5), (64, 64), (128, 16)):
        for _ in range(3):
            table, past, new, pages = make(rng, count, 90, 16, share=0.2, rows=held, spare=4 * count + 20)
            rows = [rng.choice([rng.randrange(held), rng.randrange(held), -1, held, 1 << 30, -(1 << 31)]) for _ in range(count)]
            print(count, held, flush=True)
            check(table, past, new, sum(new) + 2, pages, 16, rows=rows, wide=count < 20)
            check(table, past, [1] * count, count, pages, 16, rows=rows, wide=False)
            check(table, past, [0] * count, 0, pages, 16, rows=rows, wide=False)


def test_trees(cuda):
    rng = random.Random(4)
    for words, sizes in ((1, [26]), (1, [1, 64, 3, 0, 17]), (2, [65, 2, 128]), (16, [1024, 5, 700]), (1, [100])):
        past = [rng.randrange(100) for _ in sizes]
        parents = []
        for n in sizes:
            parents += [rng.choice([i - 1, rng.randrange(i) if i else -1, rng.randrange(max(i, 1))]) for i in range(n)]
        for bad in (False, True):
            if bad:                                          # not earlier nodes: roots
                for i in range(0, len(parents), 5):
                    parents[i] = rng.choice([-1, -(1 << 31), 1 << 30, 1023])
            width = max(-(-(p + n) // 16) for p, n in zip(past, sizes)) + 1
            at, table = 0, []
            for p in past:
                k = -(-p // 16)
                table.append(list(range(at, at + k)) + [-1] * (width - k))
                at += k
            tokens = sum(sizes) + 5
            print(words, sizes, bad, flush=True)
            check(table, past, sizes, tokens, at + 300, 16, parents=parents + [0] * 5, words=words)


def test_pages_that_run_out(cuda):
    """Too few free pages: the first sequences get them, the others' entries and slots are -1, and the call says how many."""
    rng = random.Random(2)
    for count in (1, 5, 50):
        table, past, new, pages = make(rng, count, 70, 16, share=0.5)
        used = {p for b in range(count) for p in table[b][:-(-past[b] // 16)]}
        keep = sorted(used)
        for spare in (0, 1, 3):
            names = {p: i for i, p in enumerate(keep)}
            small = [[names.get(p, -1) if p >= 0 else p for p in r] for r in table]
            check(small, past, [20] * count, 20 * count, len(keep) + spare or 1, 16, wide=count < 10)


def test_what_the_caller_gets_wrong(cuda):
    """Negative lengths, more tokens than the step holds, keys past the table, page numbers outside the cache."""
    check([[0, 1], [2, 3]], [-4, 17], [-3, 2], 2, 8, 16)
    check([[0, 1], [2, 3], [4, 5]], [5, 30, 8], [7, 9, 4], 12, 9, 16)                  # 20 new tokens, room for 12
    check([[0, 1], [2, 3]], [5, 30], [1 << 30, 1 << 30], 12, 9, 16)
    check([[0, 1], [2, 3]], [31, 20], [40, 2], 42, 9, 16)                              # 71 keys on a table of 32
    check([[0, 1], [2, 3]], [1 << 30, 3], [4, 1], 5, 9, 16)
    check([[0, -1], [100, 3]], [20, 5], [1, 2], 3, 8, 16)                              # last pages that are no pages
    check([[7, 7], [7, 2]], [20, 5], [1, 1], 2, 8, 16)                                 # one page twice in a row


def test_copies_reach_every_layer(cuda):
    """The filled rows of a replaced page, in every layer and head, and nothing else."""
    rng = random.Random(12)
    for dt, layers, hkv, ps, d in ((torch.float16, 3, 2, 16, 128), (torch.bfloat16, 1, 8, 64, 64), (torch.float16, 28, 1, 16, 8)):
        for count, held in ((6, 2), (40, 8)):
            table, past, new, pages = make(rng, count, 3 * ps, ps, rows=held, spare=3 * count)
            rows = [rng.randrange(held) for _ in range(count)]
            caches = tuple(torch.randn(layers, pages, hkv, ps, d, device="cuda").to(dt) for _ in range(2))
            want = tuple(c.clone() for c in caches)
            res = oracle(table, past, [1] * count, count, pages, ps, rows)
            for b, (src, dst) in enumerate(res[6].tolist()):
                if dst >= 0:
                    n = past[rows[b]] % ps
                    for c in want:
                        c[:, dst, :, :n] = c[:, src, :, :n]
            got = ops.ext().plan_paged(i32(table), i32(past), i32([1] * count), count, pages, ps, rows=i32(rows), caches=caches)
            assert torch.equal(got.page_table, res[0]) and torch.equal(got.copies, res[6])
            assert torch.equal(caches[0], want[0]) and torch.equal(caches[1], want[1])
            if layers == 1:                                  # one layer's caches as forward_paged hands them out
                flat = tuple(c[0].clone() for c in caches)
                ops.ext().plan_paged(i32(table), i32(past), i32([1] * count), count, pages, ps, rows=i32(rows), caches=flat)
                assert torch.equal(flat[0], caches[0][0])


def test_more_sequences_and_pages_than_one_workgroup_takes(cuda):
    rng = random.Random(77)
    count, ps = 3000, 16
    table, past, new, pages = make(rng, count, 60, ps, share=0.2)
    print(count, pages, sum(new), flush=True)
    check(table, past, new, sum(new) + 9, pages, ps, wide=False)
    check([[700001, 3]], [17], [40], 40, 700002, ps, wide=False)
    check([[i for i in range(260)]], [16 * 260 - 3], [5000], 5000, 1 << 18, ps, wide=False)
    check([[5, 6]], [20], [4097], 4097, 300, ps, wide=False)
    check([[5, 6], [7, 9]], [20, 3], [9000, 77], 9080, 900, ps, wide=False)
    table, past, new, pages = make(rng, 300, 60, ps, share=0.3)
    check(table, past, [60] * 300, 18000, pages + 2000, ps, parents=[rng.randrange(60) for _ in range(18000)], wide=False)


def test_the_same_again_on_streams_and_in_graphs(cuda):
    """Captured with one batch, replayed with others between eager calls on the same and on another stream."""
    rng = random.Random(31)
    batches = [make(rng, 12, 200, 16, share=0.4) for _ in range(4)]
    width, pages = max(len(t[0]) for t, *_ in batches) + 1, max(p for *_, p in batches)
    for wide in (width, 1 << 13):                            # (one launch, four)
        table = torch.full((12, wide), -1, dtype=torch.int32, device="cuda")
        past, new = i32([0] * 12), i32([0] * 12)
        tokens = max(sum(n) for _, _, n, _ in batches) + 3

        def load(i):
            t, p, n, _ = batches[i]
            table.fill_(-1)
            table[:, :len(t[0])] = i32(t)
            past.copy_(i32(p))
            new.copy_(i32(n))
            return [r + [-1] * (wide - len(t[0])) for r in t], p, n

        load(0)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ops.ext().plan_paged(table, past, new, tokens, pages, 16)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step = ops.ext().plan_paged(table, past, new, tokens, pages, 16)
        for i in (1, 0, 2, 3, 3):
            t, p, n = load(i)
            graph.replay()
            eager = ops.ext().plan_paged(table, past, new, tokens, pages, 16)
            torch.cuda.synchronize()
            want = oracle(t, p, list(n), tokens, pages, 16)
            for name, a, b, c in zip(NAMES, step, eager, want):
                if c is not None:
                    assert torch.equal(a, c) and torch.equal(b, c), (name, i)


def test_more_nodes_than_masks_have_room_for(cuda):
    """A chain of 1024 nodes, whose last one has them all as ancestors; new tokens past the 1024th are outside the tree."""
    ps, past, sizes = 16, [37, 0, 5], [1500, 1024, 2]
    for parent in (lambda i: i - 1, lambda i: i // 2 - (i % 2 == 0)):
        parents = [parent(i) for n in sizes for i in range(n)]
        need = [-(-(p + n) // ps) for p, n in zip(past, sizes)]
        table = [[10 * b + i if i < -(-past[b] // ps) else -1 for i in range(max(need))] for b in range(3)]
        want = oracle(table, past, list(sizes), sum(sizes), sum(need) + 9, ps, None, parents, 16)
        want[3][1024:1500], want[5][1024:1500] = past[0], 0
        got = ops.ext().plan_paged(i32(table), i32(past), i32(sizes), sum(sizes), sum(need) + 9, ps, parents=i32(parents), words=16)
        for name, a, b in zip(NAMES, got, want):
            assert torch.equal(a, b), name

"""attention_paged_tree on the GPU against its definition in 64 bits: trees and masks of any kind, at the lengths where blocks, words
and pages end, rows that attend nothing, odd values in what a row leaves out. Bounds as for attention_paged (test_gpu_paged.py):
half a step of the type for each weight and for the output, the scores' and the sums' roundings in 32 bits."""
import math
import random

import pytest
import torch

from lowbit import ops

from test_gpu_paged import U, batch, half_step, least, widened

pytestmark = pytest.mark.gpu


def tree_bits(n, seed, forest=False):
    """[n, n] bool: node i attends itself and its ancestors."""
    rng = random.Random(seed)
    seen = torch.zeros(n, n, dtype=torch.bool)
    for i in range(n):
        seen[i, i] = True
        p = -1 if i == 0 or (forest and rng.random() < 0.2) else rng.choice([i - 1, rng.randrange(i)])
        if p >= 0:
            seen[i] |= seen[p]
    return seen


def random_bits(n, seed, density):
    g = torch.Generator().manual_seed(seed)
    return torch.rand(n, n, generator=g) < density


def pack(bits, words):
    """[n, n] bool -> int64 [n, words] (a bit that no word has room for is dropped)."""
    n = bits.shape[0]
    wide = torch.zeros(n, 64 * words, dtype=torch.int64)
    wide[:, :min(n, 64 * words)] = bits[:, :64 * words].long()
    return (wide.view(n, words, 64) << torch.arange(64)).sum(-1)


def want_of(q, k, v, new, keys, bits, scale):
    """(output, bound) of one sequence's rows in 64 bits; bits [new, new] says which new tokens a row attends."""
    hq, d, hkv = q.shape[1], q.shape[2], k.shape[1]
    g, dt, base = hq // hkv, q.dtype, keys - new
    alive = torch.zeros(new, keys, dtype=torch.bool)
    for j in range(keys):
        alive[:, j] = True if j < base else bits[:, j - base]
    alive = alive.cuda()
    some = alive.any(1)
    want, tol = torch.zeros(new, hq, d, dtype=torch.float64, device="cuda"), torch.zeros(new, hq, d, dtype=torch.float64, device="cuda")
    for h in range(hq):
        kh, vh = k[:, h // g].double(), v[:, h // g].double()
        s = (q[:, h].double() @ kh.t().contiguous() * scale).masked_fill(~alive, -math.inf)
        p = torch.where(some[:, None], torch.softmax(s, -1), torch.zeros_like(s))
        want[:, h] = p @ vh
        size = p @ vh.abs()
        reach = (q[:, h].double().abs() @ kh.abs().t().contiguous() * abs(scale)).masked_fill(~alive, 0)
        ds = (d + 8) * U * reach.amax(-1, keepdim=True) if keys else torch.zeros(new, 1, device="cuda")
        tol[:, h] = size * (half_step(dt) + 2 * ds + (keys / 16 + 64) * U)
    return want, tol + half_step(dt) * want.abs() + least(dt), some


def call(x, masks, scale, max_new, max_keys, split=True):
    out = torch.full_like(x[0], 777.0)
    ops.ext().attention_paged_tree(*x[:6], masks, out, max_new, max_keys, scale, split)
    torch.cuda.synchronize()
    return out


def check(x, lens, all_bits, words, scale, bounds=((None, None),), split=(True, False)):
    first, rows = x[7], x[0].shape[0]
    masks = torch.full((rows, words), -1, dtype=torch.int64)   # (rows of no sequence: never read)
    for b, bits in enumerate(all_bits):
        masks[first[b]:first[b + 1]] = pack(bits, words)
    masks = masks.cuda()
    wants = [want_of(x[0][first[b]:first[b + 1]], *x[6][b], new, keys, all_bits[b] & (torch.arange(new) < 64 * words), scale)
             if new else None for b, (new, keys) in enumerate(lens)]
    for max_new, max_keys in bounds:
        for s in split:
            out = call(x, masks, scale, max_new or max(1, max(n for n, _ in lens)), max_keys or max(1, max(k for _, k in lens)), s)
            for b, (new, keys) in enumerate(lens):
                if not new:
                    continue
                want, tol, some = wants[b]
                got = out[first[b]:first[b + 1]]
                bad = ~((got.double() - want).abs() <= tol)
                assert not bool(bad.any()), (b, new, keys, max_new, max_keys, s, bad.nonzero()[:3].tolist())
                assert int(torch.count_nonzero(got[~some])) == 0
            assert bool((out[:first[0]] == 777.0).all()) and bool((out[first[-1]:] == 777.0).all())
    return out


HEADS = [(12, 2, 128), (28, 4, 128), (8, 8, 64), (14, 2, 64), (3, 1, 128), (40, 1, 64), (32, 8, 128)]
BATCHES = [
    [(1, 1)], [(1, 700)], [(26, 26)], [(26, 926)], [(31, 31 + 1), (32, 32 + 31), (33, 33 + 32), (5, 5 + 33)],
    [(64, 64), (63, 63 + 17), (1, 300), (0, 40), (0, 0)], [(64, 64 + 191), (2, 1000)], [(40, 4000), (3, 3)]]


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_trees(cuda, hq, hkv, d, dt):
    for i, lens in enumerate(BATCHES):
        page = (16, 32, 64, 128, 256)[(i + hq) % 5]
        x = batch(lens, hq, hkv, d, page, dt, 100 * i + hq)
        print("batch", i, lens, page, flush=True)
        bits = [tree_bits(n, 10 * i + b, forest=b % 2 == 1) for b, (n, _) in enumerate(lens)]
        one = check(x, lens, bits, 1, d ** -0.5)
        assert torch.equal(one, check(x, lens, bits, 1, d ** -0.5, split=(False,)))


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (28, 4, 128), (4, 4, 128)])
def test_trees_of_several_words(cuda, hq, hkv, d, dt):
    """More nodes than a word has bits; more words than nodes need; nodes past the words, which nobody attends."""
    for i, (lens, words) in enumerate((([(65, 65), (130, 130 + 50)], 3), ([(250, 250 + 1000), (7, 300)], 4), ([(100, 131)], 16),
                                       ([(200, 333), (64, 64)], 1), ([(1024, 1024)], 16), ([(257, 257 + 95)], 5))):
        x = batch(lens, hq, hkv, d, (16, 64, 32)[i % 3], dt, 40 * i + hq)
        print(lens, words, flush=True)
        check(x, lens, [tree_bits(n, 3 * i + b) for b, (n, _) in enumerate(lens)], words, d ** -0.5)


# the bounds choose the tile and whether keys are split: every batch under every choice
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,d", [(28, 4, 128), (14, 2, 64), (8, 8, 64), (9, 1, 128)])
def test_trees_under_every_bound(cuda, hq, hkv, d, dt):
    for i, (lens, words) in enumerate((([(1, 700), (2, 3), (0, 9), (30, 31)], 1), ([(70, 700), (1, 513), (5, 1300)], 2),
                                       ([(133, 333), (1, 2100)], 3))):
        x = widened(batch(lens, hq, hkv, d, (16, 64, 32)[i], dt, 7 * i + hq), 1 << 16)
        bits = [tree_bits(n, 5 * i + b) for b, (n, _) in enumerate(lens)]
        print(lens, flush=True)
        check(x, lens, bits, words, d ** -0.5, [(1, 100), (1, 512), (1, 60000), (64, 300), (64, 1024), (64, 60000), (500, 60000),
                                                (1 << 40, 1 << 40)], split=(True,))


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_any_mask(cuda, dt):
    """Masks that are no trees: random ones, later nodes among them, empty ones, full ones."""
    lens = [(20, 20), (33, 500), (64, 64), (1, 1), (90, 90 + 7)]
    x = batch(lens, 16, 2, 128, 16, dt, 77, extra_rows=3, first=2)
    for density in (0.0, 0.03, 0.5, 1.0):
        check(x, lens, [random_bits(n, b, density) for b, (n, _) in enumerate(lens)], 2, 0.09,
              [(None, None), (1, 100), (200, 60000)])


def test_a_causal_mask_is_causal_attention(cuda):
    """Both calls lie within the definition's bound of it, so within twice that of each other (not the same bits: the two calls cut
    rows and keys differently, which changes the order of the sums)."""
    lens = [(30, 200), (1, 900), (64, 64)]
    x = batch(lens, 28, 4, 128, 16, torch.float16, 4)
    causal = call(x, torch.cat([pack(torch.ones(n, n).tril().bool(), 1) for n, _ in lens]).cuda(), 0.09, 64, 900)
    out = torch.empty_like(x[0])
    ops.ext().attention_paged(*x[:6], out, 64, 900, 0.09)
    for b, (n, keys) in enumerate(lens):
        rows = slice(x[7][b], x[7][b + 1])
        _, tol, _ = want_of(x[0][rows], *x[6][b], n, keys, torch.ones(n, n).tril().bool(), 0.09)
        assert bool(((causal[rows].double() - out[rows].double()).abs() <= 2 * tol).all())


def test_rows_without_keys(cuda):
    """More new tokens than keys: the nodes in front of key 0 have no keys, and a row that attends only those gets zeros."""
    for lens in ([(4, 0), (6, 2), (1, 0), (70, 3), (2, 9)], [(200, 130)]):
        words = 4
        x = batch(lens, 12, 2, 128, 16, torch.bfloat16, 5, extra_rows=3, first=2)
        for density in (0.02, 0.3):
            all_bits = [random_bits(n, b, density) for b, (n, _) in enumerate(lens)]
            masks = torch.zeros(x[0].shape[0], words, dtype=torch.int64)
            for b, bits in enumerate(all_bits):
                masks[x[7][b]:x[7][b + 1]] = pack(bits, words)
            for split in (True, False):
                out = call(x, masks.cuda(), 0.1, max(n for n, _ in lens), max(1, max(k for _, k in lens)), split)
                for b, (new, keys) in enumerate(lens):
                    bits = all_bits[b].clone()
                    bits[:, :max(0, new - keys)] = False
                    at = keys - new
                    # the definition's keys: node j at key at + j, those below 0 missing
                    live = bits[:, -at:] if at < 0 else bits
                    q = x[0][x[7][b]:x[7][b + 1]]
                    k, v = x[6][b]
                    full = torch.cat([torch.ones(new, max(at, 0), dtype=torch.bool), live], 1)
                    got = out[x[7][b]:x[7][b + 1]]
                    for h in range(12):
                        s = (q[:, h].double() @ k[:, h // 6].double().t().contiguous() * 0.1).masked_fill(~full.cuda(), -math.inf)
                        some = full.any(1).cuda()
                        p = torch.where(some[:, None], torch.softmax(s, -1), torch.zeros_like(s))
                        want, size = p @ v[:, h // 6].double(), p @ v[:, h // 6].double().abs()
                        # (half a step for each weight and the output; the scores' and sums' 32 bits are far below a quarter)
                        tol = half_step(torch.bfloat16) * (size + want.abs()) + 0.5 * half_step(torch.bfloat16) * size
                        assert bool(((got[:, h].double() - want).abs() <= tol).all()), (b, h)
                        assert int(torch.count_nonzero(got[~some, h])) == 0


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new,keys", [(20, 20), (20, 700), (64, 100), (100, 1200)])
def test_odd_values_reach_only_the_rows_that_attend_them(cuda, new, keys, dt):
    """An infinity or a NaN in a node's k or v does not reach the rows of other branches: they stay within the definition's bounds. (Not
    the same bits: a score that passes one row's reference moves the references of the rows beside it, and each weight is rounded
    against the reference, half a step of the weight: half a step of sum p |v| in the output, more than a step of an output
    that is small beside its terms.)"""
    x = batch([(new, keys)], 16, 2, 128, 16, dt, new + keys)
    bits = tree_bits(new, 9)
    masks = pack(bits, 2).cuda()
    want, tol, _ = want_of(x[0], *x[6][0], new, keys, bits, 0.09)
    page, table = 16, x[3]
    for node, where, value in ((new // 2, 2, math.inf), (new - 1, 2, math.nan), (3, 1, math.nan), (new // 3, 1, math.inf)):
        key = keys - new + node
        cache = x[where]
        was = cache[table[0, key // page].long(), :, key % page].clone()
        cache[table[0, key // page].long(), :, key % page, 5] = value
        for split in (True, False):
            out = call(x, masks, 0.09, new, keys, split)
            base = call(x, masks, 0.09, new, keys, split)
            attends = bits[:, node].cuda()
            assert bool(((out[~attends].double() - want[~attends]).abs() <= tol[~attends]).all())
            odd = ~torch.isfinite(out[attends].float())
            if value != value:
                assert bool(odd.any(-1).all())
            elif where == 2:
                assert bool((out[attends][..., 5] == math.inf).all())
            assert torch.equal(torch.nan_to_num(out.float(), nan=5e4), torch.nan_to_num(base.float(), nan=5e4))
        cache[table[0, key // page].long(), :, key % page] = was


def test_strides_streams_graphs(cuda):
    """On another stream, and captured: replays with other lengths, masks and tables than those of the capture."""
    lens = [[(26, 900), (40, 300)], [(10, 77), (3, 1111)], [(26, 26), (33, 64)]]
    xs = [batch(l, 28, 4, 128, 16, torch.float16, 60 + i) for i, l in enumerate(lens)]
    rows, width, pages = max(x[0].shape[0] for x in xs), max(x[3].shape[1] for x in xs), max(x[1].shape[0] for x in xs)
    q = torch.zeros(rows, 28, 128, dtype=torch.float16, device="cuda")
    out = torch.zeros_like(q)
    kc = torch.zeros(pages, 4, 16, 128, dtype=torch.float16, device="cuda")
    vc = torch.zeros_like(kc)
    table = torch.zeros(2, width, dtype=torch.int32, device="cuda")
    starts, kv = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    masks = torch.zeros(rows, 1, dtype=torch.int64, device="cuda")
    run = lambda: ops.ext().attention_paged_tree(q, kc, vc, table, starts, kv, masks, out, 64, 1200, 0.09)   # noqa: E731

    def load(i):
        x = xs[i]
        q[:x[0].shape[0]], table[:, :x[3].shape[1]] = x[0], x[3]
        kc[:x[1].shape[0]], vc[:x[2].shape[0]] = x[1], x[2]
        starts.copy_(x[4])
        kv.copy_(x[5])
        masks[:x[0].shape[0]] = torch.cat([pack(tree_bits(n, i + b), 1) for b, (n, _) in enumerate(lens[i])]).cuda()

    load(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    eager = out.clone()
    run()
    assert torch.equal(out, eager)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        run()
    for i in (1, 2, 0, 1):
        load(i)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        out.zero_()
        run()
        torch.cuda.synchronize()
        assert torch.equal(got, out)


def test_starts_that_do_not_hold(cuda):
    """Starts past q's rows or below zero are held to them, and nothing outside out is written."""
    lens = [(4, 50), (3, 40)]
    x = list(batch(lens, 16, 2, 128, 16, torch.float16, 3))
    masks = torch.full((7, 1), -1, dtype=torch.int64, device="cuda")
    room = torch.full((7 + 8, 16, 128), 777.0, dtype=torch.float16, device="cuda")
    for starts in ([-5, 4, 1000], [0, 4, 7], [7, 7, 7], [900, 900, 900], [-3, -2, -1], [6, 2, 7]):
        x[4] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        for keys in (50, 1 << 20):
            room.fill_(777.0)
            ops.ext().attention_paged_tree(*x[:6], masks, room[4:11], 4, keys, 0.1)
            torch.cuda.synchronize()
            assert bool((room[:4] == 777.0).all()) and bool((room[11:] == 777.0).all())


def test_many_sequences(cuda):
    """More sequences than shares are balanced for at once, of equal and of very different lengths."""
    for n, hq, hkv, d in ((70, 28, 4, 128), (300, 8, 2, 64)):
        lens = [(1 + i % 7, 1 + i % 7 + (i * 37) % 200) for i in range(n)]
        lens[3], lens[n - 2] = (40, 5000), (3, 9000)
        x = batch(lens, hq, hkv, d, 32, torch.float16, n)
        check(x, lens, [tree_bits(k, i) for i, (k, _) in enumerate(lens)], 1, d ** -0.5)


@pytest.mark.parametrize("hq,hkv,d", [(28, 4, 128), (8, 8, 64)])
def test_a_step_without_new_tokens(cuda, hq, hkv, d):
    """Every row padded, after a call that leaves its split tiles in memory that the next call may get as its workspace: out stays."""
    for lens in ([(8, 5000)], [(100, 9000), (60, 7000)]):
        x = list(batch(lens, hq, hkv, d, 64, torch.float16, 5))
        bits = [tree_bits(n, b) for b, (n, _) in enumerate(lens)]
        check(x, lens, bits, 2, d ** -0.5, split=(True,))
        masks = torch.full((x[0].shape[0], 2), -1, dtype=torch.int64, device="cuda")
        x[4] = torch.full_like(x[4], x[0].shape[0])
        for starts in (x[4], torch.zeros_like(x[4])):
            x[4] = starts
            out = call(x, masks, d ** -0.5, max(n for n, _ in lens), max(k for _, k in lens))
            assert bool((out == 777.0).all())

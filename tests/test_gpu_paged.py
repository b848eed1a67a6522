"""A batch of sequences over a paged cache on the GPU: norm_rope_paged and attention_paged against their definitions in 64
bits, at the sizes and lengths where they can go wrong.

Bounds. A stored value is off by half a step of its type, eps / 2 of it (in fp16 at least 2^-25, half the smallest step).
norm_rope_paged computes the pair (a, b) = normalized x and its turn in 32 bits: the sum of squares, the root and the two
products cost under 16 roundings of 2^-24 relative to |a| + |b|, the angle's last part of a turn (rounded to 2^-25 turns =
2^-22.3 radians) and the sine another 8: 32 * 2^-24 (|a| + |b|) in all.
attention_paged rounds each weight to the type (eps / 2 of it, so at most eps / 2 * sum p |v| =: eps / 2 * A), forms scores
of D exact products in 32 bits (a score is off by ds <= (D + 8) 2^-24 sum |q k| scale, which moves the weights' sum and the
output's by that much relatively: 2 ds A) and adds n keys' products in 32 bits, at least 16 to a step: (n / 16 + 64) 2^-24 A."""
import math

import pytest
import torch

from lowbit import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def half_step(dt):
    return torch.finfo(dt).eps / 2


def least(dt):
    return 2.0 ** -25 if dt is torch.float16 else 0.0


# ---- norm_rope_paged ----

def rope_inputs(m, hq, hkv, d, page, dt, seed, pages=None, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    width = (hq + 2 * hkv) * d
    qkv = (1.5 * torch.randn(m, width + pad, generator=g, device="cuda")).to(dt)[:, :width]
    qw = (1 + 0.3 * torch.randn(d, generator=g, device="cuda")).to(dt)
    kw = (1 + 0.3 * torch.randn(d, generator=g, device="cuda")).to(dt)
    pos = torch.randint(0, 1 << 20, (m,), generator=g, device="cuda")
    inv = 1.0 / (1e6 ** (torch.arange(0, d, 2, dtype=torch.float32, device="cuda") / d))
    pages = pages or -(-m // page) + 3
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:m].clone()
    caches = torch.randn(2, pages, hkv, page, d, generator=g, device="cuda").to(dt)
    return qkv, qw, kw, pos, inv, slots, caches[0], caches[1]


def rope_want(qkv, qw, kw, eps, pos, inv, hq, hkv, d):
    """(rotated q and k heads, their bound's |a| + |b|, v heads) in 64 bits."""
    x = qkv.double().reshape(qkv.shape[0], -1, d)
    y = x[:, :hq + hkv]
    if qw is not None:
        w = torch.cat([qw.double().expand(hq, d), kw.double().expand(hkv, d)])
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w
    ang = pos.double()[:, None, None] * inv.double()
    a, b = y[..., :d // 2], y[..., d // 2:]
    out = torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1)
    size = (a.abs() + b.abs()).repeat(1, 1, 2)
    return out, size, x[:, hq + hkv:]


def check_rope(inputs, hq, hkv, d, norm=True, permuted=False, eps=1e-6):
    qkv, qw, kw, pos, inv, slots, kc, vc = inputs
    if not norm:
        qw = kw = None
    m, page, dt = qkv.shape[0], kc.shape[2], qkv.dtype
    want, size, v = rope_want(qkv, qw, kw, eps, pos, inv, hq, hkv, d)
    kc0, vc0 = kc.clone(), vc.clone()
    q = torch.full((m, hq, d), float("nan"), dtype=dt, device="cuda")
    given = qkv
    if permuted:
        from lowbit import fused
        given = qkv[:, fused.rope_permutation(hq + 2 * hkv, d).cuda()]
    ops.ext().norm_rope_paged(given, qw, kw, eps, pos, inv, slots, q, kc, vc, hq, hkv, permuted)
    tol = half_step(dt) * want.abs() + least(dt) + 32 * U * size
    assert bool(((q.double() - want[:, :hq]).abs() <= tol[:, :hq]).all())
    at = ((slots >= 0) & (slots < kc.shape[0] * page)).nonzero()[:, 0]
    p, r = slots[at] // page, slots[at] % page
    assert bool(((kc[p, :, r].double() - want[at, hq:]).abs() <= tol[at, hq:]).all())
    assert torch.equal(vc[p, :, r].double(), v[at])
    kc0[p, :, r], vc0[p, :, r] = kc[p, :, r], vc[p, :, r]
    assert torch.equal(kc, kc0) and torch.equal(vc, vc0)     # no other row is touched
    return q


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,hq,hkv,d,page", [(1, 28, 4, 128, 64), (1, 1, 1, 64, 16), (1, 1, 1, 128, 16), (2, 3, 1, 128, 16),
                                             (5, 14, 2, 64, 32), (33, 16, 2, 128, 16), (67, 12, 2, 128, 128),
                                             (130, 8, 8, 64, 16), (257, 5, 5, 128, 16), (1000, 28, 4, 128, 64),
                                             (3001, 14, 2, 64, 16), (2049, 32, 8, 128, 256), (7, 65, 13, 128, 16)])
def test_norm_rope(cuda, m, hq, hkv, d, page, dt):
    check_rope(rope_inputs(m, hq, hkv, d, page, dt, m + hq), hq, hkv, d)
    check_rope(rope_inputs(m, hq, hkv, d, page, dt, m + hq + 1), hq, hkv, d, norm=False)
    check_rope(rope_inputs(m, hq, hkv, d, page, dt, m + hq + 2, pad=40), hq, hkv, d, permuted=True)


def test_norm_rope_slots_outside_the_cache_write_nothing(cuda):
    for m in (1, 6, 40, 600):
        x = rope_inputs(m, 16, 2, 128, 16, torch.float16, m)
        x[5][::3] = -1
        x[5][1::3] = x[6].shape[0] * 16
        if m > 5:
            x[5][4], x[5][5] = -(1 << 40), 1 << 40
        check_rope(x, 16, 2, 128)


def test_norm_rope_positions(cuda):
    """Position 0 leaves the values as they are; positions past 32 bits and below 0 turn by their own angles."""
    x = list(rope_inputs(9, 12, 2, 128, 16, torch.float16, 3))
    x[3] = torch.tensor([0, 1, -1, 131071, 1 << 24, (1 << 24) + 1, (1 << 33) + 5, -(1 << 33), 7], device="cuda")
    check_rope(x, 12, 2, 128)
    x[3] = torch.zeros(9, dtype=torch.long, device="cuda")
    q = check_rope(x, 12, 2, 128, norm=False)
    assert torch.equal(q, x[0].reshape(9, -1, 128)[:, :12])


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_norm_rope_values(cuda, dt):
    """Heads of zeros, of the type's largest values (whose squares pass fp16), of its smallest, and one NaN head that stays
    alone."""
    hq, hkv, d = 8, 2, 128
    x = rope_inputs(5, hq, hkv, d, 16, dt, 11)
    heads = x[0].reshape(5, -1, d)
    heads[0] = 0
    heads[1] = 6e4 if dt is torch.float16 else 1e18
    heads[2] = 6e-8 if dt is torch.float16 else 1e-18
    check_rope(x, hq, hkv, d, eps=1e-6)
    x = rope_inputs(4, hq, hkv, d, 16, dt, 12)
    clean = check_rope(x, hq, hkv, d)
    x[0].reshape(4, -1, d)[2, 3, 77] = float("nan")
    q = torch.empty_like(clean)
    ops.ext().norm_rope_paged(x[0], x[1], x[2], 1e-6, x[3], x[4], x[5], q, x[6], x[7], hq, hkv)
    assert bool(q[2, 3].isnan().all())
    q[2, 3], clean[2, 3] = 0, 0
    assert torch.equal(q, clean)


def test_norm_rope_in_a_cache_past_32_bits(cuda):
    pages = (1 << 32) // (4 * 64 * 128 * 2) + 40           # 4 GiB of keys and 40 pages
    kc = torch.zeros(pages, 4, 64, 128, dtype=torch.float16, device="cuda")
    vc = torch.zeros_like(kc)
    x = list(rope_inputs(3, 8, 4, 128, 64, torch.float16, 4))
    x[5] = torch.tensor([pages * 64 - 1, 5, (pages - 20) * 64 + 13], device="cuda")
    q = torch.empty(3, 8, 128, dtype=torch.float16, device="cuda")
    ops.ext().norm_rope_paged(*x[:3], 1e-6, *x[3:6], q, kc, vc, 8, 4)
    want, size, v = rope_want(*x[:3], 1e-6, *x[3:5], 8, 4, 128)
    p, r = x[5] // 64, x[5] % 64
    tol = half_step(torch.float16) * want.abs() + least(torch.float16) + 32 * U * size
    assert bool(((kc[p, :, r].double() - want[:, 8:]).abs() <= tol[:, 8:]).all())
    assert torch.equal(vc[p, :, r].double(), v)
    vc[p, :, r] = 0
    assert int(torch.count_nonzero(vc)) == 0


# ---- attention_paged ----

def batch(lens, hq, hkv, d, page, dt, seed, extra_rows=0, first=0, scale=1.5):
    """Sequences of (new tokens, keys): q, caches whose unused rows hold NaN, table, starts, lengths, and every sequence's
    keys and values [keys, hkv, d]."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    need = [max(1, -(-k // page)) for _, k in lens]
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(need) + 1), -5, dtype=torch.int32, device="cuda")
    kc = torch.full((pages, hkv, page, d), float("nan"), dtype=dt, device="cuda")
    vc = torch.full_like(kc, float("inf"))
    kv, at = [], 0
    for b, (new, keys) in enumerate(lens):
        table[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
        k = torch.randn(keys, hkv, d, generator=g, device="cuda").to(dt)
        v = torch.randn(keys, hkv, d, generator=g, device="cuda").to(dt)
        j = torch.arange(keys, device="cuda")
        where = table[b].long()[j // page]
        kc[where, :, j % page], vc[where, :, j % page] = k, v
        kv.append((k, v))
    starts = [first]
    for new, _ in lens:
        starts.append(starts[-1] + new)
    q = (scale * torch.randn(starts[-1] + extra_rows, hq, d, generator=g, device="cuda")).to(dt)
    return (q, kc, vc, table, torch.tensor(starts, dtype=torch.int32, device="cuda"),
            torch.tensor([k for _, k in lens], dtype=torch.int32, device="cuda"), kv, starts)


def attend_want(q, k, v, new, keys, scale):
    """(output, bound without the output's own rounding's type) of one sequence's rows [new, hq, d] in 64 bits."""
    hq, d, hkv = q.shape[1], q.shape[2], k.shape[1]
    g, dt = hq // hkv, q.dtype
    want = torch.zeros(new, hq, d, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(want)
    last = keys - new + torch.arange(new, device="cuda")
    for h in range(hq):
        kh, vh = k[:, h // g].double(), v[:, h // g].double()
        s = q[:, h].double() @ kh.t().contiguous() * scale
        dead = torch.arange(keys, device="cuda")[None, :] > last[:, None]
        p = torch.softmax(s.masked_fill(dead, -math.inf), -1)
        p = torch.where(last[:, None] < 0, torch.zeros_like(p), p)
        want[:, h] = p @ vh
        size = p @ vh.abs()
        ds = (d + 8) * U * (q[:, h].double().abs() @ kh.abs().t().contiguous() * abs(scale)).masked_fill(dead, 0).amax(-1, keepdim=True) \
            if keys else torch.zeros(new, 1, device="cuda")
        tol[:, h] = size * (half_step(dt) + 2 * ds + (keys / 16 + 64) * U)
    return want, tol + half_step(dt) * want.abs() + least(dt)


def check_attend(x, lens, scale, max_new=None, max_keys=None, split=True):
    q, kc, vc, table, starts, kv_lens, kv, first = x
    out = torch.full_like(q, 777.0)
    ops.ext().attention_paged(q, kc, vc, table, starts, kv_lens, out, max_new or max(1, max(n for n, _ in lens)),
                              max_keys or max(1, max(k for _, k in lens)), scale, split)
    torch.cuda.synchronize()
    for b, (new, keys) in enumerate(lens):
        rows = slice(first[b], first[b + 1])
        if new == 0:
            continue
        want, tol = attend_want(q[rows], kv[b][0], kv[b][1], new, keys, scale)
        bad = ~((out[rows].double() - want).abs() <= tol)
        assert not bool(bad.any()), (b, new, keys, bad.nonzero()[:3].tolist())
    assert bool((out[:first[0]] == 777.0).all()) and bool((out[first[-1]:] == 777.0).all())
    return out


HEADS = [(12, 2, 128), (28, 4, 128), (8, 8, 64), (14, 2, 64), (3, 1, 128), (40, 1, 64), (32, 8, 128)]
BATCHES = [
    [(1, 1)], [(1, 2)], [(1, 15), (1, 16), (1, 17)], [(1, 700)], [(3, 3)], [(1, 4000), (1, 1), (1, 129)],
    [(0, 0), (1, 31), (0, 40), (1, 33), (0, 5)], [(5, 5), (1, 64), (40, 40), (1, 300)],
    [(65, 65)], [(64, 191), (1, 1000)], [(127, 1500), (2, 2), (9, 1030)], [(300, 300), (31, 257)],
    [(129, 129 + 32), (33, 33 + 95), (1, 96), (1, 97)]]


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_attention_paged(cuda, hq, hkv, d, dt):
    for i, lens in enumerate(BATCHES):
        page = (16, 32, 64, 128, 256)[(i + hq) % 5]
        x = batch(lens, hq, hkv, d, page, dt, 100 * i + hq)
        print("batch", i, lens, page, flush=True)
        one = check_attend(x, lens, d ** -0.5)
        assert torch.equal(one, check_attend(x, lens, d ** -0.5))          # the same bits again
        check_attend(x, lens, d ** -0.5, split=False)
        check_attend(x, lens, d ** -0.5, max_new=1, max_keys=1)            # bounds that are too low, and far too high
        check_attend(x, lens, d ** -0.5, max_new=1 << 40, max_keys=1 << 40)


def widened(x, keys):
    """The batch with a table of room for `keys` keys (its own pages first), so that bounds are not held to its length."""
    page = x[1].shape[2]
    table = torch.full((x[3].shape[0], -(-keys // page)), -1, dtype=torch.int32, device="cuda")
    table[:, :x[3].shape[1]] = x[3][:, :table.shape[1]]
    return x[:3] + (table,) + x[4:]


# the bounds choose the tile (at most 32 rows and few keys: one wave where the batch is large, else four; 64 rows and 1024 keys;
# 128 rows) and whether keys are split: every batch under every choice
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,d", [(28, 4, 128), (14, 2, 64), (8, 8, 64), (9, 1, 128)])
def test_attention_paged_under_every_bound(cuda, hq, hkv, d, dt):
    for i, lens in enumerate(([(1, 700), (2, 3), (0, 9), (1, 1)], [(70, 700), (1, 513), (5, 1300)], [(333, 333), (1, 2100)])):
        x = widened(batch(lens, hq, hkv, d, (16, 64, 32)[i], dt, 7 * i + hq), 1 << 16)
        for max_new, max_keys in ((1, 100), (1, 512), (1, 60000), (64, 300), (64, 1024), (64, 60000), (500, 60000)):
            print(lens, max_new, max_keys, flush=True)
            check_attend(x, lens, d ** -0.5, max_new, max_keys)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,d,n", [(28, 4, 128, 130), (16, 8, 64, 200), (4, 4, 128, 333)])
def test_attention_paged_of_many_sequences(cuda, hq, hkv, d, n, dt):
    """More sequences than a wave has lanes, among them some without new tokens and some without keys; short keys, then a few
    long ones among them, which are split while the others are not."""
    short = [(0 if i % 17 == 5 else 1 + (i % 23 == 3), 0 if i % 29 == 7 else 1 + (i * 37) % 300) for i in range(n)]
    short = [(a, max(a, b) if b else 0) for a, b in short]
    check_attend(batch(short, hq, hkv, d, 16, dt, n), short, d ** -0.5)
    long = list(short)
    for i, keys in ((2, 9000), (70, 5000), (n - 1, 20011)):
        long[i] = (1, keys)
    x = batch(long, hq, hkv, d, 32, dt, n + 1)
    one = check_attend(x, long, d ** -0.5)
    assert torch.equal(one, check_attend(x, long, d ** -0.5))
    long[n // 2] = (150, 4000)                               # and a piece of a prompt
    check_attend(batch(long, hq, hkv, d, 64, dt, n + 2), long, d ** -0.5)


def test_attention_paged_of_shared_pages(cuda):
    """Two sequences that begin with the same pages (a shared prefix), and one page twice in a sequence."""
    lens = [(3, 200), (1, 150), (40, 300)]
    x = list(batch(lens, 16, 2, 128, 16, torch.float16, 3))
    x[3][1, :8] = x[3][0, :8]
    x[3][2, 5] = x[3][2, 2]
    k1, v1 = x[6][1]
    k1[:128], v1[:128] = x[6][0][0][:128], x[6][0][1][:128]
    k2, v2 = x[6][2]
    k2[80:96], v2[80:96] = k2[32:48].clone(), v2[32:48].clone()
    check_attend(x, lens, 128 ** -0.5)


def test_attention_paged_with_starts_that_do_not_hold(cuda):
    """Starts past q's rows or below zero are held to them, and nothing outside out is written."""
    lens = [(4, 50), (3, 40)]
    x = list(batch(lens, 16, 2, 128, 16, torch.float16, 3))
    room = torch.full((7 + 8, 16, 128), 777.0, dtype=torch.float16, device="cuda")
    for starts in ([-5, 4, 1000], [0, 4, 7], [7, 7, 7], [900, 900, 900], [-3, -2, -1]):
        x[4] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        room.fill_(777.0)
        ops.ext().attention_paged(*x[:6], room[4:11], 4, 50, 0.1)
        torch.cuda.synchronize()
        assert bool((room[:4] == 777.0).all()) and bool((room[11:] == 777.0).all())


def test_attention_paged_rows_without_keys_and_of_no_sequence(cuda):
    """New tokens before a sequence's first key get zeros; rows in front of, between and behind the sequences stay."""
    for dt, lens in ((torch.float16, [(4, 0), (6, 2), (1, 0), (70, 3), (2, 9)]), (torch.bfloat16, [(1, 0)]),
                     (torch.float16, [(1, 0), (1, 500), (1, 0)]), (torch.float16, [(200, 130), (300, 0)])):
        x = batch(lens, 12, 2, 128, 16, dt, 5, extra_rows=3, first=2)
        out = check_attend(x, lens, 0.1)
        for b, (new, keys) in enumerate(lens):
            assert int(torch.count_nonzero(out[x[7][b]:x[7][b] + max(0, new - keys)])) == 0


def test_attention_paged_pages_outside_the_cache_read_as_zeros(cuda):
    for lens in ([(1, 200)], [(50, 300)], [(200, 200)]):
        x = list(batch(lens, 16, 2, 128, 16, torch.float16, 8))
        for at, bad in ((2, -1), (5, x[1].shape[0]), (9, 1 << 30), (11, -(1 << 31))):
            x[3][0, at] = bad
            for t in x[6][0]:
                t[16 * at:16 * at + 16] = 0
        check_attend(x, lens, 0.1)


def test_attention_paged_lengths_past_the_table(cuda):
    """Keys past the table's pages are not attended: positions stay where they are, the keys end earlier."""
    lens = [(3, 64)]
    x = list(batch(lens, 16, 2, 128, 16, torch.float16, 9))
    x[3] = x[3][:, :4].contiguous()
    x[5] = torch.tensor([80], dtype=torch.int32, device="cuda")             # positions 77 .. 79 of 64 keys
    out = torch.empty_like(x[0])
    ops.ext().attention_paged(*x[:6], out, 3, 80, 0.1)
    for i in range(3):
        want, tol = attend_want(x[0][i:i + 1], *x[6][0], 1, 64, 0.1)
        assert bool(((out[i:i + 1].double() - want).abs() <= tol).all())


@pytest.mark.parametrize("scale", [-0.1, 0.0, 1e-30, 2.0])
@pytest.mark.parametrize("lens", [[(1, 500)], [(90, 400), (1, 30)]])
def test_attention_paged_scales(cuda, lens, scale):
    check_attend(batch(lens, 12, 2, 128, 16, torch.float16, 5), lens, scale)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_attention_paged_growing_and_falling_scores(cuda, dt):
    """Every block of keys raises the rows' maximum far past the one before, then lowers it again."""
    for lens in ([(1, 1024)], [(64, 1024)], [(300, 1024)]):
        for flip in (False, True):
            x = batch(lens, 16, 2, 128, 64, dt, 9)
            ramp = torch.linspace(0.05, 4.0, 1024, device="cuda").to(dt)
            k = x[6][0][0] * (ramp.flip(0) if flip else ramp)[:, None, None]
            x[6][0] = (k, x[6][0][1])
            j = torch.arange(1024, device="cuda")
            x[1][x[3][0].long()[j // 64], :, j % 64] = k
            check_attend(x, lens, 128 ** -0.5)


def test_attention_paged_in_a_cache_past_32_bits(cuda):
    hq, hkv, d, page = 16, 2, 128, 64
    pages = (1 << 32) // (hkv * page * d * 2) + 60
    kc = torch.zeros(pages, hkv, page, d, dtype=torch.float16, device="cuda")
    vc = torch.zeros_like(kc)
    for lens in ([(1, 300)], [(150, 300)]):
        x = list(batch(lens, hq, hkv, d, page, torch.float16, 21))
        table = torch.full_like(x[3], -1)
        for i in range(5):
            at = int(x[3][0, i])
            table[0, i] = pages - 1 - 7 * i if i != 2 else 3
            kc[table[0, i]], vc[table[0, i]] = x[1][at], x[2][at]
        x[1], x[2], x[3] = kc, vc, table
        check_attend(x, lens, d ** -0.5)


def test_attention_paged_long_context(cuda):
    for lens in ([(1, 70001)], [(2, 33000), (1, 64000), (1, 10)], [(20, 30000)], [(1, 1 + 257 * i) for i in range(70)]):
        x = batch(lens, 28, 4, 128, 64, torch.float16, 31)
        print(lens[:4], flush=True)
        check_attend(x, lens, 128 ** -0.5)


def test_attention_paged_small_weights_keep_their_sum(cuda):
    """One key of weight 1 and value 0 beside tens of thousands of weights of 2^-24, whose sum alone makes the output."""
    n = 60000
    for new in (1, 40):
        lens = [(new, n)]
        x = batch(lens, 16, 2, 128, 64, torch.float16, 6)
        q = torch.zeros_like(x[0])
        q[..., 0] = 1
        k, v = torch.zeros_like(x[6][0][0]), (1 + 0.25 * torch.randn(n, 2, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))).half()
        k[100, :, 0], v[100] = 128.0, 0
        j = torch.arange(n, device="cuda")
        where = x[3][0].long()[j // 64]
        x[1][where, :, j % 64], x[2][where, :, j % 64] = k, v
        x[6][0] = (k, v)
        check_attend((q,) + x[1:], lens, 24 * math.log(2.0) / 128)


def test_attention_paged_captured_with_changing_lengths(cuda):
    """A graph captured once serves other lengths, starts and tables: every replay has the eager call's bits."""
    sets = [[(1, 5), (30, 31), (1, 900)], [(16, 1000), (1, 1), (15, 15)], [(0, 0), (32, 700), (0, 3)], [(1, 5000), (1, 4999), (30, 5000)]]
    data = [batch(s, 16, 2, 128, 16, torch.float16, i) for i, s in enumerate(sets)]
    pages, width = max(x[1].shape[0] for x in data), max(x[3].shape[1] for x in data)
    kc = torch.zeros(pages, 2, 16, 128, dtype=torch.float16, device="cuda")
    vc = torch.zeros_like(kc)
    q, out = torch.empty(32, 16, 128, dtype=torch.float16, device="cuda"), torch.empty(32, 16, 128, dtype=torch.float16, device="cuda")
    table = torch.zeros(3, width, dtype=torch.int32, device="cuda")
    starts, lens = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")

    def load(x):
        q.zero_()[:x[0].shape[0]] = x[0]
        kc[:x[1].shape[0]], vc[:x[2].shape[0]] = x[1], x[2]
        table.fill_(-1)[:, :x[3].shape[1]] = x[3]
        starts.copy_(x[4])
        lens.copy_(x[5])

    def call(o):
        ops.ext().attention_paged(q, kc, vc, table, starts, lens, o, 32, 5000, 128 ** -0.5)

    load(data[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        call(out)
    for i in (0, 1, 2, 3, 1, 0):
        load(data[i])
        eager = torch.full_like(out, 5.0)
        call(eager)
        out.fill_(5.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager), i
        check_attend(data[i], sets[i], 128 ** -0.5, max_new=32, max_keys=5000)


def test_paged_calls_on_two_streams_and_two_graphs_at_once(cuda):
    """Calls that run at the same time share nothing: two streams, then two graphs captured on one stream and replayed on
    two."""
    lens = [(1, 3000), (1, 2000)]
    xs = [batch(lens, 16, 2, 128, 16, torch.float16, i) for i in (1, 2)]
    want = [check_attend(x, lens, 0.1) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    outs = [torch.zeros_like(w) for w in want]
    torch.cuda.synchronize()
    for _ in range(20):
        for x, s, o in zip(xs, streams, outs):
            with torch.cuda.stream(s):
                ops.ext().attention_paged(*x[:6], o, 1, 3000, 0.1)
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))
    graphs = []
    for x, o in zip(xs, outs):
        o.zero_()
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=streams[0]):
            for _ in range(10):
                ops.ext().attention_paged(*x[:6], o, 1, 3000, 0.1)
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,d", [(16, 2, 128), (14, 2, 64)])
def test_attention_paged_of_keys_that_are_not_finite(cuda, hq, hkv, d, dt):
    """An infinity or a NaN in a token's k or v reaches the rows that attend it and no other: those before it have the bits
    that they have without it, in tiles of every kind, split and not."""
    for lens, at in (([(5, 300)], 297), ([(60, 60)], 31), ([(300, 300), (1, 40)], 150), ([(200, 1500)], 1400), ([(9, 2000)], 1995)):
        for which, bad in ((1, float("nan")), (2, float("nan")), (2, float("inf")), (2, -float("inf"))):
            x = list(batch(lens, hq, hkv, d, 16, dt, at))
            clean = torch.empty_like(x[0])
            new, keys = lens[0]
            args = (max(n for n, _ in lens), max(k for _, k in lens), d ** -0.5)
            ops.ext().attention_paged(*x[:6], clean, *args)
            x[which][x[3][0, at // 16], 0, at % 16, 5] = bad   # of the first KV head
            out = torch.empty_like(clean)
            ops.ext().attention_paged(*x[:6], out, *args)
            first, g = at - (keys - new), hq // hkv          # the first row that attends it
            hit = out[first:new, :g, 5] if which == 2 else out[first:new, :g]
            if bad != bad:
                assert bool(hit.isnan().all()), (lens, which)
            else:
                assert bool((hit == bad).all()), (lens, which, bad)
            if which == 2:
                out[first:new, :g, 5] = clean[first:new, :g, 5]
            else:
                out[first:new, :g] = clean[first:new, :g]
            assert torch.equal(out, clean), (lens, which, bad)


# ---- refusals ----

def test_paged_refusals_of_tensors(cuda):
    ext = ops.ext()
    x = rope_inputs(3, 16, 2, 128, 16, torch.float16, 0)
    q = torch.empty(3, 16, 128, dtype=torch.float16, device="cuda")

    def rope(**k):
        a = dict(zip(("qkv", "qw", "kw", "pos", "inv", "slots", "kc", "vc"), x), q=q, hq=16, hkv=2)
        a.update(k)
        ext.norm_rope_paged(a["qkv"], a["qw"], a["kw"], 1e-6, a["pos"], a["inv"], a["slots"], a["q"], a["kc"], a["vc"], a["hq"], a["hkv"])

    rope()
    for bad in (dict(qkv=x[0].float()), dict(qkv=x[0][:, :-8]), dict(qkv=x[0].t()), dict(qw=None), dict(qw=x[1].float()),
                dict(kw=x[2][:64]), dict(pos=x[3].int()), dict(pos=x[3][:2]), dict(inv=x[4].double()), dict(slots=x[5].cpu()),
                dict(q=q[:2]), dict(q=q.bfloat16()), dict(kc=x[6].bfloat16()), dict(vc=x[7][:1]), dict(kc=x[6].transpose(0, 2)),
                dict(hkv=1), dict(hq=3), dict(inv=None), dict(kc=x[6][:, :, :8].contiguous(), vc=x[7][:, :, :8].contiguous()),
                dict(qkv=torch.zeros(3, 2564, dtype=torch.float16, device="cuda")[:, :2560])):
        with pytest.raises(RuntimeError):
            rope(**bad)
    y = batch([(2, 40), (1, 17)], 16, 2, 128, 16, torch.float16, 0)

    def attend(**k):
        a = dict(zip(("q", "kc", "vc", "table", "starts", "lens"), y), out=torch.empty_like(y[0]), new=2, keys=40)
        a.update(k)
        ext.attention_paged(a["q"], a["kc"], a["vc"], a["table"], a["starts"], a["lens"], a["out"], a["new"], a["keys"], 0.1)

    attend()
    for bad in (dict(q=y[0].float()), dict(q=y[0].bfloat16()), dict(q=y[0][:, :15]), dict(q=y[0].transpose(0, 1)), dict(kc=y[1].bfloat16()),
                dict(vc=y[2][1:]), dict(table=y[3].long()), dict(table=y[3][:1]), dict(table=y[3][:, ::2]), dict(starts=y[4].long()),
                dict(starts=y[4][:2]), dict(lens=y[5][:1]), dict(lens=y[5].cpu()), dict(out=y[0][:2]), dict(out=torch.empty(3, 2048, dtype=torch.float16, device="cuda")),
                dict(new=0), dict(keys=0), dict(q=y[0][:, :, :96].contiguous())):
        with pytest.raises(RuntimeError):
            attend(**bad)
    # nothing to do is no error
    ext.attention_paged(y[0][:0], *y[1:6], y[0][:0], 1, 1, 0.1)
    ext.norm_rope_paged(x[0][:0], x[1], x[2], 1e-6, x[3][:0], x[4], x[5][:0], q[:0], x[6], x[7], 16, 2)

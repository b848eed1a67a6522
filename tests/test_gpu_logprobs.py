"""token_logprobs on the GPU against log_softmax in 64 bits, at row lengths and starts around its vectors and workgroups, with
ties, -inf, NaN and rows without a distribution.

Bounds. The row's sums are of V terms in (0, 1] in 32 bits: added in at most V / 64 + 64 steps along any path, each term good
to 4 * 2^-24 (the difference from the maximum, the exponential). The sum, its logarithm lz (at most log V) and the entropy's
second sum, of terms p (x - max), are good to r = (V / 64 + 80) 2^-24 relatively; a difference x - max is good to 2^-24 of
itself, and the exponential of d to 2^-24 |d|, which the entropy's sum weights by p: at most 40 2^-24 there (p |d| d < 1 ...
the terms with |d| > 40 are below 2^-57). A sum off by r relatively moves its logarithm by r absolutely (log(z (1 + r)) =
log z + r - ..), however small the logarithm is: a row with one likely token has z = 1 + a little, and 1 itself is rounded
to 2^-24. So: log probability r + 2^-24 (|x - max| + 3 lz + |logp|); entropy r + 2 r E + 2^-24 (|H| + 3 lz), E the second
sum over the first."""
import math

import pytest
import torch

from lowbit import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def want(x, targets, top):
    """In 64 bits: log probabilities, entropy and alternatives by (value falling, index rising), and the bounds."""
    d = x.double()
    mx = d.amax(-1, keepdim=True)
    low = d - mx
    p = low.exp()
    z = p.sum(-1, keepdim=True)
    lz = z.log()
    second = -(torch.where(p > 0, p * low, torch.zeros_like(p))).sum(-1, keepdim=True) / z
    entropy = (lz + second)[:, 0]
    t = targets.clamp(0, x.shape[1] - 1)
    at = low.gather(1, t[:, None])
    value, ids = torch.sort(d + 0.0, dim=-1, descending=True, stable=True)
    ids = ids[:, :top]
    r = (x.shape[1] / 64 + 80) * U
    bound = lambda l: r + U * (l.abs() + 3 * lz + (l - lz).abs())
    logp = (at - lz)[:, 0]
    return (logp, bound(at)[:, 0], entropy, (r + 2 * r * second + U * (second.abs() + 4 * lz))[:, 0],
            low.gather(1, ids) - lz, bound(low.gather(1, ids)), ids)


def close(got, exact, bound):
    """Within the bound; infinities and NaN where the exact value has them."""
    got = got.double()
    same = (got == exact) | (got.isnan() & exact.isnan())
    return bool((same | ((got - exact).abs() <= bound)).all())


def check(x, targets, top):
    before = x.clone()
    lp, ent, tv, ti = ops.ext().token_logprobs(x, targets, top)
    wl, bl, we, be, wv, bv, wi = want(x, targets, top)
    assert lp.dtype is torch.float32 and ent.dtype is torch.float32 and tv.dtype is torch.float32 and ti.dtype is torch.int64
    asked, inside = targets >= 0, targets < x.shape[1]
    assert bool((lp[~asked] == 0).all()) and bool(lp[~inside].isnan().all())
    assert close(lp[asked & inside], wl[asked & inside], bl[asked & inside])
    assert close(ent, we, be), (ent.double() - we).abs().max()
    assert torch.equal(ti, wi), (ti != wi).nonzero()[:4].tolist()
    assert close(tv, wv, bv)
    assert torch.equal(x.view(torch.uint8) if x.is_contiguous() else x.nan_to_num(), before.view(torch.uint8) if x.is_contiguous() else before.nan_to_num())
    return lp, ent, tv, ti


def logits(m, v, dt, seed, sd=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (sd * torch.randn(m, v, generator=g, device="cuda")).to(dt)
    return x, torch.randint(0, v, (m,), generator=g, device="cuda")


TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m,v", [(1, 1), (1, 2), (3, 7), (2, 8), (5, 9), (1, 63), (4, 64), (2, 65), (3, 511), (2, 1000), (1, 4096),
                                 (300, 1025), (2, 8191), (7, 32000), (1, 50257), (1, 151936), (3, 151665), (17, 151936),
                                 (520, 20011), (1100, 700)])
def test_logprobs(cuda, m, v, dt):
    x, t = logits(m, v, dt, m + v)
    for top in sorted({0, 1, min(5, v), min(20, v), min(32, v)}):
        one = check(x, t, top)
        assert all(torch.equal(a, b) for a, b in zip(one, check(x, t, top)))


@pytest.mark.parametrize("dt", TYPES)
def test_logprobs_of_rows_at_any_start(cuda, dt):
    """Rows that start anywhere in a 16-byte piece, apart from each other, and one row read for all."""
    for shift in range(9):
        x, t = logits(6, 3001, dt, shift)
        check(x[:, shift:2900 + shift], t.clamp(max=2899), 9)
        check(x[1:, shift:], t[1:].clamp(max=3000 - shift), 9)
    x, t = logits(1, 5000, dt, 3)
    check(x.expand(7, 5000), t.expand(7).contiguous(), 4)
    check(logits(9, 40000, dt, 4)[0][::3], torch.zeros(3, dtype=torch.long, device="cuda"), 4)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m,v", [(1, 151936), (4, 3000), (600, 2500)])
def test_logprobs_ties_go_to_the_lower_index(cuda, m, v, dt):
    x, t = logits(m, v, dt, 1)
    check(torch.zeros_like(x), t, 32)                       # every logit the same
    check((x * 0.7).round(), t, 32)                         # whole numbers
    y = torch.full_like(x, -2.0)
    y[:, v // 2:] = 1.0                                     # many more equal largest ones than alternatives
    check(y, t, 20)
    y[:, v // 3], y[:, v // 3 + 1] = 0.0, -0.0
    y[:, v // 2:] = -1.0
    check(y, t, 5)
    y[:, -1] = 3.0
    check(y, t, 32)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("order", ["rising", "falling", "block"])
def test_logprobs_sorted_rows(cuda, dt, order):
    """The largest values side by side, where few lanes hold all of them, growing or falling along the row."""
    v = 151936
    x = torch.linspace(-20, 20, v, device="cuda", dtype=torch.float32)
    if order == "falling":
        x = x.flip(0)
    if order == "block":
        x = torch.cat([x[:1000], x[-40:], x[1000:-40]])
    rows = torch.stack([x, x.roll(777)]).to(dt)
    check(rows, torch.tensor([5, v - 1], device="cuda"), 32)
    check(rows[:1], torch.tensor([v // 2], device="cuda"), 32)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m,v", [(2, 151936), (5, 999), (700, 1500)])
def test_logprobs_of_masked_rows(cuda, dt, m, v):
    """Banned tokens at -inf or the type's lowest value, down to one that is left; rows far above and below zero."""
    x, t = logits(m, v, dt, 2)
    for keep in (3, 40, v // 2):
        y = torch.full_like(x, -math.inf)
        y[:, 5:5 + keep] = x[:, 5:5 + keep]
        check(y, t, 32)
        y[y == -math.inf] = torch.finfo(dt).min
        check(y, t, 8)
    y = torch.full_like(x, -math.inf)
    y[:, v - 1] = 7.0
    lp, ent, *_ = check(y, torch.full_like(t, v - 1), 3)
    assert bool((lp == 0).all()) and bool((ent == 0).all())
    for shift in (3e4, -3e4):
        check((x.float() + shift).to(dt), t, 8)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m,v", [(3, 151936), (4, 100), (530, 1300)])
def test_logprobs_of_rows_without_a_distribution(cuda, dt, m, v):
    x, t = logits(m, v, dt, 5)
    x[0] = -math.inf
    x[1, 17] = math.inf
    x[2, v - 2] = math.nan
    x[2, 3] = math.nan
    lp, ent, tv, ti = ops.ext().token_logprobs(x, t, 6)
    for r in range(3):
        assert bool(lp[r].isnan()) and bool(ent[r].isnan()) and bool(tv[r].isnan().all())
    assert ti[0].tolist() == [0, 1, 2, 3, 4, 5] and int(ti[1, 0]) == 17 and ti[2, :2].tolist() == [3, v - 2]
    check(x[3:], t[3:], 6)
    none = t.clone()
    none[:] = -100
    assert bool((ops.ext().token_logprobs(x, none)[0] == 0).all())


def test_logprobs_targets(cuda):
    x, t = logits(6, 5000, torch.float16, 6)
    t[:5] = torch.tensor([-1, -100, 5000, 4999, 0], device="cuda")
    t[5] = 1 << 40
    check(x, t, 2)


def test_logprobs_past_32_bits(cuda):
    """A row that starts past 2^32 values, in a tensor of which only two rows are written."""
    big = torch.empty((1 << 32) // 8192 + 3, 8192, dtype=torch.float16, device="cuda")
    x, t = logits(2, 8192, torch.float16, 7)
    big[0], big[-1] = x[0], x[1]
    check(big[::big.shape[0] - 1], t, 5)


@pytest.mark.parametrize("m", [1, 5, 700])
def test_logprobs_captured(cuda, m):
    x, t = logits(m, 50000, torch.float16, 8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.ext().token_logprobs(x, t, 7)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = ops.ext().token_logprobs(x, t, 7)
    for seed in (8, 9, 10, 8):
        a, b = logits(m, 50000, torch.float16, seed)
        x.copy_(a)
        t.copy_(b)
        eager = ops.ext().token_logprobs(x, t, 7)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager))


def test_logprobs_on_two_streams(cuda):
    data = [logits(2, 151936, torch.float16, s) for s in (1, 2)]
    exact = [ops.ext().token_logprobs(*d, 10) for d in data]
    streams = [torch.cuda.Stream() for _ in data]
    torch.cuda.synchronize()
    results = []
    for _ in range(20):
        for d, s in zip(data, streams):
            with torch.cuda.stream(s):
                results.append(ops.ext().token_logprobs(*d, 10))
    torch.cuda.synchronize()
    for i, r in enumerate(results):
        assert all(torch.equal(a, b) for a, b in zip(r, exact[i % 2]))


def test_logprobs_refusals(cuda):
    x, t = logits(4, 100, torch.float16, 0)
    for args in ((x.double(), t), (x[0], t), (x, t[:3]), (x, t.int()), (x, t.cpu()), (x, t, 33), (x, t, -1), (x[:, :5], t, 6),
                 (x.t(), torch.zeros(100, dtype=torch.long, device="cuda")), (x[:, ::2], t), (x[:, :0], t)):
        with pytest.raises(RuntimeError):
            ops.ext().token_logprobs(*args)
    lp, ent, tv, ti = ops.ext().token_logprobs(x[:0], t[:0], 3)
    assert lp.shape == (0,) and ent.shape == (0,) and tv.shape == (0, 3) and ti.shape == (0, 3)

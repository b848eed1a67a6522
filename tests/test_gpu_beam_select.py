"""beam_select on the GPU against its definition in 64 bits: which beams and tokens, in which order, and their scores.

A score is score + (x - max) - log z with z summed in 32 bits: about V / 512 sequential additions a lane and the joins' cost at most
(V / 512 + 80) 2^-24 of z, typically its root; the exponentials are off by at most |x - max| 2^-23 of themselves, of which those that
matter lie within 20 of the maximum. So log z is off by at most E = (V / 512 + 80 + 40) 2^-24, and a score by E and its own rounding,
2^-24 of it. Two beams' candidates have to come in order where their exact scores differ by more, so inputs whose order is tested
give a request's beams the same logits and scores a little off the types' grids, by more than what rounds; equal ones are tested
with beams of equal scores and equal logits at the same alignment, whose sums are the same bits."""
import math

import pytest
import torch

from lowbit import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def exact(logits, scores, n, finished=None, pad=0):
    """(scores, beams, tokens) by a stable sort of all candidates in 64 bits."""
    requests, beams = scores.shape
    v = logits.shape[1]
    x = logits.double().view(requests, beams, v)
    top = x.amax(-1, keepdim=True)
    lse = (x - top).exp().sum(-1, keepdim=True).log()
    value = scores.double()[:, :, None] + ((x - top) - lse)
    value = torch.where(torch.isfinite(scores)[:, :, None] & torch.isfinite(lse), value, torch.full_like(value, -math.inf))
    if finished is not None:
        done = torch.full_like(value, -math.inf)
        done[:, :, pad] = torch.where(torch.isfinite(scores), scores.double(), torch.full_like(scores, -math.inf).double())
        value = torch.where(finished[:, :, None], done, value)
    value, at = torch.sort(value.view(requests, -1), dim=1, descending=True, stable=True)
    return value[:, :n], at[:, :n] // v, at[:, :n] % v


def check(logits, scores, n, finished=None, pad=0, order=True):
    v = logits.shape[1]
    want, beam, token = exact(logits, scores, n, finished, pad)
    got = ops.ext().beam_select(logits, scores, n, finished, pad)
    torch.cuda.synchronize()
    err = (v / 512 + 120) * U
    same = (got[0].double() == want) | ((got[0].double() - want).abs() <= err + U * want.abs())
    assert bool(same.all()), (got[0][~same][:4], want[~same][:4])
    if order:
        assert torch.equal(got[1], beam), (got[1] != beam).nonzero()[:4]
        assert torch.equal(got[2], token), (got[2] != token).nonzero()[:4]
    again = ops.ext().beam_select(logits, scores, n, finished, pad)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    return got


def inputs(requests, beams, v, dt, seed, std=2.2):
    """Logits of a few likely tokens a row, the same for a request's beams. Scores are multiples of 1/8 and 2^-14 for each beam
    before (64 beams: 2^-8, below the 16-bit types' steps at the likely logits): no two candidates of different beams tie."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(requests, 1, v, generator=g, device="cuda") * std - 2
    likely = torch.randint(0, v, (requests, 1, min(12, v)), generator=g, device="cuda")
    x.scatter_add_(2, likely, 5.0 + 5.0 * torch.rand(likely.shape, generator=g, device="cuda"))
    x = x.expand(-1, beams, -1)
    scores = -torch.randint(0, 40, (requests, beams), generator=g, device="cuda").float() / 8
    scores = scores - torch.arange(beams, device="cuda").float() * 2.0 ** -14
    return x.reshape(-1, v).to(dt).contiguous(), scores


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("requests,beams,v,n", [(1, 1, 1000, 1), (1, 4, 151936, 8), (3, 2, 32000, 32), (2, 16, 4096, 32), (9, 5, 20000, 5),
                                                (1, 64, 2048, 32), (600, 1, 4096, 3), (5, 8, 512, 16), (40, 4, 8192, 8)])
def test_beams(cuda, requests, beams, v, n, dt):
    x, scores = inputs(requests, beams, v, dt, requests + v)
    check(x, scores, n)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("requests,beams,v,n", [(1, 3, 151665, 6), (4, 5, 32001, 10), (2, 7, 2049, 14), (33, 2, 4099, 4)])
def test_rows_of_different_logits(cuda, requests, beams, v, n, dt):
    """Every row has its own logits, at any alignment: the scores, and that each is the one of its beam and token."""
    g = torch.Generator(device="cuda").manual_seed(v)
    x = (torch.randn(requests * beams, v, generator=g, device="cuda") * 2.5).to(dt)
    scores = -10 * torch.rand(requests, beams, generator=g, device="cuda")
    got = check(x, scores, n, order=False)
    lse = torch.logsumexp(x.double(), -1).view(requests, beams)
    own = scores.double().gather(1, got[1]) + x.double().view(requests, -1).gather(1, got[1] * v + got[2]) - lse.gather(1, got[1])
    assert bool(((own - got[0].double()).abs() <= (v / 512 + 120) * U + U * own.abs()).all())
    flat = got[1] * v + got[2]
    assert all(len(set(r)) == n for r in flat.tolist())


@pytest.mark.parametrize("v", [1, 2, 3, 7, 8, 31, 33, 64])
def test_small_vocabularies(cuda, v):
    """Fewer tokens than places, than lanes, than a vector holds."""
    for dt in (torch.float16, torch.float32):
        for beams in (1, 2, 5):
            for n in {1, min(3, beams * v), min(32, beams * v)}:
                x, scores = inputs(3, beams, v, dt, v + beams)
                scores = -torch.arange(beams, device="cuda").float().expand(3, -1).contiguous() * 0.2503
                check(x, scores, n)


def test_ties(cuda):
    """All logits equal; all equal but a few; two values; scores that make rows tie: by beam, then by token."""
    for v in (96, 4096, 50000):
        for dt in (torch.float16, torch.float32):
            x = torch.zeros(6, v, dtype=dt, device="cuda")
            check(x, torch.zeros(2, 3, device="cuda"), 9)
            x[:, v - 1] = 3
            check(x, torch.zeros(2, 3, device="cuda"), 32)
            x[:, ::2] = -1
            check(x, torch.tensor([[0.0, -1.3, 0.0], [-2.1, 0.0, -2.1]], device="cuda"), 20)
            x.copy_(torch.linspace(-5, 5, v, device="cuda").to(dt))
            check(x, torch.zeros(2, 3, device="cuda"), 20)


def test_beams_that_hold_nothing(cuda):
    """The first step: one beam of each request has a score, the others -inf; then requests of which none has one."""
    x, scores = inputs(4, 4, 5000, torch.float16, 1)
    scores[:, 1:] = -math.inf
    check(x, scores, 8)
    scores[1] = -math.inf
    got = check(x, scores, 8)
    assert got[2][1].tolist() == list(range(8)) and bool((got[1][1] == 0).all()) and bool((got[0][1] == -math.inf).all())
    scores[2, 0], scores[3, 0] = math.nan, math.inf
    got = check(x, scores, 8)
    assert bool((got[0][2:] == -math.inf).all())


@pytest.mark.parametrize("pad", [0, 3, 4999])
def test_finished_beams(cuda, pad):
    """A finished beam is one candidate; where all are, the places behind them are -inf."""
    x, scores = inputs(6, 4, 5000, torch.bfloat16, 2)
    scores = -torch.tensor([0.5003, 1.2571, 7.0311, 30.007], device="cuda").expand(6, -1).contiguous()
    finished = torch.zeros(6, 4, dtype=torch.bool, device="cuda")
    finished[1, 0] = finished[2, :3] = finished[3] = True
    finished[4, 1] = finished[4, 3] = True
    got = check(x, scores, 8, finished, pad)
    assert got[2][3, :4].tolist() == [pad] * 4 and got[1][3, :4].tolist() == [0, 1, 2, 3]
    scores[4, 1] = -math.inf                                  # finished, and nothing held
    check(x, scores, 8, finished, pad)


def test_masked_and_odd_logits(cuda):
    """Tokens at -inf or the type's lowest value, rows of those alone, rows with a NaN or an infinity."""
    for dt in (torch.float16, torch.bfloat16, torch.float32):
        for v in (300, 9000):
            x, _ = inputs(8, 2, v, dt, 3)
            scores = torch.tensor([[0.0, -0.5003]], device="cuda").expand(8, -1).contiguous()
            x[0] = -math.inf                                  # no distribution
            x[2, 5:] = -math.inf                              # five tokens left
            x[3, 1:] = -math.inf
            x[4, :v // 2] = torch.finfo(dt).min
            x[6, v // 3] = math.nan
            x[8, v - 1] = math.inf
            x[10], x[11] = math.nan, -math.inf
            x[12] = torch.finfo(dt).min
            x[13] = torch.finfo(dt).max
            x[14, 0], x[14, v - 1] = -0.0, 0.0
            check(x, scores, 12)


def test_strides_and_streams(cuda):
    """Rows that lie apart, rows that are one row, a view that starts at an odd address."""
    base, scores = inputs(3, 4, 6001, torch.float16, 5)
    wide = torch.empty(12, 7003, dtype=torch.float16, device="cuda").fill_(99.0)
    wide[:, 1:6002] = base
    a = check(wide[:, 1:6002], scores, 8)
    one = base[:1].expand(12, -1)
    check(one, scores, 8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = ops.ext().beam_select(wide[:, 1:6002], scores, 8)
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_captured(cuda):
    x, scores = inputs(2, 4, 30000, torch.float16, 6)
    finished = torch.zeros(2, 4, dtype=torch.bool, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.ext().beam_select(x, scores, 8, finished, 2)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = ops.ext().beam_select(x, scores, 8, finished, 2)
    for seed in (7, 8, 9, 7):
        y, t = inputs(2, 4, 30000, torch.float16, seed)
        x.copy_(y)
        scores.copy_(t)
        finished[0, seed % 4] = True
        graph.replay()
        eager = check(x, scores, 8, finished, 2)
        assert all(torch.equal(a, b) for a, b in zip(got, eager))
    # no requests: empty answers
    empty = ops.ext().beam_select(x[:0], scores[:0], 8)
    assert [tuple(t.shape) for t in empty] == [(0, 8)] * 3

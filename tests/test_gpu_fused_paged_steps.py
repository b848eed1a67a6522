"""FusedQwen2.forward_paged in a captured step, and steps that ask for no logits or hold no token.

Bound as in test_gpu_fused_paged.py; a replay has the bits of the eager step."""
import pytest
import torch

from lowbit import _native, decode, fused
from test_gpu_fused_paged import Pages, rel

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("quant", ["int4", "fp16", "fp16_gemv"])
def test_a_captured_step_serves_other_batches(cuda, quant):
    """A step of 8 tokens and 3 sequences captured once: decode tokens, pieces of prompts and drafts with padded tokens behind
    them, on changing tables, each against the eager step and each sequence alone."""
    model = fused.FusedQwen2(decode.random_model("tiny", seed=6), 64, quant)
    gen = torch.Generator(device="cuda").manual_seed(3)
    texts = [torch.randint(0, 1024, (n,), generator=gen, device="cuda") for n in (23, 9, 17)]
    want = [model(t, torch.arange(t.shape[0], device="cuda")).clone() for t in texts]
    caches, eager_caches = model.paged_caches(16, 16), model.paged_caches(16, 16)
    i64, i32 = dict(dtype=torch.int64, device="cuda"), dict(dtype=torch.int32, device="cuda")
    fixed = (torch.zeros(8, **i64), torch.zeros(8, **i64), torch.full((8,), -1, **i64), torch.zeros(3, 4, **i32),
             torch.zeros(4, **i32), torch.zeros(3, **i32))
    call = lambda c: model.forward_paged(*fixed, c, 8, 64)
    side = _native.capture_stream(cuda)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(caches)
        call(caches)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = call(caches)
    pool, done = Pages(16, 16, 3, 4), [0, 0, 0]
    for news in ((8, 0, 0), (3, 1, 4), (1, 1, 1), (0, 7, 1), (5, 0, 3), (6, 0, 2), (0, 0, 6)):
        tokens = torch.cat([t[d:d + n] for t, d, n in zip(texts, done, news)])
        positions, slots, table, starts, lens = pool.step(news)
        n = tokens.shape[0]
        for f, x in zip(fixed, (tokens, positions, slots, table, starts, lens)):
            f.fill_(-1) if f is fixed[2] else f.zero_()
            f[:x.shape[0]] = x
        eager = call(eager_caches)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[:n], eager[:n])
        assert torch.equal(caches[0], eager_caches[0]) and torch.equal(caches[1], eager_caches[1])
        for b, k in enumerate(news):
            if k:
                assert rel(got[int(starts[b]):int(starts[b]) + k], want[b][done[b]:done[b] + k]) < 1e-2, (news, b)
            done[b] += k


@pytest.mark.parametrize("quant", ["int4", "fp16"])
def test_steps_without_logits_or_tokens(cuda, quant):
    model = fused.FusedQwen2(decode.random_model("tiny", seed=6), 64, quant)
    tokens = torch.randint(0, 1024, (20,), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    pool = Pages(8, 16, 1, 4)
    step = pool.step((20,))
    a, b = model.paged_caches(8, 16), model.paged_caches(8, 16)
    full = model.forward_paged(tokens, *step, a, 20, 20)
    none = model.forward_paged(tokens, *step, b, 20, 20, rows=torch.empty(0, dtype=torch.long, device="cuda"))
    assert none.shape == (0, full.shape[1]) and none.dtype is full.dtype
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])              # the keys are written all the same
    empty = model.forward_paged(tokens[:0], step[0][:0], step[1][:0], step[2], torch.zeros(2, dtype=torch.int32, device="cuda"),
                                step[4], b, 1, 20)
    assert empty.shape == (0, full.shape[1])
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])

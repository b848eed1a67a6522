"""FusedQwen2 over paged caches: a batch whose prompts arrive in pieces together with decode tokens of others, against the
forward over one sequence's own contiguous cache, and the scores of a text.

Bound: the two forwards share the projections; the rotation (64-bit angles and one rounding against fp16 cos and sin) and the
attention round differently, a few steps of 2^-11 of the values in each of two layers, whose sum stays under 1e-2 of the
logits' norm."""
import pytest
import torch

from lowbit import decode, fused, ops

pytestmark = pytest.mark.gpu


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


class Pages:
    """Hands out pages of a pool at random and keeps each sequence's table."""

    def __init__(self, pages, size, sequences, width, seed=0):
        self.free = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
        self.size, self.table, self.lens = size, torch.zeros(sequences, width, dtype=torch.int32), [0] * sequences

    def step(self, news):
        """Rows for news[b] new tokens of every sequence: what forward_paged takes (on the GPU)."""
        positions, slots, starts = [], [], [0]
        for b, n in enumerate(news):
            for p in range(self.lens[b], self.lens[b] + n):
                if p % self.size == 0:
                    self.table[b, p // self.size] = self.free.pop()
                positions.append(p)
                slots.append(int(self.table[b, p // self.size]) * self.size + p % self.size)
            self.lens[b] += n
            starts.append(starts[-1] + n)
        i32 = dict(dtype=torch.int32, device="cuda")
        return (torch.tensor(positions, device="cuda"), torch.tensor(slots, device="cuda"), self.table.cuda(),
                torch.tensor(starts, **i32), torch.tensor(self.lens, **i32))


@pytest.mark.parametrize("quant", ["int4", "fp16", "fp16_gemv"])
@pytest.mark.parametrize("page", [16, 64])
def test_paged_batch_matches_each_sequence_alone(cuda, quant, page):
    model = fused.FusedQwen2(decode.random_model("tiny", seed=3), 512, quant)
    gen = torch.Generator(device="cuda").manual_seed(page)
    texts = [torch.randint(0, 1024, (n,), generator=gen, device="cuda") for n in (150, 37, 301)]
    want = [model(t, torch.arange(t.shape[0], device="cuda")).clone() for t in texts]
    # pieces of the three texts: prompts together, a prompt's piece with decode tokens, decode tokens alone, a pause
    steps = [(100, 20, 1), (1, 1, 250), (48, 0, 1), (1, 1, 1), (0, 15, 48)]
    pool = Pages(64, page, 3, 32)
    caches = model.paged_caches(64, page)
    done = [0, 0, 0]
    for news in steps:
        tokens = torch.cat([t[d:d + n] for t, d, n in zip(texts, done, news)])
        positions, slots, table, starts, lens = pool.step(news)
        got = model.forward_paged(tokens, positions, slots, table, starts, lens, caches, max(news), max(pool.lens))
        last = model.forward_paged(tokens, positions, slots, table, starts, lens, caches, max(news), max(pool.lens),
                                   rows=starts[1:].long() - 1) if all(news) else None
        for b, n in enumerate(news):
            rows = slice(int(starts[b]), int(starts[b + 1]))
            if n:
                assert rel(got[rows], want[b][done[b]:done[b] + n]) < 1e-2, (news, b)
            if last is not None:                            # the same step again: the same keys are written
                assert rel(last[b], want[b][done[b] + n - 1]) < 1e-2
            done[b] += n
    assert done == [150, 37, 301]


def test_paged_batch_with_padded_rows(cuda):
    """Tokens behind the last sequence, with slots of -1: the others' logits and caches are as without them."""
    model = fused.FusedQwen2(decode.random_model("tiny", seed=4), 64, "int4")
    gen = torch.Generator(device="cuda").manual_seed(1)
    tokens = torch.randint(0, 1024, (12,), generator=gen, device="cuda")
    pool = Pages(8, 16, 2, 4)
    positions, slots, table, starts, lens = pool.step((5, 7))
    a, b = model.paged_caches(8, 16), model.paged_caches(8, 16)
    want = model.forward_paged(tokens, positions, slots, table, starts, lens, a, 7, 7)
    pad = lambda t, v: torch.cat([t, torch.full((3,), v, device="cuda", dtype=t.dtype)])
    got = model.forward_paged(pad(tokens, 0), pad(positions, 0), pad(slots, -1), table, starts, lens, b, 7, 7)
    assert rel(got[:12], want) < 1e-2 and bool(got.isfinite().all())
    assert rel(b[0], a[0]) < 1e-2 and torch.equal(b[0] == 0, a[0] == 0)


@pytest.mark.parametrize("quant", ["int4", "fp16"])
def test_score_of_a_text(cuda, quant):
    model = fused.FusedQwen2(decode.random_model("tiny", seed=5), 256, quant)
    tokens = torch.randint(0, 1024, (90,), generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    logp, entropy, values, ids = model.score(tokens, 4)
    logits = model(tokens, torch.arange(90, device="cuda"))[:-1]
    for got, want in zip((logp, entropy, values, ids), ops.ext().token_logprobs(logits, tokens[1:].contiguous(), 4)):
        assert torch.equal(got, want)
    exact = torch.log_softmax(logits.double(), -1)
    assert float((logp.double() - exact.gather(1, tokens[1:, None])[:, 0]).abs().max()) < 1e-5
    assert torch.equal(ids[:, 0], logits.argmax(-1)) and logp.shape == entropy.shape == (89,) and ids.shape == values.shape == (89, 4)

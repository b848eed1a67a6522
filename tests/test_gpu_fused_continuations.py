"""FusedQwen2 with several continuations of a request: trees of drafted tokens verified step by step against greedy decoding, and beam
search against one that runs every beam's whole text through the forward over a contiguous cache.

Bound: as in test_gpu_fused_paged.py the two forwards' logits differ by under 1e-2 of their norm; `near` is that of the logits at
hand (their root mean square times 1e-2, times 8 for the largest of 1024)."""
import random

import pytest
import torch

from lowbit import _native, decode, fused, ops

from test_gpu_fused_paged import rel

pytestmark = pytest.mark.gpu


def near(logits):
    return 8e-2 * float(logits.double().pow(2).mean().sqrt())


def alone(model, text):
    return model(text, torch.arange(text.shape[0], device="cuda"))


def drafts(truth, at, nodes, rng, vocab):
    """A tree below truth[at]: most nodes carry what really follows, some another token, some twice the same."""
    tokens, parents, depth = [int(truth[at])], [-1], [0]
    while len(tokens) < nodes:
        p = rng.choice([len(tokens) - 1, rng.randrange(len(tokens))])
        right = int(truth[min(at + depth[p] + 1, len(truth) - 1)])
        tokens.append(right if rng.random() < 0.6 else rng.randrange(vocab))
        parents.append(p)
        depth.append(depth[p] + 1)
    return tokens, parents


@pytest.mark.parametrize("quant", ["int4", "fp16"])
@pytest.mark.parametrize("captured", [False, True])
def test_trees_give_the_greedy_text(cuda, quant, captured):
    model = fused.FusedQwen2(decode.random_model("tiny", seed=7), 256, quant)
    rng, size, width, pages, longest, most = random.Random(1), 16, 16, 40, 6, 24
    gen = torch.Generator(device="cuda").manual_seed(4)
    texts = [torch.randint(0, 1024, (n,), generator=gen, device="cuda") for n in (21, 33, 16)]
    # what greedy decoding over the contiguous cache makes of them, to draft from
    truth = []
    for t in texts:
        for _ in range(30):
            t = torch.cat([t, alone(model, t)[-1].argmax(-1, keepdim=True)])
        truth.append(t)
    caches = model.paged_caches(pages, size)
    i32 = dict(dtype=torch.int32, device="cuda")
    table = torch.full((3, width), -1, **i32)
    step = ops.ext().plan_paged(table, torch.zeros(3, **i32), torch.tensor([t.shape[0] - 1 for t in texts], **i32),
                                sum(t.shape[0] - 1 for t in texts), pages, size, out=table)
    model.forward_paged(torch.cat([t[:-1] for t in texts]), step.positions, step.slots, table, step.q_starts, step.kv_lens, caches, 40,
                        40, rows=step.q_starts[:0].long())
    total = 3 * most
    tokens, parents = torch.zeros(total, dtype=torch.int64, device="cuda"), torch.full((total,), -1, **i32)
    past, new = torch.tensor([t.shape[0] - 1 for t in texts], **i32), torch.zeros(3, **i32)
    run = lambda: model.verify_trees(tokens, parents, table, past, new, caches, most, 256, longest)   # noqa: E731
    graph = None
    if captured:
        side = _native.capture_stream(torch.device("cuda", 0))
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run()                                           # (no new tokens: nothing is written)
            run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = run()
    said = [t.tolist() for t in texts]
    for turn in range(6):
        flat, above, sizes = [], [], []
        for b in range(3):
            n = rng.choice([1, 2, 9, most])
            t, p = drafts(truth[b], len(said[b]) - 1, n, rng, 1024)
            t[0] = said[b][-1]
            flat, above = flat + t, above + p
            sizes.append(n)
        pad = total - len(flat)
        tokens.copy_(torch.tensor(flat + [0] * pad, device="cuda"))
        parents.copy_(torch.tensor(above + [-1] * pad, **i32))
        new.copy_(torch.tensor(sizes, **i32))
        if captured:
            graph.replay()
        else:
            got = run()
        accepted, counts, lens, missing = got
        torch.cuda.synchronize()
        assert int(missing) == 0
        for b in range(3):
            n = int(counts[b])
            assert 1 <= n <= min(longest, sizes[b])
            assert int(lens[b]) == len(said[b]) - 1 + n
            fresh = accepted[b, :n].tolist()
            ref = alone(model, torch.tensor(said[b] + fresh[:-1], device="cuda"))[-n:].double()
            for i, t in enumerate(fresh):                   # every token the greedy one, as far as the two forwards agree
                assert float(ref[i, t]) >= float(ref[i].max()) - near(ref)
            said[b] += fresh
            # the keys kept are the text's
            keys = int(lens[b])
            j = torch.arange(keys, device="cuda")
            where = table[b].long()[j // size]
            for paged, plain in zip(caches, (model.k_cache, model.v_cache)):
                assert rel(paged[:, where, :, j % size].transpose(0, 1), plain[:, :, :keys].transpose(1, 2)) < 1e-2
        past.copy_(lens)
    assert min(len(a) - t.shape[0] for a, t in zip(said, texts)) >= 6
    assert max(len(a) - t.shape[0] for a, t in zip(said, texts)) > 8   # (drafts are confirmed: more than a token a step)


def plain_search(model, prompt, beams, steps, eos):
    """Beam search over whole texts in 64 bits: [(score, tokens)], best first."""
    alive = [(0.0, [])]
    for _ in range(steps):
        options = []
        for w, (score, text) in enumerate(alive):
            if text and text[-1] == eos:
                options.append((-score, w, eos))
                continue
            logp = torch.log_softmax(alone(model, torch.cat([prompt, torch.tensor(text, dtype=torch.int64, device="cuda")]))[-1].double(), -1)
            best, ids = torch.sort(logp, descending=True, stable=True)
            options += [(-(score + float(v)), w, int(i)) for v, i in zip(best[:beams], ids[:beams])]
        options.sort()
        alive = [(-s, alive[w][1] + [t]) for s, w, t in options[:beams]]
    return alive


@pytest.mark.parametrize("quant", ["int4", "fp16"])
@pytest.mark.parametrize("beams,page_size", [(1, 16), (4, 16), (3, 64), (8, 16)])
def test_beam_search(cuda, quant, beams, page_size):
    """The scores are those of the plain search's beams as far as the two forwards agree (an error of the logits changes a
    token's log probability by at most twice `near`, and a beam's by that for each step), and each beam's score is its text's."""
    model = fused.FusedQwen2(decode.random_model("tiny", seed=8), 128, quant)
    gen = torch.Generator(device="cuda").manual_seed(beams)
    prompts = [torch.randint(0, 1024, (n,), generator=gen, device="cuda") for n in (15, 40, 1)]
    steps, eos = 7, None
    tokens, scores = model.beam_search(prompts, beams, steps, page_size=page_size)
    assert tokens.shape == (3, beams, steps) and scores.shape == (3, beams)
    for r, prompt in enumerate(prompts):
        tol = 2 * steps * near(alone(model, prompt))
        want = plain_search(model, prompt, beams, steps, eos)
        assert bool((scores[r, :-1] >= scores[r, 1:]).all())
        for w in range(beams):
            assert abs(float(scores[r, w]) - want[w][0]) <= tol
            text = torch.cat([prompt, tokens[r, w]])
            logp = torch.log_softmax(alone(model, text)[:-1].double(), -1).gather(1, text[1:, None])[-steps:, 0]
            assert abs(float(scores[r, w]) - float(logp.sum())) <= tol
        assert len({tuple(t) for t in tokens[r].tolist()}) == beams


def test_beam_search_ends_beams(cuda):
    """A token that is likely after many texts as the end: beams that took it stay as they are, eos behind it."""
    model = fused.FusedQwen2(decode.random_model("tiny", seed=9), 128, "int4")
    prompt = torch.randint(0, 1024, (20,), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    free, _ = model.beam_search([prompt], 4, 6)
    eos = int(free[0, 0, 2])
    tokens, scores = model.beam_search([prompt, prompt[:9]], 4, 6, eos=eos)
    ended = 0
    for r, p in enumerate((prompt, prompt[:9])):
        tol = 12 * near(alone(model, p))
        for w in range(4):
            t = tokens[r, w].tolist()
            n = t.index(eos) + 1 if eos in t else 6
            ended += n < 6
            assert t[n:] == [eos] * (6 - n)
            text = torch.cat([p, tokens[r, w, :n]])
            logp = torch.log_softmax(alone(model, text)[:-1].double(), -1).gather(1, text[1:, None])[-n:, 0]
            assert abs(float(scores[r, w]) - float(logp.sum())) <= tol
    assert ended > 0


def test_refusals(cuda):
    model = fused.FusedQwen2(decode.random_model("tiny", seed=9), 64, "fp16")
    one = torch.zeros(1, dtype=torch.int64, device="cuda")
    for prompts, beams, steps in (([], 2, 3), ([one[:0]], 2, 3), ([one], 0, 3), ([one], 33, 3), ([one], 2, 0)):
        with pytest.raises(ValueError):
            model.beam_search(prompts, beams, steps)

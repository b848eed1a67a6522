"""FusedQwen2.verify_trees where the cache runs out of pages: what a sequence has is kept, and the step can be made again when pages
are free."""
import pytest
import torch

from lowbit import decode, fused, ops

from test_gpu_fused_continuations import alone, near
from test_gpu_fused_paged import rel

pytestmark = pytest.mark.gpu

SIZE, WIDTH = 16, 8
I32 = dict(dtype=torch.int32, device="cuda")


def i32(x):
    return torch.tensor(x, **I32)


def start(model, lens, pages, seed):
    """Texts of `lens` tokens, all keys but the last token's in the first pages of a cache of `pages`, their table and lengths."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    texts = [torch.randint(0, 1024, (n,), generator=gen, device="cuda") for n in lens]
    caches, table = model.paged_caches(pages, SIZE), torch.full((len(lens), WIDTH), -1, **I32)
    fresh = [n - 1 for n in lens]
    step = ops.ext().plan_paged(table, torch.zeros_like(i32(fresh)), i32(fresh), sum(fresh), pages, SIZE, out=table)
    assert int(step.missing) == 0
    model.forward_paged(torch.cat([t[:-1] for t in texts]), step.positions, step.slots, table, step.q_starts, step.kv_lens, caches,
                        max(fresh), max(fresh), rows=step.q_starts[:0].long())
    return texts, caches, table, i32(fresh)


def chain(model, text, nodes):
    """A chain of `nodes` drafts that greedy decoding over the contiguous cache confirms: text's last token and what follows."""
    t = text
    for _ in range(nodes):
        t = torch.cat([t, alone(model, t)[-1].argmax(-1, keepdim=True)])
    return t[len(text) - 1:]


def step_of(model, trees, table, past, caches, longest=32):
    """verify_trees over chains; a sequence without one pauses."""
    sizes = [len(t) for t in trees]
    parents = i32([i - 1 for n in sizes for i in range(n)])
    return model.verify_trees(torch.cat([t for t in trees if len(t)]), parents, table, past, i32(sizes), caches, max(sizes), 128, longest)


def keys_of(caches, table, b, keys):
    j = torch.arange(keys, device="cuda")
    return [c[:, table[b].long()[j // SIZE], :, j % SIZE].transpose(0, 1) for c in caches]


def greedy(model, text, fresh):
    """Whether each of `fresh` is the greedy token after what comes before it, as far as two forwards agree."""
    ref = alone(model, torch.cat([text, fresh[:-1]]))[-len(fresh):].double()
    return all(float(ref[i, int(t)]) >= float(ref[i].max()) - near(ref) for i, t in enumerate(fresh))


def test_a_page_that_cannot_be_copied_stays(cuda):
    """Two sequences on the same 20 keys, whose second page both would write, and no free page for a copy: the second one's row still
    names the page, its keys are still there, and with a page it goes on."""
    model = fused.FusedQwen2(decode.random_model("tiny", seed=11), 128, "fp16")
    texts, caches, table, past = start(model, [21, 17], 3, 5)
    other = table[1, 0].clone()                              # (16 keys of a third sequence, which ends below)
    table = torch.stack([table[0], table[0], table[1]])
    past = torch.stack([past[0], past[0], past[1]])
    before, empty = table.clone(), texts[0][:0]
    drafts = chain(model, texts[0], 4)[:4]
    accepted, counts, lens, missing = step_of(model, [drafts, drafts, empty], table, past, caches)
    assert int(missing) == 1
    assert torch.equal(table[:, :2], before[:, :2])
    alone(model, texts[0][:20])
    for got, plain in zip(keys_of(caches, table, 1, 20), (model.k_cache, model.v_cache)):
        assert rel(got, plain[:, :, :20].transpose(1, 2)) < 1e-2
    past = torch.stack([lens[0], past[1], torch.zeros_like(past[2])])
    accepted, counts, lens, missing = step_of(model, [accepted[0, counts[0] - 1:counts[0]], drafts, empty], table, past, caches)
    assert int(missing) == 0 and int(table[1, 1]) == int(other)
    assert int(counts[1]) == 4 and greedy(model, texts[0], accepted[1, :4])


def test_a_step_short_of_pages(cuda):
    """Three sequences that want six pages of two: the first gets them, the second keeps what fits its last page, the third nothing. When
    the first has ended, the others go on, and every key is the text's."""
    model = fused.FusedQwen2(decode.random_model("tiny", seed=12), 128, "int4")
    texts, caches, table, past = start(model, [14, 15, 17], 5, 6)
    nodes, longest = 20, 32
    accepted, counts, lens, missing = step_of(model, [chain(model, t, nodes)[:nodes] for t in texts], table, past, caches, longest)
    assert int(missing) == 4
    assert 1 <= int(counts[0]) <= nodes and 1 <= int(counts[1]) <= 2 and int(counts[2]) == 0
    assert lens.tolist() == [13 + int(counts[0]), 14 + int(counts[1]), 16]
    assert accepted[2].tolist() == [-1] * longest
    for turn in range(2):
        for b in range(3):
            fresh = accepted[b, :int(counts[b])]
            if len(fresh):
                assert greedy(model, texts[b], fresh)
                texts[b] = torch.cat([texts[b], fresh])
            assert int(lens[b]) == len(texts[b]) - 1 or (turn and b == 0)
            if turn and b == 0:
                continue
            alone(model, texts[b])
            for got, plain in zip(keys_of(caches, table, b, int(lens[b])), (model.k_cache, model.v_cache)):
                assert rel(got, plain[:, :, :int(lens[b])].transpose(1, 2)) < 1e-2
        if turn:
            break
        past = torch.stack([torch.zeros_like(lens[0]), lens[1], lens[2]])
        trees = [texts[0][:0]] + [chain(model, t, 9)[:9] for t in texts[1:]]
        accepted, counts, lens, missing = step_of(model, trees, table, past, caches, longest)
        assert int(missing) == 0 and counts.tolist()[0] == 0 and min(counts.tolist()[1:]) >= 1

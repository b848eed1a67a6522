"""The operators behind several continuations of one request over the paged KV cache, through the entry points a user's
program calls (own) or in their plain form (elementary torch operations, rounded once at the end): beams, and trees of drafted
tokens that a step verifies together.

Every case is a dict of plain values with a "kind":

    plan     ops.ext().plan_paged(...)            the tables of a step from its sequences' lengths: `chunks` sequences with
                                                  `new_lo` .. `new_hi` new tokens and `ones` sequences with one, each on
                                                  `past_lo` .. `past_hi` cached ones; `tree`: the new tokens are draft trees
    reorder  ops.ext().plan_paged(rows=...)       a beam step's tables: `beams` continuations of each of `requests` prompts go on
                                                  from the rows that were selected; pages that two of them would write are copied
                                                  in all `layers`
    tree     ops.ext().attention_paged_tree(...)  `seqs` sequences' trees of `new_lo` .. `new_hi` drafted tokens over their pages
    accept   ops.ext().accept_drafts(...)         the drafted tokens that the model's own picks confirm, their rows of the cache
                                                  moved together in all `layers`
    beam     ops.ext().beam_select(...)           the `n` best continuations of `requests` x `beams` rows of logits

Cache layout: [layers, pages, KV heads, page size, head dim]; row r of page p is slot p * page size + r.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
SIZE = {"float16": 2, "bfloat16": 2, "float32": 4}


def listed():
    return [
        # the tables of one request's draft tree: launch and host latency
        {"name": "plan_tree_1", "kind": "plan", "chunks": 1, "new_lo": 26, "new_hi": 26, "ones": 0, "past_lo": 700,
         "past_hi": 700, "page": 64, "tree": True, "pad": 0},
        # a full server's step: decode tokens of 250 requests and pieces of six prompts, padded to a captured step's size
        {"name": "plan_256", "kind": "plan", "chunks": 6, "new_lo": 100, "new_hi": 1500, "ones": 250, "past_lo": 300,
         "past_hi": 30000, "page": 16, "tree": False, "pad": 300},
        # a beam step of 16 requests: half of the beams give way to others, whose last page they share until now
        {"name": "reorder_128", "kind": "reorder", "requests": 16, "beams": 8, "prompt_lo": 100, "prompt_hi": 2000,
         "made_lo": 1, "made_hi": 200, "layers": 28, "hkv": 2, "dim": 128, "page": 16, "dtype": "float16"},
        # one request's draft tree on a short context
        {"name": "tree_1", "kind": "tree", "seqs": 1, "new_lo": 26, "new_hi": 26, "past_lo": 900, "past_hi": 900, "hq": 16,
         "hkv": 2, "dim": 128, "page": 64, "dtype": "float16"},
        # a batch of requests' trees, contexts that differ
        {"name": "tree_16", "kind": "tree", "seqs": 16, "new_lo": 31, "new_hi": 63, "past_lo": 300, "past_hi": 8000, "hq": 28,
         "hkv": 4, "dim": 128, "page": 16, "dtype": "bfloat16"},
        # two trees on long documents
        {"name": "tree_long", "kind": "tree", "seqs": 2, "new_lo": 40, "new_hi": 48, "past_lo": 30000, "past_hi": 60000,
         "hq": 28, "hkv": 4, "dim": 128, "page": 64, "dtype": "float16"},
        # wide trees (several words of mask a token), heads of 64
        {"name": "tree_wide", "kind": "tree", "seqs": 8, "new_lo": 90, "new_hi": 250, "past_lo": 100, "past_hi": 4000, "hq": 14,
         "hkv": 2, "dim": 64, "page": 32, "dtype": "float16"},
        # one request's tree verified: latency
        {"name": "accept_1", "kind": "accept", "seqs": 1, "new_lo": 26, "new_hi": 26, "past_lo": 900, "past_hi": 900,
         "layers": 36, "hkv": 2, "dim": 128, "page": 64, "dtype": "float16"},
        # a batch's trees verified
        {"name": "accept_64", "kind": "accept", "seqs": 64, "new_lo": 31, "new_hi": 63, "past_lo": 100, "past_hi": 1000,
         "layers": 28, "hkv": 4, "dim": 128, "page": 16, "dtype": "bfloat16"},
        # one request's first beam step: all but one of the beams hold nothing yet
        {"name": "beam_1x4", "kind": "beam", "requests": 1, "beams": 4, "vocab": 151936, "n": 8, "dtype": "float16",
         "first": True, "done": 0.0},
        # several requests, logits in fp32, a vocabulary whose rows do not start on 16 bytes
        {"name": "beam_9x5", "kind": "beam", "requests": 9, "beams": 5, "vocab": 151665, "n": 5, "dtype": "float32",
         "first": False, "done": 0.2},
        # a full batch of wide beams
        {"name": "beam_64x8", "kind": "beam", "requests": 64, "beams": 8, "vocab": 151936, "n": 16, "dtype": "float16",
         "first": False, "done": 0.1},
    ]


def _spread(rng, lo, hi):
    """A whole number from lo .. hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = [(12, 2, 128), (16, 2, 128), (28, 4, 128), (32, 8, 128), (14, 2, 64), (8, 8, 64), (8, 1, 128)]
MOST_READ = 120_000 * 4 * 128                               # keys x KV heads x head dim of a drawn batch of trees
MOST_CACHE = 280_000_000                                    # values of a drawn cache


def draw(rng):
    kind = rng.choice(["plan", "reorder", "tree", "tree", "tree", "accept", "beam", "beam"])
    if kind == "beam":
        requests, beams = _spread(rng, 1, 60), rng.choice([1, 2, 3, 4, 5, 8, 16])
        vocab = _spread(rng, 1000, min(152000, 500 * 151936 // (2 * requests * beams)))
        return {"kind": kind, "requests": requests, "beams": beams, "vocab": vocab, "n": rng.choice([beams, 2 * beams]),
                "dtype": rng.choice(sorted(DTYPES)), "first": rng.random() < 0.2, "done": rng.choice([0.0, 0.1, 0.6])}
    page = rng.choice([16, 32, 64, 128])
    if kind == "plan":
        past_hi = _spread(rng, 1, 30000)
        if rng.random() < 0.4:
            return {"kind": kind, "chunks": _spread(rng, 1, 200), "new_lo": rng.choice([1, 8, 30]),
                    "new_hi": rng.choice([31, 64, 130]), "ones": rng.choice([0, 3]), "past_lo": max(1, past_hi // 9),
                    "past_hi": past_hi, "page": page, "tree": True, "pad": rng.choice([0, 17])}
        return {"kind": kind, "chunks": rng.choice([0, 1, 5]), "new_lo": 9, "new_hi": _spread(rng, 9, 1500),
                "ones": _spread(rng, 1, 240), "past_lo": max(1, past_hi // 9), "past_hi": past_hi, "page": page, "tree": False,
                "pad": rng.choice([0, 1, 200])}
    hq, hkv, dim = rng.choice(HEADS)
    half = rng.choice(["float16", "bfloat16"])
    if kind == "reorder":
        requests, beams = _spread(rng, 1, 14), rng.choice([2, 3, 4, 5, 8, 16])
        prompt, made = _spread(rng, 16, 1500), _spread(rng, 1, 150)
        rows = requests * (prompt + beams * (made + 3 * page))
        layers = max(1, min(rng.choice([1, 24, 28, 36]), MOST_CACHE // (2 * rows * hkv * dim)))
        return {"kind": kind, "requests": requests, "beams": beams, "prompt_lo": max(1, prompt // 4), "prompt_hi": prompt,
                "made_lo": max(1, made // 4), "made_hi": made, "layers": layers, "hkv": hkv, "dim": dim, "page": page,
                "dtype": half}
    seqs = _spread(rng, 1, 60)
    new_hi = _spread(rng, 2, 250 if kind == "tree" and rng.random() < 0.3 else 64)
    shape = {"kind": kind, "seqs": seqs, "new_lo": max(1, new_hi // rng.choice([1, 2, 8])), "new_hi": new_hi}
    if kind == "tree":
        most = max(65, min(MOST_READ // (hkv * dim * seqs), 9_000_000_000 // (seqs * new_hi * hq * dim) * 2))
        past_hi = _spread(rng, 1, min(60000, most))
        return {**shape, "past_lo": max(1, past_hi // rng.choice([1, 4, 20])), "past_hi": past_hi, "hq": hq, "hkv": hkv, "dim": dim,
                "page": page, "dtype": half}
    past_hi = _spread(rng, 1, 800)
    layers = max(1, min(rng.choice([24, 28, 36]), MOST_CACHE // (2 * seqs * (past_hi + new_hi + 3 * page) * hkv * dim)))
    return {**shape, "past_lo": max(1, past_hi // 4), "past_hi": past_hi, "layers": layers, "hkv": hkv, "dim": dim, "page": page,
            "dtype": half}


# ---- inputs, from the seed alone; lengths and trees belong to the case, not to the seed ----

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(1000003 * int(seed) + 71)


def _normal(shape, gen, std=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * std).to(dtype)


def _noise(shape, gen, dtype):
    """Values for a cache: quick to make, as many as there are."""
    x = torch.empty(shape, dtype=dtype, device="cuda")
    return x.uniform_(-1.7, 1.7, generator=gen)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _rng(case):
    return random.Random(" ".join("%s=%s" % (k, case[k]) for k in sorted(case) if k != "name"))


def _lengths(case):
    """(new tokens, cached tokens) of every sequence."""
    rng = _rng(case)

    def past():
        return _spread(rng, case["past_lo"], case["past_hi"])

    chunks = case["seqs"] if "seqs" in case else case["chunks"]
    pairs = [(_spread(rng, case["new_lo"], case["new_hi"]), past()) for _ in range(chunks)]
    pairs += [(1, past()) for _ in range(case.get("ones", 0))]
    rng.shuffle(pairs)
    return pairs


def _tree(nodes, rng):
    """Parents of a draft tree's nodes: node 0 is the token chosen last, each other one hangs below an earlier one, most of
    them within the first few levels, as drafted trees are."""
    parents, depth = [-1], [0]
    for i in range(1, nodes):
        p = min(rng.randrange(i), rng.randrange(i)) if rng.random() < 0.6 else i - 1
        while depth[p] >= 8:
            p = parents[p]
        parents.append(p)
        depth.append(depth[p] + 1)
    return parents


def _trees(case):
    rng = _rng(case)
    return [_tree(n, rng) for n, _ in _lengths(case)]


def _starts(lens):
    starts = [0]
    for n, _ in lens:
        starts.append(starts[-1] + n)
    return starts


def _words(lens):
    return max(1, -(-max(n for n, _ in lens) // 64))


def _tables(held, pages, width, gen):
    """A table whose rows hold `held` pages each, all different, in no order; -1 behind them."""
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    count = _ints(held, torch.long)
    ends = count.cumsum(0)
    col = torch.arange(width, device="cuda")
    at = (ends - count)[:, None] + col
    return torch.where(col < count[:, None], order[at.clamp(max=pages - 1)], -1).to(torch.int32).contiguous()


def _plan_inputs(case, seed):
    gen, page = _gen(seed), case["page"]
    lens = _lengths(case)
    held = [-(-p // page) for _, p in lens]
    need = [-(-(p + n) // page) for n, p in lens]
    pages, width = sum(need) + sum(need) // 8 + 5, max(need) + 3
    table = _tables(held, pages, width, gen)
    s = {"table": table, "past": _ints([p for _, p in lens]), "new": _ints([n for n, _ in lens]), "pages": pages,
         "tokens": sum(n for n, _ in lens) + case["pad"], "words": _words(lens), "parents": None}
    if case["tree"]:
        s["parents"] = _ints([p for t in _trees(case) for p in t] + [-1] * case["pad"])
    return s


def _reorder_inputs(case, seed):
    gen, page, beams = _gen(seed), case["page"], case["beams"]
    rng, choose = _rng(case), random.Random(1000003 * int(seed) + 5)
    rows, past, held, at = [], [], [], 0
    for r in range(case["requests"]):
        prompt = _spread(rng, case["prompt_lo"], case["prompt_hi"])
        made = _spread(rng, case["made_lo"], case["made_hi"])
        shared = prompt // page                             # full pages of the prompt, one copy for all beams
        own_pages = -(-(prompt + made) // page) - shared
        prefix = list(range(at, at + shared))
        at += shared
        for b in range(beams):
            held.append(prefix + list(range(at, at + own_pages)))
            at += own_pages
            past.append(prompt + made)
            rows.append(r * beams + (b if choose.random() < 0.5 else choose.randrange(beams)))
    pages, width = at + 2 * len(rows) + 7, max(len(h) for h in held) + 2
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    index = _ints([h + [-1] * (width - len(h)) for h in held], torch.long)
    table = torch.where(index >= 0, order[index.clamp(min=0)], -1).to(torch.int32)
    shape = (case["layers"], pages, case["hkv"], page, case["dim"])
    k, v = _noise(shape, gen, DTYPES[case["dtype"]]), _noise(shape, gen, DTYPES[case["dtype"]])
    return {"table": table, "past": _ints(past), "new": _ints([1] * len(rows)), "pages": pages, "tokens": len(rows), "words": 1,
            "parents": None, "rows": _ints(rows), "caches": (k, v)}


def _tree_inputs(case, seed):
    gen, dt, page = _gen(seed), DTYPES[case["dtype"]], case["page"]
    hq, hkv, dim = case["hq"], case["hkv"], case["dim"]
    lens = _lengths(case)
    need = [-(-(p + n) // page) for n, p in lens]
    pages = sum(need) + 3
    table = _tables(need, pages, max(need), gen).clamp(min=0)
    q = _normal((sum(n for n, _ in lens), hq, dim), gen, 1.5, dt)
    k, v = _normal((pages, hkv, page, dim), gen, 1.0, dt), _normal((pages, hkv, page, dim), gen, 1.0, dt)
    return lens, q, k, v, table


def _mask_words(case):
    """The masks as the plan of the step makes them: bit i of a token's words for node i of its sequence, itself and its
    ancestors."""
    words, rows = _words(_lengths(case)), []
    for parents in _trees(case):
        bits = []
        for i, p in enumerate(parents):
            bits.append((1 << i) | (bits[p] if p >= 0 else 0))
        rows += bits
    signed = [[((b >> (64 * w)) & (2 ** 64 - 1)) for w in range(words)] for b in rows]
    return _ints([[x - 2 ** 64 if x >= 2 ** 63 else x for x in r] for r in signed], torch.int64)


def _accept_inputs(case, seed):
    gen, page = _gen(seed), case["page"]
    choose = random.Random(1000003 * int(seed) + 7)
    lens, trees = _lengths(case), _trees(case)
    need = [-(-(p + n) // page) for n, p in lens]
    pages = sum(need) + 3
    table = _tables(need, pages, max(need) + 1, gen)
    tokens, picks, parents = [], [], []
    for tree in trees:
        # drafted tokens; the model picks other ones but along the way to one node, a draft that it confirms
        drafted = [choose.randrange(151000) for _ in tree]
        picked = [151000 + choose.randrange(900) for _ in tree]
        node = choose.randrange(len(tree))
        while node > 0:
            picked[tree[node]] = drafted[node]
            node = tree[node]
        tokens += drafted
        picks += picked
        parents += tree
    shape = (case["layers"], pages, case["hkv"], page, case["dim"])
    return {"lens": lens, "table": table, "tokens": _ints(tokens, torch.int64), "picks": _ints(picks, torch.int64),
            "parents": _ints(parents), "q_starts": _ints(_starts(lens)), "kv_lens": _ints([n + p for n, p in lens]),
            "longest": 9, "caches": (_noise(shape, gen, DTYPES[case["dtype"]]), _noise(shape, gen, DTYPES[case["dtype"]]))}


def _beam_inputs(case, seed):
    """Logits as a language model's: most of the vocabulary far below a few likely tokens."""
    gen, requests, beams, vocab = _gen(seed), case["requests"], case["beams"], case["vocab"]
    rows = requests * beams
    x = _normal((rows, vocab), gen, 2.2)
    x -= 2.0
    likely = torch.randint(0, vocab, (rows, 12), generator=gen, device="cuda")
    x.scatter_add_(1, likely, 6.0 + 5.0 * torch.rand(rows, 12, generator=gen, device="cuda"))
    scores = -30.0 * torch.rand(requests, 1, generator=gen, device="cuda") \
        - 4.0 * torch.rand(requests, beams, generator=gen, device="cuda")
    finished = torch.rand(requests, beams, generator=gen, device="cuda") < case["done"]
    if case["first"]:
        x = x.view(requests, beams, vocab)
        x = x[:, :1].expand(-1, beams, -1).reshape(rows, vocab)   # the prompt's, the same for every beam
        scores = torch.full_like(scores, -math.inf)
        scores[:, 0] = 0.0
        finished.zero_()
    return x.to(DTYPES[case["dtype"]]).contiguous(), scores, finished


def prepare(case, seed):
    kind, state = case["kind"], {"case": case}
    if kind == "plan":
        state.update(_plan_inputs(case, seed), rows=None, caches=None)
        state["table_out"] = torch.empty_like(state["table"])
    elif kind == "reorder":
        state.update(_reorder_inputs(case, seed))
        state["table_out"] = torch.empty_like(state["table"])
    elif kind == "tree":
        lens, q, k, v, table = _tree_inputs(case, seed)
        state.update(lens=lens, starts=_starts(lens), q=q, k=k, v=v, table=table, out=torch.empty_like(q),
                     q_starts=_ints(_starts(lens)), kv_lens=_ints([n + p for n, p in lens]), masks=_mask_words(case),
                     max_new=max(n for n, _ in lens), max_keys=max(n + p for n, p in lens))
    elif kind == "accept":
        state.update(_accept_inputs(case, seed))
    else:
        state["logits"], state["scores"], state["finished"] = _beam_inputs(case, seed)
    if own:
        package = os.path.join(os.getcwd(), "lowbit-kernels_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
        from lowbit import ops
        state["ext"] = ops.ext()
    return state


# ---- one pass ----

def _plain_plan(s):
    page, pages, tokens = s["case"]["page"], s["pages"], s["tokens"]
    rows = torch.arange(s["new"].shape[0], device="cuda") if s["rows"] is None else s["rows"].long()
    table, past, new = s["table"].long()[rows], s["past"].long()[rows], s["new"].long()
    batch, width = table.shape
    col, b = torch.arange(width, device="cuda"), torch.arange(batch, device="cuda")
    have, need = (past + page - 1) // page, (past + new + page - 1) // page
    # pages in use, and those that a sequence would write and another one reads
    kept = col < have[:, None]
    used = torch.zeros(pages + 1, dtype=torch.bool, device="cuda")
    used[torch.where(kept, table, pages)] = True
    whole = torch.zeros_like(used)
    whole[torch.where(col < (past // page)[:, None], table, pages)] = True
    part = past % page > 0
    tail = torch.where(part, table.gather(1, (have - 1).clamp(min=0)[:, None])[:, 0], pages)
    writes = part & (new > 0)
    other = (tail[:, None] == tail) & (b[:, None] != b)
    first = (past > past[:, None]) | ((past == past[:, None]) & (b < b[:, None]) & writes)
    whole[pages] = False
    copy = writes & (whole[tail] | (other & first).any(1))
    # free pages in order, to the sequences in order
    want = need - have + copy
    upto = want.cumsum(0)
    free = torch.cat([torch.nonzero(~used[:pages])[:, 0], torch.full((batch * width + batch,), -1, device="cuda")])
    from_free = (upto - want + copy)[:, None] + (col - have[:, None]).clamp(min=0)
    table = torch.where(kept, table, torch.where(col < need[:, None], free[from_free], -1))
    target = free[(upto - want).clamp(min=0)]
    at = torch.where(copy, have - 1, width)
    table = torch.cat([table, table[:, :1]], 1).scatter(1, at[:, None], target[:, None])[:, :width]
    missing = (upto[-1:] - (~used[:pages]).sum()).clamp(min=0)
    # tokens
    ends = new.cumsum(0)
    t = torch.arange(tokens, device="cuda")
    seq = torch.searchsorted(ends, t, right=True).clamp(max=batch - 1)
    i = t - (ends - new)[seq]
    real = t < ends[-1]
    key = past[seq] + i
    slot = table[seq, (key // page).clamp(max=width - 1)]
    slots = torch.where(real & (slot >= 0), slot * page + key % page, -1)
    out = [table.to(torch.int32), torch.cat([torch.zeros_like(ends[:1]), ends]).to(torch.int32), (past + new).to(torch.int32)]
    if s["parents"] is None:
        out += [torch.where(real, key, 0), slots]
    else:
        # ancestors by doubling: a token has its own bit and those of what lies above it
        above = s["parents"].long()
        above = torch.where(above >= 0, above + t - i, t)
        depth = (above != t).long()
        bits = torch.zeros(tokens, 64 * s["words"], dtype=torch.bool, device="cuda")
        bits[t, i.clamp(max=bits.shape[1] - 1)] = real
        for _ in range(max(1, (bits.shape[1] - 1).bit_length())):
            bits, depth, above = bits | bits[above], depth + depth[above], above[above]
        bit = torch.ones(64, dtype=torch.int64, device="cuda") << torch.arange(64, device="cuda")
        masks = (bits.view(tokens, -1, 64) * bit).sum(-1)
        out += [torch.where(real, past[seq] + depth, 0), slots, masks]
    copies = torch.where(copy[:, None], torch.stack([tail, target], 1), -1).to(torch.int32)
    out += [copies, missing.to(torch.int32)]
    if s["caches"] is not None:
        at, row = copies[:, 0].long(), torch.arange(page, device="cuda")
        ok = (copy & (target >= 0))[:, None] & (row < (past % page)[:, None])
        which, r = torch.nonzero(ok, as_tuple=True)
        for c in s["caches"]:
            c[:, copies[which, 1].long(), :, r] = c[:, at[which], :, r]
        out += list(s["caches"])
    return out


def _plain_tree(s):
    case = s["case"]
    hq, hkv, dim, page = (case[k] for k in ("hq", "hkv", "dim", "page"))
    per, scale = hq // hkv, dim ** -0.5
    bit = torch.ones(64, dtype=torch.int64, device="cuda") << torch.arange(64, device="cuda")
    for b, (new, past) in enumerate(s["lens"]):
        keys, first = past + new, s["starts"][b]
        at = s["table"][b, :-(-keys // page)].long()
        k = s["k"][at].transpose(0, 1).reshape(hkv, -1, dim)[:, :keys].float()
        v = s["v"][at].transpose(0, 1).reshape(hkv, -1, dim)[:, :keys].float()
        q = s["q"][first:first + new].float().view(new, hkv, per, dim).transpose(0, 1).reshape(hkv, new * per, dim)
        x = torch.matmul(q, k.transpose(1, 2).contiguous()) * scale
        seen = ((s["masks"][first:first + new, :, None] & bit) != 0).view(new, -1)[:, :new].repeat_interleave(per, 0)
        x[:, :, past:] = x[:, :, past:].masked_fill(~seen, -math.inf)
        p = (x - x.amax(-1, keepdim=True)).exp()
        o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
        s["out"][first:first + new] = o.view(hkv, new, per, dim).transpose(0, 1).reshape(new, hq, dim).to(s["out"].dtype)
    return s["out"]


def _plain_accept(s):
    page, longest = s["case"]["page"], s["longest"]
    starts, kv = s["q_starts"].long(), s["kv_lens"].long()
    new = starts[1:] - starts[:-1]
    batch, nodes = new.shape[0], int(max(n for n, _ in s["lens"]))
    node = torch.arange(nodes, device="cuda")
    at = (starts[:-1, None] + node).clamp(max=s["tokens"].shape[0] - 1)
    there = node < new[:, None]
    token = torch.where(there, s["tokens"][at], -1)
    parent = torch.where(there, s["parents"].long()[at], -2)
    pick = s["picks"][at]
    path = torch.full((batch, longest), -1, dtype=torch.long, device="cuda")
    cur, alive = torch.zeros(batch, dtype=torch.long, device="cuda"), new > 0
    last = cur
    for d in range(longest):
        path[:, d] = torch.where(alive, cur, -1)
        last = torch.where(alive, cur, last)
        hit = (parent == cur[:, None]) & (token == pick.gather(1, cur[:, None])) & (node > cur[:, None])
        alive = alive & hit.any(1)
        cur = torch.where(alive, hit.long().argmax(1), cur)
    count = (path >= 0).sum(1)
    step = torch.arange(longest, device="cuda")
    said = torch.where(path >= 0, pick.gather(1, path.clamp(min=0)), -1)   # a confirmed node's token is its parent's pick
    past = kv - new
    src, dst = past[:, None] + path, past[:, None] + step
    b, d = torch.nonzero((path >= 0) & (src != dst), as_tuple=True)
    src, dst = src[b, d], dst[b, d]
    table = s["table"].long()
    for c in s["caches"]:
        c[:, table[b, dst // page], :, dst % page] = c[:, table[b, src // page], :, src % page]
    return (path.to(torch.int32), count.to(torch.int32), said, (past + count).to(torch.int32)) + s["caches"]


def _order(x):
    """x as whole numbers in its order (-0 as +0)."""
    bits = (x + 0.0).view(torch.int32)
    return torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)


def _plain_beam(s):
    case = s["case"]
    requests, beams, vocab, n = (case[k] for k in ("requests", "beams", "vocab", "n"))
    x = s["logits"].float()
    # a row's n likeliest, equal ones by index; scores in 64 bits, since which of two rows' tokens comes first goes by them
    key = (_order(x).long() << 32) + (vocab - 1 - torch.arange(vocab, device="cuda"))
    ids = vocab - 1 - (torch.topk(key, n, dim=-1)[0] & 0xFFFFFFFF)
    top = x.amax(-1, keepdim=True)
    lse = (x.double() - top).exp().sum(-1, keepdim=True).log() + top
    value = s["scores"].double().view(-1, 1) + (x.gather(1, ids).double() - lse)
    # a beam that holds nothing has every token at -inf, a finished one its score for the token 0
    ids = torch.where(torch.isfinite(s["scores"]).view(-1, 1) & ~s["finished"].view(-1, 1), ids, torch.arange(n, device="cuda"))
    done = torch.full_like(value, -math.inf)
    done[:, 0] = s["scores"].double().view(-1)
    value = torch.where(s["finished"].view(-1, 1), done, value).view(requests, beams * n)
    best, at = torch.sort(value, dim=1, descending=True, stable=True)
    at = at[:, :n]
    return best[:, :n].float(), at // n, ids.view(requests, beams * n).gather(1, at)


def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if not own:
        return {"plan": _plain_plan, "reorder": _plain_plan, "tree": _plain_tree, "accept": _plain_accept,
                "beam": _plain_beam}[kind](state)
    ext = state["ext"]
    if kind in ("plan", "reorder"):
        step = ext.plan_paged(state["table"], state["past"], state["new"], state["tokens"], state["pages"], case["page"],
                              rows=state["rows"], parents=state["parents"], words=state["words"], caches=state["caches"],
                              out=state["table_out"])
        out = [step.page_table, step.q_starts, step.kv_lens, step.positions, step.slots]
        if state["parents"] is not None:
            out.append(step.masks)
        out += [step.copies, step.missing]
        return out + list(state["caches"] or ())
    if kind == "tree":
        ext.attention_paged_tree(state["q"], state["k"], state["v"], state["table"], state["q_starts"], state["kv_lens"],
                                 state["masks"], state["out"], state["max_new"], state["max_keys"], case["dim"] ** -0.5)
        return state["out"]
    if kind == "accept":
        return ext.accept_drafts(state["tokens"], state["picks"], state["parents"], state["q_starts"], state["kv_lens"],
                                 state["table"], state["caches"], state["longest"]) + state["caches"]
    return ext.beam_select(state["logits"], state["scores"], case["n"], state["finished"], 0)


# ---- what a pass cannot do without ----

def work(case):
    kind = case["kind"]
    if kind == "plan":
        lens, page = _lengths(case), case["page"]
        tokens = sum(n for n, _ in lens)
        held, need = sum(-(-p // page) for _, p in lens), sum(-(-(p + n) // page) for n, p in lens)
        width = max(-(-(p + n) // page) for n, p in lens) + 3
        tree = (4 + 8 * _words(lens)) * tokens if case["tree"] else 0
        return {"bytes": 4 * held + 4 * len(lens) * width + 16 * (tokens + case["pad"]) + 16 * len(lens) + tree,
                "flops": 2 * need + 4 * tokens}
    if kind == "reorder":
        s = case["requests"] * case["beams"]
        # about a third of the beams get a copy of half a page
        row = 2 * case["layers"] * case["hkv"] * case["dim"] * SIZE[case["dtype"]]
        mean = -(-(case["prompt_hi"] + case["made_hi"]) // (2 * case["page"]))
        return {"bytes": 2 * row * (s // 3) * (case["page"] // 2) + 8 * s * mean + 40 * s, "flops": 8 * s * mean}
    if kind == "tree":
        lens, size = _lengths(case), SIZE[case["dtype"]]
        rows, keys = sum(n for n, _ in lens), sum(n + p for n, p in lens)
        pairs = sum(n * p for n, p in lens) + sum(bin(m).count("1") for m in _bits(case))
        pages = sum(-(-(n + p) // case["page"]) for n, p in lens)
        return {"bytes": 2 * rows * case["hq"] * case["dim"] * size + 2 * keys * case["hkv"] * case["dim"] * size
                + 4 * pages + 8 * len(lens) + 8 * rows * _words(lens),
                "flops": 4 * pairs * case["hq"] * case["dim"]}
    if kind == "accept":
        lens = _lengths(case)
        row = 2 * case["layers"] * case["hkv"] * case["dim"] * SIZE[case["dtype"]]
        depth = sum(_depths(t) for t in _trees(case))       # the mean over the node that is confirmed
        return {"bytes": int(2 * row * depth) + 20 * sum(n for n, _ in lens) + (4 + 8) * 9 * len(lens),
                "flops": sum(n for n, _ in lens)}
    live = case["requests"] if case["first"] else case["requests"] * case["beams"] * (1.0 - case["done"])
    n = int(live * case["vocab"])
    return {"bytes": n * SIZE[case["dtype"]] + case["requests"] * (5 * case["beams"] + 20 * case["n"]), "flops": 4 * n}


def _bits(case):
    masks = []
    for parents in _trees(case):
        bits = []
        for i, p in enumerate(parents):
            bits.append((1 << i) | (bits[p] if p >= 0 else 0))
        masks += bits
    return masks


def _depths(parents):
    depth = []
    for p in parents:
        depth.append(0 if p < 0 else depth[p] + 1)
    return sum(depth) / len(depth)


# ---- the same from the definitions, in 64 bits ----

def _exact_plan(case, seed):
    s = _plan_inputs(case, seed) if case["kind"] == "plan" else _reorder_inputs(case, seed)
    page = case["page"]
    table, past, new = s["table"].tolist(), s["past"].tolist(), s["new"].tolist()
    rows = s["rows"].tolist() if case["kind"] == "reorder" else list(range(len(new)))
    past = [past[r] for r in rows]
    kept = [table[r][:-(-past[b] // page)] for b, r in enumerate(rows)]
    readers = {}
    for b, held in enumerate(kept):
        for p in held:
            readers.setdefault(p, []).append(b)
    free = iter([p for p in range(s["pages"]) if p not in readers])
    copies, moved = [], []
    for b, held in enumerate(kept):
        pair = [-1, -1]
        if past[b] % page and new[b]:
            others = [c for c in readers[held[-1]] if c != b]
            # it may write where nobody reads on: the others end where it does, and come after it or write nothing
            if any(past[c] > past[b] or len(kept[c]) != len(held) or (past[c] == past[b] and c < b and new[c]) for c in others):
                pair = [held[-1], next(free)]
                moved.append((b, pair[0], pair[1], past[b] % page))
        copies.append(pair)
        held = held[:-1] + [pair[1]] if pair[1] >= 0 else held
        while len(held) * page < past[b] + new[b]:
            held = held + [next(free)]
        kept[b] = held
    positions, slots, masks = [], [], []
    trees = _trees(case) if s["parents"] is not None else None
    for b in range(len(rows)):
        bits, depth = [], []
        for i in range(new[b]):
            key = past[b] + i
            slots.append(kept[b][key // page] * page + key % page)
            if trees is None:
                positions.append(key)
            else:
                p = trees[b][i]
                bits.append((1 << i) | (bits[p] if p >= 0 else 0))
                depth.append(0 if p < 0 else depth[p] + 1)
                positions.append(past[b] + depth[i])
        masks += bits
    pad = s["tokens"] - len(slots)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    width = s["table"].shape[1]
    out = [_ints([k + [-1] * (width - len(k)) for k in kept]), _ints(starts), _ints([p + n for p, n in zip(past, new)]),
           _ints(positions + [0] * pad, torch.int64), _ints(slots + [-1] * pad, torch.int64)]
    if trees is not None:
        out.append(torch.cat([_mask_words(case), torch.zeros(pad, s["words"], dtype=torch.int64, device="cuda")]))
    out += [_ints(copies), _ints([0])]
    if case["kind"] == "reorder":
        for c in s["caches"]:
            for _, src, dst, n in moved:
                c[:, dst, :, :n] = c[:, src, :, :n]
            out.append(c)
    return out


def _exact_tree(case, seed):
    lens, q, k, v, table = _tree_inputs(case, seed)
    hq, hkv, dim, page = (case[x] for x in ("hq", "hkv", "dim", "page"))
    masks, out, first = _bits(case), torch.empty(q.shape, dtype=torch.float64, device="cuda"), 0
    for b, (new, past) in enumerate(lens):
        key = torch.arange(past + new, device="cuda")
        where = table[b].long()[key // page]
        seen = torch.ones(new, past + new, dtype=torch.bool)
        seen[:, past:] = torch.tensor([[bool(m >> j & 1) for j in range(new)] for m in masks[first:first + new]])
        seen = seen.cuda()
        for h in range(hkv):
            kb, vb = k[where, h, key % page].double(), v[where, h, key % page].double()
            for g in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                score = q[first:first + new, g].double() @ kb.t().contiguous() / math.sqrt(dim)
                out[first:first + new, g] = torch.softmax(score.masked_fill(~seen, -math.inf), -1) @ vb
        first += new
    return out


def _exact_accept(case, seed):
    s = _accept_inputs(case, seed)
    page, longest = case["page"], s["longest"]
    tokens, picks, parents, table = (s[k].tolist() for k in ("tokens", "picks", "parents", "table"))
    paths, counts, accepted, ends, first, src, dst = [], [], [], [], 0, [], []
    for b, (new, past) in enumerate(s["lens"]):
        path = [0]
        while len(path) < longest:
            below = [c for c in range(path[-1] + 1, new) if parents[first + c] == path[-1]
                     and tokens[first + c] == picks[first + path[-1]]]
            if not below:
                break
            path.append(below[0])
        for d, c in enumerate(path):
            if c != d:
                src.append((table[b][(past + c) // page], (past + c) % page))
                dst.append((table[b][(past + d) // page], (past + d) % page))
        said = [tokens[first + c] for c in path[1:]] + [picks[first + path[-1]]]
        paths.append(path + [-1] * (longest - len(path)))
        accepted.append(said + [-1] * (longest - len(path)))
        counts.append(len(path))
        ends.append(past + len(path))
        first += new
    out = [_ints(paths), _ints(counts), _ints(accepted, torch.int64), _ints(ends)]
    for c in s["caches"]:
        rows = [c[:, p, :, r].clone() for p, r in src]      # all of them read before one is written
        for x, (p, r) in zip(rows, dst):
            c[:, p, :, r] = x
        out.append(c)
    return tuple(out)


def _exact_beam(case, seed):
    logits, scores, finished = _beam_inputs(case, seed)
    requests, beams, vocab, n = (case[k] for k in ("requests", "beams", "vocab", "n"))
    best, parent, token = [], [], []
    for r in range(requests):
        value = torch.log_softmax(logits[r * beams:(r + 1) * beams].double(), -1) + scores[r].double()[:, None]
        value[finished[r]] = -math.inf
        value[:, 0] = torch.where(finished[r], scores[r].double(), value[:, 0])
        value, flat = value.view(-1), None
        bound = torch.topk(value, n)[0][-1]
        flat = torch.cat([torch.nonzero(value > bound)[:, 0], torch.nonzero(value == bound)[:n, 0]])
        rank = torch.sort(value[flat], descending=True, stable=True)[1][:n]
        flat = flat[rank]
        # equal ones by index
        pairs = sorted(zip((-value[flat]).tolist(), flat.tolist()))
        flat = torch.tensor([i for _, i in pairs], device="cuda")
        best.append(value[flat])
        parent.append(flat // vocab)
        token.append(flat % vocab)
    return torch.stack(best), torch.stack(parent), torch.stack(token)


def exact(case, seed):
    return {"plan": _exact_plan, "reorder": _exact_plan, "tree": _exact_tree, "accept": _exact_accept,
            "beam": _exact_beam}[case["kind"]](case, seed)

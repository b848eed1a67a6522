"""The serving operators this library is measured on, through the entry points a user's program calls (own) or in their
plain form (elementary torch operations in 32 bits, rounded once at the end): what a batched decoder with a paged KV cache
runs between its projections and on its logits.

Every case is a dict of plain values with a "kind":

    norm_rope   ops.ext().norm_rope_paged(...)   `tokens` rows of a q|k|v projection: RMSNorm of every q and k head, the
                                                 position rotation, k and v into the pages of the cache
    attend      ops.ext().attention_paged(...)   new tokens of several sequences over their pages: `chunks` sequences with
                                                 `new_lo` .. `new_hi` new tokens and `ones` sequences with one, each on
                                                 `past_lo` .. `past_hi` cached tokens
    logprobs    ops.ext().token_logprobs(...)    log probabilities of given tokens, entropy and the `top` alternatives of
                                                 `rows` rows of logits

Cache layout: [pages, KV heads, page size, head dim]; row r of page p is slot p * page size + r.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
SIZE = {"float16": 2, "bfloat16": 2, "float32": 4}
EPS = 1e-6
THETA = 1e6


def listed():
    return [
        # one request's decode step: launch and host latency
        {"name": "norm_rope_1", "kind": "norm_rope", "tokens": 1, "hq": 28, "hkv": 4, "dim": 128, "page": 64,
         "dtype": "float16"},
        # a decode step of a batch of requests
        {"name": "norm_rope_67", "kind": "norm_rope", "tokens": 67, "hq": 16, "hkv": 2, "dim": 128, "page": 16,
         "dtype": "bfloat16"},
        # a full batch of prompt tokens
        {"name": "norm_rope_8192", "kind": "norm_rope", "tokens": 8192, "hq": 28, "hkv": 4, "dim": 128, "page": 64,
         "dtype": "float16"},
        # one request's decode step on a short context
        {"name": "attend_1", "kind": "attend", "chunks": 0, "new_lo": 1, "new_hi": 1, "ones": 1, "past_lo": 700,
         "past_hi": 700, "hq": 16, "hkv": 2, "dim": 128, "page": 64, "dtype": "float16"},
        # a decode step of 64 requests whose contexts differ
        {"name": "attend_64", "kind": "attend", "chunks": 0, "new_lo": 1, "new_hi": 1, "ones": 64, "past_lo": 300,
         "past_hi": 8000, "hq": 32, "hkv": 8, "dim": 128, "page": 16, "dtype": "bfloat16"},
        # a decode step of a few requests on long documents
        {"name": "attend_long", "kind": "attend", "chunks": 0, "new_lo": 1, "new_hi": 1, "ones": 3, "past_lo": 40000,
         "past_hi": 70000, "hq": 28, "hkv": 4, "dim": 128, "page": 64, "dtype": "float16"},
        # a mixed step: a piece of a long prompt together with the decode tokens of other requests
        {"name": "attend_mixed", "kind": "attend", "chunks": 1, "new_lo": 500, "new_hi": 500, "ones": 31, "past_lo": 300,
         "past_hi": 6000, "hq": 16, "hkv": 2, "dim": 128, "page": 32, "dtype": "float16"},
        # several short prompts batched, heads of 64
        {"name": "attend_prompts", "kind": "attend", "chunks": 6, "new_lo": 33, "new_hi": 1500, "ones": 0, "past_lo": 0,
         "past_hi": 0, "hq": 14, "hkv": 2, "dim": 64, "page": 16, "dtype": "float16"},
        # one long prompt
        {"name": "attend_8000", "kind": "attend", "chunks": 1, "new_lo": 8000, "new_hi": 8000, "ones": 0, "past_lo": 0,
         "past_hi": 0, "hq": 28, "hkv": 4, "dim": 128, "page": 64, "dtype": "float16"},
        # the sampled token of one decode step with its alternatives, as a serving interface reports them
        {"name": "logprobs_1", "kind": "logprobs", "rows": 1, "vocab": 151936, "top": 20, "dtype": "float16"},
        # the same for a batch, logits in fp32
        {"name": "logprobs_48", "kind": "logprobs", "rows": 48, "vocab": 151936, "top": 5, "dtype": "float32"},
        # a text scored token by token (perplexity), a vocabulary whose rows do not start on 16 bytes
        {"name": "logprobs_2047", "kind": "logprobs", "rows": 2047, "vocab": 151665, "top": 8, "dtype": "float16"},
    ]


def _spread(rng, lo, hi):
    """A whole number from lo .. hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = [(12, 2, 128), (16, 2, 128), (28, 4, 128), (32, 8, 128), (14, 2, 64), (8, 8, 64), (8, 1, 128)]
MOST_PAIRS = 28 * 128 * 32_000_000                          # query-key pairs x heads x head dim of the largest listed case
MOST_KEYS = 300_000 * 4 * 128                               # keys x KV heads x head dim of a decode step


def draw(rng):
    kind = rng.choice(["norm_rope", "attend", "attend", "attend", "logprobs", "logprobs"])
    if kind == "logprobs":
        vocab = _spread(rng, 1000, 152000)
        return {"kind": kind, "rows": _spread(rng, 1, min(2000, 2047 * 151665 // (2 * vocab))), "vocab": vocab,
                "top": rng.choice([1, 5, _spread(rng, 2, 32)]), "dtype": rng.choice(sorted(DTYPES))}
    hq, hkv, dim = rng.choice(HEADS)
    common = {"hq": hq, "hkv": hkv, "dim": dim, "page": rng.choice([16, 32, 64, 128]),
              "dtype": rng.choice(["float16", "bfloat16"])}
    if kind == "norm_rope":
        return {"kind": kind, "tokens": _spread(rng, 1, 6000), **common}
    case = {"kind": kind, "chunks": 0, "new_lo": 1, "new_hi": 1, "ones": 0, "past_lo": 0, "past_hi": 0, **common}
    shape = rng.choice(["decode", "mixed", "prompts", "drafts"])
    per_key, per_pair = hkv * dim, hq * dim
    if shape == "decode":
        case["ones"] = _spread(rng, 1, 200)
        case["past_hi"] = _spread(rng, 64, min(60000, max(65, MOST_KEYS // (per_key * case["ones"]))))
        case["past_lo"] = case["past_hi"] // rng.choice([1, 2, 10])
    elif shape == "drafts":                                 # a few drafted tokens of each request verified together
        case["chunks"] = _spread(rng, 1, 100)
        case["new_lo"], case["new_hi"] = 2, rng.choice([3, 5, 9])
        case["past_hi"] = _spread(rng, 64, min(30000, max(65, MOST_KEYS // (per_key * case["chunks"]))))
        case["past_lo"] = case["past_hi"] // 4
    elif shape == "mixed":
        case["chunks"], case["ones"] = rng.choice([1, 1, 2]), _spread(rng, 1, 60)
        case["new_hi"] = _spread(rng, 17, 1500)
        case["new_lo"] = max(1, case["new_hi"] // 2)
        case["past_hi"] = _spread(rng, 16, 5000)
    else:
        case["chunks"] = _spread(rng, 1, 12)
        case["new_hi"] = _spread(rng, 9, min(6000, int(math.sqrt(MOST_PAIRS / (per_pair * case["chunks"])))))
        case["new_lo"] = max(1, case["new_hi"] // rng.choice([1, 3, 20]))
        if rng.random() < 0.4:
            case["past_hi"] = _spread(rng, 1, max(2, min(8000, MOST_PAIRS // (4 * per_pair * case["chunks"] * case["new_hi"]))))
    return case


# ---- inputs, from the seed alone ----

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(1000003 * int(seed) + 29)


def _normal(shape, gen, std=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * std).to(dtype)


def _inv_freq(dim):
    return 1.0 / (THETA ** (torch.arange(0, dim, 2, dtype=torch.float32, device="cuda") / dim))


def _norm_rope_inputs(case, seed):
    gen, dt = _gen(seed), DTYPES[case["dtype"]]
    t, hq, hkv, dim, page = (case[k] for k in ("tokens", "hq", "hkv", "dim", "page"))
    qkv = _normal((t, (hq + 2 * hkv) * dim), gen, 1.5, dt)
    qw, kw = (1 + 0.2 * _normal((dim,), gen)).to(dt), (1 + 0.2 * _normal((dim,), gen)).to(dt)
    # a batch: runs of positions of several requests, far into their contexts
    starts = torch.randint(0, 120000, (-(-t // 512),), generator=gen, device="cuda")
    positions = starts.repeat_interleave(512)[:t] + torch.arange(t, device="cuda") % 512
    pages = -(-t // page) + 8
    slots = torch.randperm(pages, generator=gen, device="cuda").repeat_interleave(page)[:t] * page \
        + torch.arange(t, device="cuda") % page
    cache = _normal((2, pages, hkv, page, dim), gen, 1.0, dt)
    return qkv, qw, kw, positions, _inv_freq(dim), slots, cache[0], cache[1]


def _lengths(case):
    """(new tokens, keys in all) of every sequence; they belong to the case, not to the seed."""
    rng = random.Random("%(chunks)s %(ones)s %(new_lo)s %(new_hi)s %(past_lo)s %(past_hi)s" % case)

    def past():
        lo, hi = max(1, case["past_lo"]), max(1, case["past_hi"])
        return 0 if case["past_hi"] == 0 else _spread(rng, lo, hi)

    pairs = []
    for _ in range(case["chunks"]):
        new = _spread(rng, case["new_lo"], case["new_hi"])
        pairs.append((new, new + past()))
    pairs += [(1, 1 + past()) for _ in range(case["ones"])]
    rng.shuffle(pairs)
    return pairs


def _attend_inputs(case, seed):
    gen, dt = _gen(seed), DTYPES[case["dtype"]]
    hq, hkv, dim, page = (case[k] for k in ("hq", "hkv", "dim", "page"))
    lens = _lengths(case)
    need = [-(-keys // page) for _, keys in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros(len(lens), max(need), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    q = _normal((sum(n for n, _ in lens), hq, dim), gen, 1.5, dt)
    k = _normal((pages, hkv, page, dim), gen, 1.0, dt)
    v = _normal((pages, hkv, page, dim), gen, 1.0, dt)
    return lens, q, k, v, table


def _logits(case, seed):
    """Logits as a language model's: most of the vocabulary far below a few likely tokens."""
    gen, rows, vocab = _gen(seed), case["rows"], case["vocab"]
    x = _normal((rows, vocab), gen, 2.2)
    x -= 2.0
    likely = torch.randint(0, vocab, (rows, 12), generator=gen, device="cuda")
    x.scatter_add_(1, likely, 6.0 + 5.0 * torch.rand(rows, 12, generator=gen, device="cuda"))
    other = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    targets = torch.where(torch.rand(rows, generator=gen, device="cuda") < 0.7, likely[:, 0], other)
    return x.to(DTYPES[case["dtype"]]), targets


def prepare(case, seed):
    kind = case["kind"]
    state = {"case": case}
    if kind == "norm_rope":
        names = ("qkv", "qw", "kw", "positions", "inv_freq", "slots", "k_cache", "v_cache")
        state.update(zip(names, _norm_rope_inputs(case, seed)))
        state["q"] = torch.empty(case["tokens"], case["hq"], case["dim"], dtype=state["qkv"].dtype, device="cuda")
    elif kind == "attend":
        lens, q, k, v, table = _attend_inputs(case, seed)
        starts = [0]
        for n, _ in lens:
            starts.append(starts[-1] + n)
        state.update(lens=lens, starts=starts, q=q, k=k, v=v, table=table, out=torch.empty_like(q),
                     q_starts=torch.tensor(starts, dtype=torch.int32, device="cuda"),
                     kv_lens=torch.tensor([n for _, n in lens], dtype=torch.int32, device="cuda"),
                     max_new=max(n for n, _ in lens), max_keys=max(n for _, n in lens))
    else:
        state["logits"], state["targets"] = _logits(case, seed)
    if own:
        package = os.path.join(os.getcwd(), "lowbit-kernels_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
        from lowbit import ops
        state["ext"] = ops.ext()
    return state


# ---- one pass ----

def _plain_norm_rope(s):
    case = s["case"]
    t, hq, hkv, dim, page = (case[k] for k in ("tokens", "hq", "hkv", "dim", "page"))
    heads = s["qkv"].view(t, hq + 2 * hkv, dim).float()
    q, k, v = heads[:, :hq], heads[:, hq:hq + hkv], s["qkv"].view(t, hq + 2 * hkv, dim)[:, hq + hkv:]
    angle = s["positions"].double()[:, None] * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def rotated(x, w):
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
        a, b = x[..., :dim // 2], x[..., dim // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(s["qkv"].dtype)

    s["q"].copy_(rotated(q, s["qw"]))
    at, row = s["slots"] // page, s["slots"] % page
    s["k_cache"][at, :, row] = rotated(k, s["kw"])
    s["v_cache"][at, :, row] = v
    return s["q"], s["k_cache"], s["v_cache"]


def _plain_attend(s):
    case = s["case"]
    hq, hkv, dim, page = (case[k] for k in ("hq", "hkv", "dim", "page"))
    per, scale = hq // hkv, dim ** -0.5
    for b, (new, keys) in enumerate(s["lens"]):
        at = s["table"][b, :-(-keys // page)].long()
        k = s["k"][at].transpose(0, 1).reshape(hkv, -1, dim)[:, :keys].float()
        v = s["v"][at].transpose(0, 1).reshape(hkv, -1, dim)[:, :keys].float()
        kt = k.transpose(1, 2).contiguous()
        first = s["starts"][b]
        for i in range(0, new, 2048):
            n = min(2048, new - i)
            q = s["q"][first + i:first + i + n].float().view(n, hkv, per, dim).transpose(0, 1).reshape(hkv, n * per, dim)
            x = torch.matmul(q, kt) * scale
            if new > 1:
                last = torch.arange(keys - new + i, keys - new + i + n, device="cuda").repeat_interleave(per)
                x = x.masked_fill(torch.arange(keys, device="cuda")[None, :] > last[:, None], -math.inf)
            p = (x - x.amax(-1, keepdim=True)).exp()
            o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
            s["out"][first + i:first + i + n] = o.view(hkv, n, per, dim).transpose(0, 1).reshape(n, hq, dim).to(s["out"].dtype)
    return s["out"]


def _order(x):
    """x as whole numbers in its order (-0 as +0)."""
    bits = (x + 0.0).view(torch.int32)
    return torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)


def _plain_logprobs(s):
    x = s["logits"].float()
    vocab, top = x.shape[1], s["case"]["top"]
    low = x - x.amax(-1, keepdim=True)
    e = low.exp()
    total = e.sum(-1, keepdim=True)
    lse = total.log()
    logp = (torch.gather(low, 1, s["targets"][:, None]) - lse)[:, 0]
    # H = log Z - sum p (x - max)
    entropy = (lse - (e * low).sum(-1, keepdim=True) / total)[:, 0]
    # equal values: the lower index first
    key = (_order(x).long() << 32) + (vocab - 1 - torch.arange(vocab, device=x.device))
    ids = vocab - 1 - (torch.topk(key, top, dim=-1)[0] & 0xFFFFFFFF)
    return logp, entropy, torch.gather(low, 1, ids) - lse, ids


def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if not own:
        return {"norm_rope": _plain_norm_rope, "attend": _plain_attend, "logprobs": _plain_logprobs}[kind](state)
    ext = state["ext"]
    if kind == "norm_rope":
        ext.norm_rope_paged(state["qkv"], state["qw"], state["kw"], EPS, state["positions"], state["inv_freq"],
                            state["slots"], state["q"], state["k_cache"], state["v_cache"], case["hq"], case["hkv"])
        return state["q"], state["k_cache"], state["v_cache"]
    if kind == "attend":
        ext.attention_paged(state["q"], state["k"], state["v"], state["table"], state["q_starts"], state["kv_lens"],
                            state["out"], state["max_new"], state["max_keys"], case["dim"] ** -0.5)
        return state["out"]
    return ext.token_logprobs(state["logits"], state["targets"], case["top"])


# ---- what a pass cannot do without ----

def work(case):
    kind = case["kind"]
    if kind == "norm_rope":
        t, size = case["tokens"], SIZE[case["dtype"]]
        row = (case["hq"] + 2 * case["hkv"]) * case["dim"]
        return {"bytes": 2 * t * row * size + 16 * t + 2 * case["dim"] * size + 2 * case["dim"],
                "flops": 10 * t * (case["hq"] + case["hkv"]) * case["dim"]}
    if kind == "attend":
        lens, size = _lengths(case), SIZE[case["dtype"]]
        rows, keys = sum(n for n, _ in lens), sum(n for _, n in lens)
        pairs = sum(n * (k - n) + n * (n + 1) // 2 for n, k in lens)
        pages = sum(-(-k // case["page"]) for _, k in lens)
        return {"bytes": 2 * rows * case["hq"] * case["dim"] * size + 2 * keys * case["hkv"] * case["dim"] * size
                + 4 * pages + 8 * len(lens),
                "flops": 4 * pairs * case["hq"] * case["dim"]}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * SIZE[case["dtype"]] + case["rows"] * (16 + 12 * case["top"]), "flops": 6 * n}


# ---- the same in 64 bits ----

def _exact_norm_rope(case, seed):
    qkv, qw, kw, positions, inv_freq, slots, k_cache, v_cache = _norm_rope_inputs(case, seed)
    hq, hkv, dim, page = (case[k] for k in ("hq", "hkv", "dim", "page"))
    half = dim // 2
    x = qkv.double().unflatten(1, (-1, dim))
    theta = torch.outer(positions.double(), inv_freq.double())
    turn = torch.polar(torch.ones_like(theta), theta)       # the pair (x_i, x_{i + half}) as a complex number, turned

    def head(h, w):
        y = h / (h.pow(2).sum(-1, keepdim=True) / dim + EPS).sqrt() * w.double()
        z = torch.complex(y[..., :half].contiguous(), y[..., half:].contiguous()) * turn
        return torch.cat((z.real, z.imag), -1)

    q = torch.stack([head(x[:, h], qw) for h in range(hq)], 1)
    kc, vc = k_cache.double(), v_cache.double()
    for h in range(hkv):
        kc[slots // page, h, slots % page] = head(x[:, hq + h], kw)
        vc[slots // page, h, slots % page] = x[:, hq + hkv + h]
    return q, kc, vc


def _exact_attend(case, seed):
    lens, q, k, v, table = _attend_inputs(case, seed)
    hq, hkv, dim, page = (case[k] for k in ("hq", "hkv", "dim", "page"))
    out, first = torch.empty(q.shape, dtype=torch.float64, device="cuda"), 0
    for b, (new, keys) in enumerate(lens):
        slot = torch.arange(keys, device="cuda")
        where = table[b].long()[slot // page]
        for h in range(hkv):
            kb, vb = k[where, h, slot % page].double(), v[where, h, slot % page].double()
            for g in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                for i in range(0, new, 4096):
                    rows = slice(first + i, first + min(new, i + 4096))
                    score = q[rows, g].double() @ kb.t().contiguous() / math.sqrt(dim)
                    if new > 1:
                        own_key = keys - new + i + torch.arange(score.shape[0], device="cuda")
                        score[slot[None, :] > own_key[:, None]] = -math.inf
                    out[rows, g] = torch.softmax(score, -1) @ vb
        first += new
    return out


def _exact_logprobs(case, seed):
    logits, targets = _logits(case, seed)
    top = case["top"]
    parts = []
    for i in range(0, case["rows"], 128):
        x = logits[i:i + 128].double()
        logp = x - torch.logsumexp(x, -1, keepdim=True)
        value, ids = torch.sort(x, dim=-1, descending=True, stable=True)
        parts.append((logp.gather(1, targets[i:i + 128, None])[:, 0], -(logp.exp() * logp).sum(-1),
                      logp.gather(1, ids[:, :top]), ids[:, :top].clone()))
    return tuple(torch.cat(p) for p in zip(*parts))


def exact(case, seed):
    return {"norm_rope": _exact_norm_rope, "attend": _exact_attend, "logprobs": _exact_logprobs}[case["kind"]](case, seed)

"""Operators around a key/value cache held in 8 bits, and the scoring of given tokens: what is measured of them.

* ``store``    - queries and keys rotated, keys and values appended to a paged cache of 8-bit codes with a scale per block of tokens
                 and head; what the requests' cache then holds is read back as values;
* ``attend``   - attention over such a cache: single tokens of requests that hold ``context`` tokens, portions of ``new`` tokens
                 behind ``past`` ones, or both in one step;
* ``logprobs`` - log probabilities of given tokens, entropy, rank and the best alternatives from rows of logits.

A block is ``block`` consecutive positions of one request and kv head; its scale s is its largest magnitude and a code c stands for
c s / 127.  Appending to a block that is partly filled may raise its scale; its codes are then rounded again.
"""
from __future__ import annotations

import math
import random

import torch

own = False

# heads, kv heads, head size of the repository's configurations
HEADS = {"7b": (28, 4, 128), "14b": (40, 8, 128), "1.5b": (12, 2, 128)}
THETA = 1000000.0
VOCABULARY = 152064


def listed():
    return [
        # one user's decode step: one token appended, latency alone
        {"name": "store-7b-b1", "kind": "store", "shape": "7b", "singles": 1, "context": 300, "portions": 0, "new": 0, "past": 0,
         "page": 64, "block": 1, "dtype": "bfloat16"},
        # a full batch's decode step, blocks of a page's sixteen tokens: scales may rise, codes be rounded again
        {"name": "store-14b-b64-block16", "kind": "store", "shape": "14b", "singles": 64, "context": 512, "portions": 0, "new": 0,
         "past": 0, "page": 16, "block": 16, "dtype": "bfloat16"},
        # a prompt
        {"name": "store-7b-prompt-2048", "kind": "store", "shape": "7b", "singles": 0, "context": 0, "portions": 1, "new": 2048,
         "past": 0, "page": 64, "block": 1, "dtype": "bfloat16"},
        # one user's generation
        {"name": "decode-7b-b1-c2048", "kind": "attend", "shape": "7b", "singles": 1, "context": 2048, "portions": 0, "new": 0,
         "past": 0, "page": 64, "block": 1, "window": 0, "sink": False, "dtype": "bfloat16"},
        # a small batch on the benchmark's pages of sixteen, blocks of a page
        {"name": "decode-7b-b8-c2048-block16", "kind": "attend", "shape": "7b", "singles": 8, "context": 2048, "portions": 0, "new": 0,
         "past": 0, "page": 16, "block": 16, "window": 0, "sink": False, "dtype": "bfloat16"},
        # a full batch: the cache's bytes are what a step reads beside the weights
        {"name": "decode-14b-b64-c4096", "kind": "attend", "shape": "14b", "singles": 64, "context": 4096, "portions": 0, "new": 0,
         "past": 0, "page": 64, "block": 1, "window": 0, "sink": False, "dtype": "bfloat16"},
        # few requests deep in long contexts
        {"name": "decode-14b-b4-c32768", "kind": "attend", "shape": "14b", "singles": 4, "context": 32768, "portions": 0, "new": 0,
         "past": 0, "page": 64, "block": 1, "window": 0, "sink": False, "dtype": "bfloat16"},
        # a prompt in one step
        {"name": "prompt-7b-2048", "kind": "attend", "shape": "7b", "singles": 0, "context": 0, "portions": 1, "new": 2048,
         "past": 0, "page": 64, "block": 1, "window": 0, "sink": False, "dtype": "bfloat16"},
        # a mixed step of the scheduler's budget: single tokens beside a long prompt's portion
        {"name": "mixed-14b-b63-1985", "kind": "attend", "shape": "14b", "singles": 63, "context": 2048, "portions": 1, "new": 1985,
         "past": 6143, "page": 64, "block": 1, "window": 0, "sink": False, "dtype": "bfloat16"},
        # the float32 path of the same cache
        {"name": "decode-7b-b2-c1000-f32", "kind": "attend", "shape": "7b", "singles": 2, "context": 1000, "portions": 0, "new": 0,
         "past": 0, "page": 64, "block": 1, "window": 0, "sink": False, "dtype": "float32"},
        # the token that a request has just drawn, with the five best beside it
        {"name": "logprobs-r1-top5", "kind": "logprobs", "rows": 1, "vocab": VOCABULARY, "top": 5, "dtype": "float32"},
        # a prompt scored in one step, with the twenty best at every place
        {"name": "logprobs-r1024-top20", "kind": "logprobs", "rows": 1024, "vocab": VOCABULARY, "top": 20, "dtype": "float32"},
    ]


def _spread(rng, low, high):
    """A whole number between the two, even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng: random.Random):
    kind = rng.choice(["store", "attend", "attend", "logprobs"])
    if kind == "logprobs":
        vocab = _spread(rng, 1000, VOCABULARY)
        rows = _spread(rng, 1, max(1, min(4096, 1024 * VOCABULARY // vocab)))
        return {"kind": kind, "rows": rows, "vocab": vocab, "top": rng.choice([0, 1, 5, 20, 32]), "dtype": rng.choice(["float32", "float32", "bfloat16"])}
    case = {"kind": kind, "shape": rng.choice(sorted(HEADS)), "singles": 0, "context": 0, "portions": 0, "new": 0, "past": 0,
            "page": rng.choice([16, 32, 64])}
    case["block"] = rng.choice([1, 1, 4, 16, case["page"]])
    what = rng.choice(["singles", "singles", "portions", "both"])
    if what != "portions":
        case["singles"] = _spread(rng, 1, 64)
        case["context"] = _spread(rng, 2, min(32768, 262144 // case["singles"]) if kind == "attend" else 512)
    if what != "singles":
        case["portions"] = _spread(rng, 1, 4)
        case["new"] = _spread(rng, 2, 2048 // case["portions"])
        case["past"] = rng.choice([0, _spread(rng, 1, 5500 if kind == "attend" else 1000)])
    case["dtype"] = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    if case["dtype"] == "float32":           # the float32 path is for small work: a check of a model, not its service
        case["singles"], case["context"] = min(case["singles"], 8), min(case["context"], 2000)
        case["new"], case["past"] = min(case["new"], 200), min(case["past"], 1000)
    if kind == "attend":
        case["window"] = rng.choice([0, 0, 0, _spread(rng, 16, 4096)])
        case["sink"] = rng.random() < 0.25
    return case


def _lengths(case):
    """(tokens brought, tokens held afterwards) of every request: single tokens first; their contexts are ragged."""
    rng = random.Random(7)
    single = [max(1, case["context"] - rng.randrange(max(1, case["context"] // 2))) if i else case["context"] for i in range(case["singles"])]
    return [1] * case["singles"] + [case["new"]] * case["portions"], single + [case["past"] + case["new"]] * case["portions"]


def _index(case, device):
    brought, held = _lengths(case)
    rng = random.Random(11)
    page = case["page"]
    need = [-(-n // page) for n in held]
    order = list(range(sum(need) + 2))
    rng.shuffle(order)
    width, at, table = max(need), 0, []
    for n in need:
        table.append(order[at:at + n] + [-1] * (width - n))
        at += n
    positions = [p for b, h in zip(brought, held) for p in range(h - b, h)]
    seq = [s for s, b in enumerate(brought) for _ in range(b)]
    start = [0]
    for b in brought:
        start.append(start[-1] + b)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    return {"brought": brought, "held": held, "pages": len(order), "table": ints(table), "positions": ints(positions), "seq": ints(seq),
            "q_start": ints(start), "start_pos": ints([h - b for b, h in zip(brought, held)])}


def prepare(case, seed):
    device = torch.device("cuda:0")
    gen = torch.Generator(device=device).manual_seed(seed)
    dtype = getattr(torch, case["dtype"])
    normal = lambda *shape: torch.randn(shape, generator=gen, device=device)  # noqa: E731
    if case["kind"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        # a model's logits: a broad body and a few candidates that stand out; the given tokens are among those or anywhere
        logits = normal(rows, vocab) * 2.0
        picks = torch.randint(0, vocab, (rows, 8), generator=gen, device=device)
        logits.scatter_add_(1, picks, normal(rows, 8).abs() * 5.0 + 4.0)
        anywhere = torch.randint(0, vocab, (rows,), generator=gen, device=device)
        tokens = torch.where(torch.rand(rows, generator=gen, device=device) < 0.7, picks[:, 0], anywhere)
        return {"case": case, "logits": logits.to(dtype), "tokens": tokens.to(torch.int32)}
    heads, kv_heads, dim = HEADS[case["shape"]]
    index = _index(case, device)
    pages, page, blocks = index["pages"], case["page"], case["page"] // case["block"]
    state = {"case": case, **index}
    for name in ("k", "v"):
        # codes and scales as normal keys and values leave them
        state[name + "_pages"] = (normal(pages, kv_heads, page, dim) * 36.0).round_().clamp_(-127.0, 127.0).to(torch.int8)
        state[name + "_scale"] = 3.5 + 0.3 * normal(pages, kv_heads, blocks)
    tokens = index["positions"].numel()
    if case["kind"] == "store":
        rows = normal(tokens, (heads + 2 * kv_heads) * dim)
        # a few channels of the keys stand out, as projections with biases make them
        rows[:, heads * dim:(heads + kv_heads) * dim:16] *= 3.0
        state["qkv"] = rows.to(dtype)
        angles = torch.arange(max(index["held"]), device=device, dtype=torch.float32)[:, None] * (
            THETA ** (-torch.arange(0, dim, 2, device=device, dtype=torch.float32) / dim))
        state["cos"], state["sin"] = angles.cos(), angles.sin()
    else:
        state["q"] = (normal(tokens, heads * dim) * 1.5).to(dtype)
        state["sink"] = normal(heads) if case["sink"] else None
    return state


# ----------------------------------------------------------------------------
# plain forms
# ----------------------------------------------------------------------------
def _rotated(rows, cos, sin, positions):
    """rows [T, n, dim]: numbers d and d + dim/2 of a head turned by their position's angle."""
    half = rows.shape[-1] // 2
    c, s = cos[positions.long()][:, None], sin[positions.long()][:, None]
    lo, hi = rows[..., :half], rows[..., half:]
    return torch.cat([lo * c - hi * s, lo * s + hi * c], dim=-1)


def _append(codes, scale, rows, state):
    """Codes [pages, kv, page, dim] and scales [pages, kv, blocks] with the new rows [T, kv, dim], both as new tensors."""
    block, page = state["case"]["block"], state["case"]["page"]
    blocks = page // block
    pos, seq = state["positions"].long(), state["seq"].long()
    where = state["table"][seq, pos // page].long()
    at = where * blocks + pos % page // block                                              # block among all pages' blocks
    fresh = (pos // block * block) >= state["start_pos"].long()[seq]                       # the block begins in this step
    old = scale.transpose(1, 2).reshape(-1, scale.shape[1]).clone()                        # [pages * blocks, kv]
    old[at[fresh]] = 0.0
    new = old.index_reduce(0, at, rows.abs().amax(-1).to(old.dtype), "amax")
    ratio = torch.where(new > 0, old / new, 0.0)
    by_block = codes.unflatten(2, (blocks, block)).permute(0, 2, 1, 3, 4).flatten(0, 1)    # [pages * blocks, kv, block, dim]
    moved = torch.round(by_block * old[..., None, None] / new.clamp_min(1e-30)[..., None, None])
    moved = torch.where((ratio < 1.0)[..., None, None], moved, by_block.to(moved.dtype)).to(torch.int8)
    s = new[at][..., None]
    moved[at, :, pos % block] = torch.where(s > 0, torch.round(rows * 127.0 / s.clamp_min(1e-30)), 0.0).to(torch.int8)
    codes = moved.unflatten(0, (-1, blocks)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    return codes, new.unflatten(0, (-1, blocks)).transpose(1, 2)


def _values(codes, scale):
    return codes * (scale.repeat_interleave(codes.shape[2] // scale.shape[2], dim=2) / 127.0)[..., None]


def _runs_of_64(values, state):
    """The requests' positions one after the other in runs of 64, [runs, kv, 64, dim]; behind a request's last: zero."""
    page = state["case"]["page"]
    runs = [-(-n // 64) for n in state["held"]]
    device = values.device
    seq = torch.repeat_interleave(torch.arange(len(runs), device=device), torch.tensor(runs, device=device))
    first = torch.cumsum(torch.tensor([0] + runs[:-1], device=device), 0)
    pos = ((torch.arange(sum(runs), device=device) - first[seq]) * 64)[:, None] + torch.arange(64, device=device)
    held = torch.tensor(state["held"], device=device)[seq][:, None]
    where = state["table"].long()[seq[:, None], (pos // page).clamp_max(state["table"].shape[1] - 1)].clamp_min(0)
    picked = values[where, :, pos % page]                                                   # [runs, 64, kv, dim]
    return torch.where((pos < held)[..., None, None], picked, 0.0).transpose(1, 2).contiguous()


def _attend(q, k, v, start, length, scale, window, sink):
    """q [S, Q, heads, dim] behind ``start`` [S] positions; k, v [S, C, kv, dim]; ``length`` [S]: tokens held.  [S, Q, heads * dim]."""
    group = q.shape[2] // k.shape[2]
    scores = torch.einsum("sqkgd,sckd->skgqc", q.unflatten(2, (k.shape[2], group)), k) * scale
    pos = start[:, None] + torch.arange(q.shape[1], device=q.device)
    key = torch.arange(k.shape[1], device=q.device)
    seen = (key <= pos[..., None]) & (key < length[:, None, None])
    if window > 0:
        seen &= key > pos[..., None] - window
    scores = torch.where(seen[:, None, None], scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    if sink is not None:
        sink = sink.to(q.dtype).view(1, k.shape[2], group, 1, 1)
        top = torch.maximum(top, sink)
    p = torch.exp(scores - top)
    below = p.sum(-1, keepdim=True)
    if sink is not None:
        below = below + torch.exp(sink - top)
    return torch.einsum("skgqc,sckd->sqkgd", p / below, v).flatten(2)


def _attention(state, dtype):
    case = state["case"]
    heads, kv_heads, dim = HEADS[case["shape"]]
    singles, page = case["singles"], case["page"]
    q, out = state["q"].to(dtype).view(-1, heads, dim), []
    sink = state["sink"]
    held = torch.tensor(state["held"], device=q.device)

    def part(first, last, rows, new):
        pos = torch.arange(max(state["held"][first:last]), device=q.device)
        where = state["table"][first:last][:, pos // page].clamp_min(0).long()
        block = (pos % page) // case["block"]
        k, v = (state[n + "_pages"][where, :, pos % page].to(dtype) * (state[n + "_scale"][where, :, block].to(dtype) / 127.0)[..., None]
                for n in ("k", "v"))
        return _attend(rows.unflatten(0, (last - first, new)), k, v, state["start_pos"][first:last].long(), held[first:last], dim ** -0.5,
                       case["window"], sink).flatten(0, 1)

    if singles:
        out.append(part(0, singles, q[:singles], 1))
    if case["portions"]:
        out.append(part(singles, len(state["held"]), q[singles:], case["new"]))
    return torch.cat(out)


def _logprobs(logits, tokens, top):
    """Log probability of each row's token, entropy, rank, and the ``top`` best with theirs; ties go to the lowest index."""
    highest = logits.amax(-1, keepdim=True)
    shifted = logits - highest
    e = torch.exp(shifted)
    total = e.sum(-1, keepdim=True)
    own_one = logits.gather(1, tokens.long()[:, None])
    entropy = torch.log(total[:, 0]) - (e * shifted).sum(-1) / total[:, 0]
    index = torch.arange(logits.shape[1], device=logits.device)
    rank = ((logits > own_one) | ((logits == own_one) & (index < tokens[:, None]))).sum(-1)
    # one whole number per logit that orders like it, the lower index first among equals
    bits = (logits.to(torch.float32) + 0.0).view(torch.int32).to(torch.int64)
    order = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF)) * (1 << 20) - index
    ids = torch.topk(order, top, dim=-1).indices
    log_z = highest + torch.log(total)
    return (own_one - log_z)[:, 0], entropy, rank.to(torch.int32), ids.to(torch.int32), logits.gather(1, ids) - log_z


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    dtype = getattr(torch, case["dtype"])
    if case["kind"] == "logprobs":
        return dict(zip(("logprob", "entropy", "rank", "top_ids", "top_logprobs"), _logprobs(state["logits"].float(), state["tokens"], case["top"])))
    if case["kind"] == "attend":
        return {"out": _attention(state, torch.float32).to(dtype)}
    heads, kv_heads, dim = HEADS[case["shape"]]
    rows = state["qkv"].float().view(-1, heads + 2 * kv_heads, dim)
    rotated = _rotated(rows[:, :heads + kv_heads], state["cos"], state["sin"], state["positions"])
    k_codes, k_scale = _append(state["k_pages"], state["k_scale"], rotated[:, heads:], state)
    v_codes, v_scale = _append(state["v_pages"], state["v_scale"], rows[:, heads + kv_heads:], state)
    for name, t in (("k_pages", k_codes), ("v_pages", v_codes), ("k_scale", k_scale), ("v_scale", v_scale)):
        state[name].copy_(t)
    return {"q": rotated[:, :heads].flatten(1).to(dtype), "k_scale": state["k_scale"], "v_scale": state["v_scale"],
            "k": _runs_of_64(_values(state["k_pages"], state["k_scale"]), state).to(torch.bfloat16),
            "v": _runs_of_64(_values(state["v_pages"], state["v_scale"]), state).to(torch.bfloat16)}


def _run_own(state):
    from aegean_tge_b200 import ops
    case = state["case"]
    if case["kind"] == "logprobs":
        return dict(zip(("logprob", "entropy", "rank", "top_ids", "top_logprobs"), ops.token_logprobs(state["logits"], state["tokens"], top=case["top"])))
    heads, kv_heads, dim = HEADS[case["shape"]]
    cache = (state["k_pages"], state["v_pages"], state["k_scale"], state["v_scale"])
    if case["kind"] == "attend":
        return {"out": ops.attention_8bit(state["q"], *cache, state["table"], state["q_start"], state["start_pos"], state["positions"], state["seq"],
                                          len(state["held"]), max(state["brought"]), max(state["held"]), heads, kv_heads, dim, dim ** -0.5,
                                          window=case["window"], sink=state["sink"], decode_prefix=case["singles"], ctx_lens=state["held"])}
    q = ops.rope_kv_store_8bit(state["qkv"], state["cos"], state["sin"], dim, state["positions"], state["seq"], state["q_start"], state["table"],
                               *cache, heads, kv_heads, dim)
    k, v, _ = ops.read_cache_8bit(*cache, state["table"], state["q_start"], state["start_pos"], state["held"], torch.bfloat16)
    return {"q": q, "k_scale": state["k_scale"], "v_scale": state["v_scale"], "k": k, "v": v}


# ----------------------------------------------------------------------------
def work(case):
    if case["kind"] == "logprobs":
        count = case["rows"] * case["vocab"]
        return {"bytes": count * (4 if case["dtype"] == "float32" else 2) + case["rows"] * (16 + 8 * case["top"]), "flops": 5 * count}
    heads, kv_heads, dim = HEADS[case["shape"]]
    size = 4 if case["dtype"] == "float32" else 2
    brought, held = _lengths(case)
    tokens = sum(brought)
    entry = 2 * kv_heads * (dim + 4 / case["block"])                 # codes and scales of a position
    if case["kind"] == "store":
        runs = sum(-(-n // 64) for n in held)
        return {"bytes": int(tokens * ((2 * heads + 2 * kv_heads) * dim * size + 4 * dim + entry) + sum(held) * entry + runs * 64 * 2 * kv_heads * dim * 2),
                "flops": 3 * tokens * (heads + kv_heads) * dim + 4 * tokens * kv_heads * dim + 2 * sum(held) * kv_heads * dim}
    window = case["window"] or 1 << 30
    keys = sum(min(h, b + window - 1) for b, h in zip(brought, held))
    pairs = sum(sum(min(p + 1, window) for p in range(h - b, h)) for b, h in zip(brought, held))
    return {"bytes": int(keys * entry + 2 * tokens * heads * dim * size), "flops": 4 * heads * dim * pairs}


def exact(case, seed):
    """The definitions in 64 bits on the same inputs."""
    s = prepare(case, seed)
    if case["kind"] == "logprobs":
        x, t = s["logits"].double(), s["tokens"].long()
        z = torch.logsumexp(x, -1, keepdim=True)
        p = torch.softmax(x, -1)
        best = torch.sort(x, dim=-1, descending=True).values[:, :case["top"]] if case["top"] else x[:, :0]
        return {"logprob": (x - z)[torch.arange(len(t), device=x.device), t], "entropy": (z[:, 0] - (p * x).sum(-1)), "rank": None, "top_ids": None,
                "top_logprobs": best - z}
    heads, kv_heads, dim = HEADS[case["shape"]]
    group, page, block = heads // kv_heads, case["page"], case["block"]
    if case["kind"] == "attend":
        q = s["q"].double().view(-1, kv_heads, group, dim)
        rows, at = [], 0
        for r, (b, h) in enumerate(zip(s["brought"], s["held"])):
            pos = torch.arange(h, device=q.device)
            where = s["table"][r, pos // page].long()
            k, v = (s[n + "_pages"][where, :, pos % page].double() * s[n + "_scale"][where, :, pos % page // block].double()[..., None] / 127
                    for n in ("k", "v"))
            mine = pos[h - b:, None]
            hidden = (pos > mine) | (pos <= mine - (case["window"] or 1 << 30))
            heads_out = []
            for j in range(kv_heads):
                z = (q[at:at + b, j] @ k[:, j].T) * dim ** -0.5                              # [b, group, h]
                z.masked_fill_(hidden[:, None], -math.inf)
                norm = torch.logsumexp(z, -1)
                if case["sink"]:
                    norm = torch.logaddexp(norm, s["sink"].double().view(kv_heads, group)[j])
                heads_out.append(torch.exp(z - norm[..., None]) @ v[:, j])
            rows.append(torch.stack(heads_out, 1).flatten(1))
            at += b
        return {"out": torch.cat(rows)}
    x = s["qkv"].double().view(-1, heads + 2 * kv_heads, dim)
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"].long()][:, None]
    y = torch.complex(x[:, :heads + kv_heads, :dim // 2], x[:, :heads + kv_heads, dim // 2:]) * turn
    y = torch.cat([y.real, y.imag], -1)
    out = {"q": y[:, :heads].flatten(1)}
    for n, rows in (("k", y[:, heads:]), ("v", x[:, heads + kv_heads:])):
        scale, read, at = s[n + "_scale"].double(), [], 0
        for r, (b, h) in enumerate(zip(s["brought"], s["held"])):
            pos = torch.arange(h, device=x.device)
            where = s["table"][r, pos // page].long()
            first, blocks = h - b, -(-h // block)
            of = pos // block
            lead = pos[::block]                                                              # a position of every block
            old = scale[where[lead], :, lead % page // block]                                # [blocks, kv]
            old = torch.where((lead >= first)[:, None], 0.0, old)
            mine = rows[at:at + b].abs().amax(-1)
            new = old.index_reduce(0, of[first:], mine, "amax")
            codes = s[n + "_pages"][where, :, pos % page].double()
            again = torch.round(codes[:first] * old[of[:first]][..., None] / new[of[:first]][..., None])
            grown = (new > old)[of[:first]][..., None]
            codes[:first] = torch.where(grown, again, codes[:first])
            codes[first:] = torch.round(127 * rows[at:at + b] / new[of[first:]][..., None])
            scale[where[lead], :, lead % page // block] = new
            values = codes * new[of][..., None] / 127
            read.append(torch.cat([values, values.new_zeros((-h % 64, kv_heads, dim))]).view(-1, 64, kv_heads, dim).transpose(1, 2))
            at += b
        out[n + "_scale"], out[n] = scale, torch.cat(read)
    return out

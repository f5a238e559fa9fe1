"""Operators around a key/value cache held in 4 bits: what is measured of them.

* ``store``  - queries and keys normalised (if the layer does that) and rotated, keys and values appended to a paged cache of 4-bit
               codes; what was appended is read back as values;
* ``read``   - what requests hold in such a cache, as values;
* ``attend`` - attention over such a cache: single tokens of requests that hold ``context`` tokens, portions of ``new`` tokens behind
               ``past`` ones, or both in one step.

An entry (a position's key or value of one kv head) is cut into groups of 32 numbers, each with a step and a base in bfloat16; a code c of
0..15 stands for base + (c - 8) step.  Codes of four neighbours share 16 bits, the first in the lowest four; those sixteen bits follow one
another by their place in the group, then by group: numbers 32 j + 4 g .. 32 j + 4 g + 3 are the (g * groups + j)-th.
"""
from __future__ import annotations

import math
import random

import torch

own = False

# heads, kv heads, head size
HEADS = {"28/4x128": (28, 4, 128), "40/8x128": (40, 8, 128), "12/2x128": (12, 2, 128), "14/2x64": (14, 2, 64)}
THETA = 1000000.0
EPS = 1e-6


def listed():
    return [
        # one user's decode step: one token appended, latency alone
        {"name": "store-28-b1", "kind": "store", "shape": "28/4x128", "singles": 1, "context": 300, "portions": 0, "new": 0, "past": 0,
         "page": 64, "norm": False, "pairs": False, "dtype": "bfloat16"},
        # a full batch's decode step of a design that normalises the queries and keys of every head
        {"name": "store-40-b64-norm", "kind": "store", "shape": "40/8x128", "singles": 64, "context": 4096, "portions": 0, "new": 0,
         "past": 0, "page": 16, "norm": True, "pairs": False, "dtype": "bfloat16"},
        # a prompt; the rotation turns neighbours
        {"name": "store-28-prompt-2048-norm-pairs", "kind": "store", "shape": "28/4x128", "singles": 0, "context": 0, "portions": 1,
         "new": 2048, "past": 0, "page": 64, "norm": True, "pairs": True, "dtype": "bfloat16"},
        # a prompt's portion behind what an earlier step stored
        {"name": "read-28-c2048", "kind": "read", "shape": "28/4x128", "singles": 0, "context": 0, "portions": 1, "new": 512, "past": 1536,
         "page": 64, "window": 0, "dtype": "bfloat16"},
        # long contexts as values
        {"name": "read-40-b4-c32768", "kind": "read", "shape": "40/8x128", "singles": 4, "context": 32768, "portions": 0, "new": 0, "past": 0,
         "page": 64, "window": 0, "dtype": "bfloat16"},
        # one user's generation
        {"name": "decode-28-b1-c2048", "kind": "attend", "shape": "28/4x128", "singles": 1, "context": 2048, "portions": 0, "new": 0,
         "past": 0, "page": 64, "window": 0, "sink": False, "dtype": "bfloat16"},
        # a small batch on pages of sixteen, a window and a learned sink
        {"name": "decode-28-b8-c2048-window", "kind": "attend", "shape": "28/4x128", "singles": 8, "context": 2048, "portions": 0, "new": 0,
         "past": 0, "page": 16, "window": 1000, "sink": True, "dtype": "bfloat16"},
        # a full batch: the cache's bytes are what a step reads beside the weights
        {"name": "decode-40-b64-c4096", "kind": "attend", "shape": "40/8x128", "singles": 64, "context": 4096, "portions": 0, "new": 0,
         "past": 0, "page": 64, "window": 0, "sink": False, "dtype": "bfloat16"},
        # few requests deep in long contexts, which such a cache is for
        {"name": "decode-40-b4-c65536", "kind": "attend", "shape": "40/8x128", "singles": 4, "context": 65536, "portions": 0, "new": 0,
         "past": 0, "page": 64, "window": 0, "sink": False, "dtype": "bfloat16"},
        # a prompt in one step
        {"name": "prompt-28-2048", "kind": "attend", "shape": "28/4x128", "singles": 0, "context": 0, "portions": 1, "new": 2048,
         "past": 0, "page": 64, "window": 0, "sink": False, "dtype": "bfloat16"},
        # a mixed step of the scheduler's budget: single tokens beside a long prompt's portion
        {"name": "mixed-40-b63-1985", "kind": "attend", "shape": "40/8x128", "singles": 63, "context": 2048, "portions": 1, "new": 1985,
         "past": 6143, "page": 64, "window": 0, "sink": False, "dtype": "bfloat16"},
        # the float32 path of the same cache, heads of 64
        {"name": "decode-14-b2-c1000-f32", "kind": "attend", "shape": "14/2x64", "singles": 2, "context": 1000, "portions": 0, "new": 0,
         "past": 0, "page": 64, "window": 0, "sink": False, "dtype": "float32"},
    ]


def _spread(rng, low, high):
    """A whole number between the two, even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng: random.Random):
    kind = rng.choice(["store", "store", "read", "attend", "attend", "attend"])
    case = {"kind": kind, "shape": rng.choice(sorted(HEADS)), "singles": 0, "context": 0, "portions": 0, "new": 0, "past": 0,
            "page": rng.choice([16, 32, 64])}
    what = rng.choice(["singles", "singles", "portions", "both"])
    if what != "portions":
        case["singles"] = _spread(rng, 1, 64)
        most = 131072 if kind == "read" else 262144
        case["context"] = _spread(rng, 2, min(65536, most // case["singles"]))
    if what != "singles":
        case["portions"] = _spread(rng, 1, 4)
        case["new"] = _spread(rng, 2, 2048 // case["portions"])
        case["past"] = rng.choice([0, _spread(rng, 1, 5500)])
    case["dtype"] = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    if case["dtype"] == "float32":           # the float32 path is for small work: a check of a model, not its service
        case["singles"], case["context"] = min(case["singles"], 8), min(case["context"], 2000)
        case["new"], case["past"] = min(case["new"], 200), min(case["past"], 1000)
    if kind == "store":
        case["norm"], case["pairs"] = rng.random() < 0.5, rng.random() < 0.35
    else:
        case["window"] = rng.choice([0, 0, 0, _spread(rng, 16, 4096)])
    if kind == "attend":
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
    heads, kv_heads, dim = HEADS[case["shape"]]
    index = _index(case, device)
    pages, page, groups = index["pages"], case["page"], dim // 32
    state = {"case": case, **index}
    for name in ("k", "v"):
        # codes, steps and bases as normal keys and values leave them: sixteen steps across a group's 32 numbers
        nibbles = lambda: (normal(pages, kv_heads, page, 16 * groups) * 3.6 + 7.7).round_().clamp_(0.0, 15.0).to(torch.uint8)  # noqa: E731
        state[name + "_pages"] = nibbles() | (nibbles() << 4)
        step, base = 0.27 + 0.03 * normal(pages, kv_heads, page, groups), 0.2 * normal(pages, kv_heads, page, groups)
        if name == "k":                      # a group of channels stands out, as projections with biases make them
            step[..., 0] *= 1.5
        state[name + "_groups"] = torch.stack([step.clamp_min_(0.05), base], -1).flatten(-2).to(torch.bfloat16)
    tokens = index["positions"].numel()
    if case["kind"] == "store":
        rows = normal(tokens, (heads + 2 * kv_heads) * dim)
        rows[:, heads * dim:(heads + kv_heads) * dim:16] *= 1.5
        state["qkv"] = rows.to(dtype)
        angles = torch.arange(max(index["held"]), device=device, dtype=torch.float64)[:, None] * (
            THETA ** (-torch.arange(0, dim, 2, device=device, dtype=torch.float64) / dim))
        state["cos"], state["sin"] = angles.cos().float(), angles.sin().float()
        state["q_norm"] = 1.0 + 0.2 * normal(dim) if case["norm"] else None
        state["k_norm"] = 1.0 + 0.2 * normal(dim) if case["norm"] else None
    elif case["kind"] == "attend":
        state["q"] = (normal(tokens, heads * dim) * 1.5).to(dtype)
        state["sink"] = normal(heads) if case["sink"] else None
    return state


# ----------------------------------------------------------------------------
# plain forms
# ----------------------------------------------------------------------------
def _normalised(rows, weight):
    """rows [T, n, dim]: every head over its root mean square (the mean in 64 bits), times a weight per number."""
    mean = (rows.double().square().mean(-1, keepdim=True) + EPS).float()
    return rows * (1.0 / torch.sqrt(mean)) * weight


def _rotated(rows, cos, sin, positions, pairs):
    """rows [T, n, dim]: numbers d and d + dim/2 of a head (pairs: 2d and 2d + 1) turned by their position's angle."""
    c, s = cos[positions.long()][:, None], sin[positions.long()][:, None]
    half = rows.shape[-1] // 2
    lo, hi = (rows[..., ::2], rows[..., 1::2]) if pairs else (rows[..., :half], rows[..., half:])
    lo, hi = lo * c - hi * s, lo * s + hi * c
    return torch.stack([lo, hi], -1).flatten(-2) if pairs else torch.cat([lo, hi], -1)


def _bfloat16_above(x):
    """The smallest bfloat16 that is no smaller than x >= 0 (float32)."""
    return (((x.view(torch.int32) + 0xFFFF) >> 16) << 16).view(torch.float32)


def _entries(rows):
    """rows [T, kv, dim] (float32) as codes [T, kv, dim / 2] and (step, base) pairs [T, kv, dim / 16]."""
    x = rows.unflatten(-1, (-1, 32))
    low, high = x.amin(-1), x.amax(-1)
    base = (low + (high - low) * (8.0 / 15.0)).to(torch.bfloat16).float()
    step = _bfloat16_above(torch.maximum((high - base) / high.new_full((), 7.0), (base - low) * 0.125))
    steps = (x - base[..., None]) / torch.where(step > 0, step, 1.0)[..., None]
    codes = (torch.round(steps) + 8.0).clamp(0.0, 15.0).to(torch.uint8)                      # [T, kv, groups, 32]
    codes = codes.unflatten(-1, (8, 2, 2)).transpose(-4, -3)                                 # [T, kv, 8, groups, 2, 2]
    return (codes[..., 0] | (codes[..., 1] << 4)).flatten(-3), torch.stack([step, base], -1).flatten(-2).to(torch.bfloat16)


def _values(codes, pairs):
    """What codes [..., dim / 2] with pairs [..., dim / 16] stand for: [..., dim] in float32."""
    groups = codes.shape[-1] // 16
    c = torch.stack([codes & 15, codes >> 4], -1).unflatten(-2, (8, groups, 2)).transpose(-4, -3)
    step, base = pairs.float().unflatten(-1, (groups, 2)).unbind(-1)
    return ((c.flatten(-3).float() - 8.0) * step[..., None] + base[..., None]).flatten(-2)


def _runs_of_64(state, name, window):
    """The requests' positions one after the other in runs of 64, [runs, kv, 64, dim]; behind a request's last: zero.  With a window
    from the first run on that the step's queries see."""
    page = state["case"]["page"]
    first = [max(h - b - window + 1, 0) // 64 if window else 0 for b, h in zip(state["brought"], state["held"])]
    runs = [-(-h // 64) - f for f, h in zip(first, state["held"])]
    device = state["table"].device
    ints = lambda v: torch.tensor(v, device=device)  # noqa: E731
    seq = torch.repeat_interleave(torch.arange(len(runs), device=device), ints(runs))
    before = torch.cumsum(ints([0] + runs[:-1]), 0)
    pos = ((torch.arange(sum(runs), device=device) - before[seq] + ints(first)[seq]) * 64)[:, None] + torch.arange(64, device=device)
    where = state["table"].long()[seq[:, None], (pos // page).clamp_max(state["table"].shape[1] - 1)].clamp_min(0)
    picked = _values(state[name + "_pages"][where, :, pos % page], state[name + "_groups"][where, :, pos % page])   # [runs, 64, kv, dim]
    return torch.where((pos < ints(state["held"])[seq][:, None])[..., None, None], picked, 0.0).transpose(1, 2).contiguous()


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
        sink = sink.view(1, k.shape[2], group, 1, 1)
        top = torch.maximum(top, sink)
    p = torch.exp(scores - top)
    below = p.sum(-1, keepdim=True)
    if sink is not None:
        below = below + torch.exp(sink - top)
    return torch.einsum("skgqc,sckd->sqkgd", p / below, v).flatten(2)


def _attention(state):
    case = state["case"]
    heads, kv_heads, dim = HEADS[case["shape"]]
    singles, page = case["singles"], case["page"]
    q = state["q"].float().view(-1, heads, dim)
    device, outs = q.device, []
    for first, last, rows in ((0, singles, q[:singles][:, None]), (singles, len(state["held"]), q[singles:].unflatten(0, (case["portions"], -1)) if case["portions"] else None)):
        if last == first:
            continue
        held = torch.tensor(state["held"][first:last], device=device)
        pos = torch.arange(max(state["held"][first:last]), device=device)
        where = state["table"][first:last].long()[:, pos // page].clamp_min(0)
        k, v = (_values(state[n + "_pages"][where, :, pos % page], state[n + "_groups"][where, :, pos % page]) for n in ("k", "v"))   # [S, C, kv, dim]
        outs.append(_attend(rows, k, v, held - rows.shape[1], held, dim ** -0.5, case["window"], state["sink"]).flatten(0, 1))
    return torch.cat(outs)


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    if case["kind"] == "attend":
        return {"out": _attention(state).to(state["q"].dtype)}
    if case["kind"] == "read":
        return {n: _runs_of_64(state, n, case["window"]).to(getattr(torch, case["dtype"])) for n in ("k", "v")}
    heads, kv_heads, dim = HEADS[case["shape"]]
    rows = state["qkv"].float().view(-1, heads + 2 * kv_heads, dim)
    q, k, v = rows.split([heads, kv_heads, kv_heads], 1)
    if case["norm"]:
        q, k = _normalised(q, state["q_norm"]), _normalised(k, state["k_norm"])
    q, k = (_rotated(x, state["cos"], state["sin"], state["positions"], case["pairs"]) for x in (q, k))
    pos = state["positions"].long()
    where = state["table"][state["seq"].long(), pos // case["page"]].long()
    for name, x in (("k", k), ("v", v)):
        codes, pairs = _entries(x)
        state[name + "_pages"][where, :, pos % case["page"]] = codes
        state[name + "_groups"][where, :, pos % case["page"]] = pairs
    return {"q": q.flatten(1).to(state["qkv"].dtype), "k": _runs_of_64(state, "k", 1).to(torch.bfloat16), "v": _runs_of_64(state, "v", 1).to(torch.bfloat16)}


def _run_own(state):
    from aegean_tge_b200 import ops
    case = state["case"]
    heads, kv_heads, dim = HEADS[case["shape"]]
    cache = (state["k_pages"], state["v_pages"], state["k_groups"], state["v_groups"])
    if case["kind"] == "attend":
        return {"out": ops.attention_4bit(state["q"], *cache, state["table"], state["q_start"], state["start_pos"], state["positions"], state["seq"],
                                          len(state["held"]), max(state["brought"]), max(state["held"]), heads, kv_heads, dim, dim ** -0.5,
                                          window=case["window"], sink=state["sink"], decode_prefix=case["singles"], ctx_lens=state["held"])}
    if case["kind"] == "read":
        k, v, _ = ops.read_cache_4bit(*cache, state["table"], state["q_start"], state["start_pos"], state["held"], dim, getattr(torch, case["dtype"]),
                                      window=case["window"], q_lens=state["brought"])
        return {"k": k, "v": v}
    q = ops.norm_rope_kv_store_4bit(state["qkv"], state["cos"], state["sin"], dim, state["positions"], state["seq"], len(state["held"]), state["table"],
                                    *cache, heads, kv_heads, dim, q_norm=state["q_norm"], k_norm=state["k_norm"], eps=EPS, pairs=case["pairs"])
    # what the step appended: the runs that its queries would see through a window of themselves
    k, v, _ = ops.read_cache_4bit(*cache, state["table"], state["q_start"], state["start_pos"], state["held"], dim, torch.bfloat16, window=1,
                                  q_lens=state["brought"])
    return {"q": q, "k": k, "v": v}


# ----------------------------------------------------------------------------
def work(case):
    heads, kv_heads, dim = HEADS[case["shape"]]
    size = 4 if case["dtype"] == "float32" else 2
    brought, held = _lengths(case)
    tokens = sum(brought)
    entry = 2 * kv_heads * (dim // 2 + dim // 8)                      # codes, steps and bases of a position
    if case["kind"] == "store":
        positions = sum(h - (h - b) // 64 * 64 for b, h in zip(brought, held))
        runs = sum(-(-h // 64) - (h - b) // 64 for b, h in zip(brought, held))
        return {"bytes": int(tokens * ((2 * heads + 2 * kv_heads) * dim * size + 4 * dim + entry) + positions * entry + runs * 64 * 2 * kv_heads * dim * 2),
                "flops": (7 if case["norm"] else 3) * tokens * (heads + kv_heads) * dim + 6 * tokens * 2 * kv_heads * dim + 2 * positions * 2 * kv_heads * dim}
    window = case["window"] or 1 << 30
    if case["kind"] == "read":
        first = [max(h - b - window + 1, 0) // 64 * 64 for b, h in zip(brought, held)]
        positions = sum(h - f for h, f in zip(held, first))
        return {"bytes": int(positions * entry + sum(-(-(h - f) // 64) for h, f in zip(held, first)) * 64 * 2 * kv_heads * dim * size),
                "flops": 2 * positions * 2 * kv_heads * dim}
    keys = sum(min(h, b + window - 1) for b, h in zip(brought, held))
    pairs = sum(sum(min(p + 1, window) for p in range(h - b, h)) for b, h in zip(brought, held))
    return {"bytes": int(keys * entry + 2 * tokens * heads * dim * size), "flops": 4 * heads * dim * pairs}


def exact(case, seed):
    """The definitions in 64 bits on the same inputs."""
    s = prepare(case, seed)
    heads, kv_heads, dim = HEADS[case["shape"]]
    group, page, groups = heads // kv_heads, case["page"], dim // 32
    # where number d of an entry lies: its byte, and how far up in it
    d = torch.arange(dim, device=s["table"].device)
    byte, up = (d % 32 // 4 * groups + d // 32) * 2 + d % 4 // 2, d % 2 * 4

    def held(name, r, first, last):
        """Positions first .. last of request r as values [positions, kv, dim]."""
        pos = torch.arange(first, last, device=d.device)
        where = s["table"][r, pos // page].long()
        codes = (s[name + "_pages"][where, :, pos % page][..., byte].int() >> up) & 15
        pair = s[name + "_groups"][where, :, pos % page].double()
        return pair[..., 2 * (d // 32) + 1] + (codes - 8).double() * pair[..., 2 * (d // 32)]

    def in_runs(x):
        return torch.cat([x, x.new_zeros((-x.shape[0] % 64, kv_heads, dim))]).view(-1, 64, kv_heads, dim).transpose(1, 2)

    if case["kind"] == "read":
        first = [max(h - b - case["window"] + 1, 0) // 64 * 64 if case["window"] else 0 for b, h in zip(s["brought"], s["held"])]
        if sum(s["held"]) * kv_heads * dim > 1 << 28:
            return None
        return {n: torch.cat([in_runs(held(n, r, f, h)) for r, (f, h) in enumerate(zip(first, s["held"]))]) for n in ("k", "v")}
    if case["kind"] == "attend":
        q = s["q"].double().view(-1, kv_heads, group, dim)
        rows, at = [], 0
        for r, (b, h) in enumerate(zip(s["brought"], s["held"])):
            pos = torch.arange(h, device=q.device)
            k, v = held("k", r, 0, h), held("v", r, 0, h)
            mine = pos[h - b:, None]
            hidden = (pos > mine) | (pos <= mine - (case["window"] or 1 << 30))
            of_heads = []
            for j in range(kv_heads):
                z = (q[at:at + b, j] @ k[:, j].T) * dim ** -0.5                              # [b, group, h]
                z.masked_fill_(hidden[:, None], -math.inf)
                norm = torch.logsumexp(z, -1)
                if case["sink"]:
                    norm = torch.logaddexp(norm, s["sink"].double().view(kv_heads, group)[j])
                of_heads.append(torch.exp(z - norm[..., None]) @ v[:, j])
            rows.append(torch.stack(of_heads, 1).flatten(1))
            at += b
        return {"out": torch.cat(rows)}
    x = s["qkv"].double().view(-1, heads + 2 * kv_heads, dim)
    q, k, v = x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]
    if case["norm"]:
        q, k = (y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / dim + EPS) * w.double() for y, w in ((q, s["q_norm"]), (k, s["k_norm"])))
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"].long()][:, None]

    def turned(y):
        if case["pairs"]:
            return torch.view_as_real(torch.view_as_complex(y.reshape(*y.shape[:-1], dim // 2, 2)) * turn).flatten(-2)
        z = torch.complex(y[..., :dim // 2], y[..., dim // 2:]) * turn
        return torch.cat([z.real, z.imag], -1)

    out = {"q": turned(q).flatten(1)}
    for name, y in (("k", turned(k)), ("v", v)):
        y = y.reshape(-1, kv_heads, groups, 32)
        low, high = y.min(-1, keepdim=True).values, y.max(-1, keepdim=True).values
        base = (low + 8 * (high - low) / 15).to(torch.bfloat16).double()
        least = torch.maximum((high - base) / 7, (base - low) / 8)
        near = least.to(torch.bfloat16)
        step = torch.where(near.double() < least, (near.view(torch.int16) + 1).view(torch.bfloat16), near).double()
        codes = torch.where(step > 0, torch.round((y - base) / step.clamp_min(1e-300)), 0.0).clamp(-8, 7)
        y, read, at = (base + codes * step).flatten(-2), [], 0
        for r, (b, h) in enumerate(zip(s["brought"], s["held"])):
            before = held(name, r, (h - b) // 64 * 64, h - b)
            read.append(in_runs(torch.cat([before, y[at:at + b]])))
            at += b
        out[name] = torch.cat(read)
    return out

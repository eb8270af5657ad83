"""The measured work of the cache-step operators: what goes into a paged cache, how a tree of drafted
tokens reads it, which keys the attention uses, and how a cache that has grown too long is cut down.

Kinds of cases:

    norm_rope   qk_norm_rope_append: RMS norms of each head's query and key rows, the rotation by one
                or several position axes, and the rows' way into the cache, in one pass
    tree        paged_tree_attention: drafted tokens that see the cached context and their ancestors
    mass        paged_decode_mass: a decode step that also adds each key's attention weight to a total
    window      paged_window_mass: the weights that a prompt's last tokens give to each of its keys
    evict       evict_kv: the keys with the largest totals kept and moved to fresh pages
    commit      compact_kv in place: an accepted branch's rows moved behind the context

`run` computes a case in plain torch, in 32 bits and with angles in 64, or, with `own` true, by the
framework's operators.  Pools are [pages, 16, kv heads, head_dim], their pages in a random order.
"""
from __future__ import annotations

import math
import random

import torch

own = False

PAGE = 16
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEVICE = "cuda"
EPS = 1e-6
BASE = 1e6          # of the rotation's frequencies

# Head layouts (q heads, kv heads, head_dim) of the repository's configurations and tests.
LAYOUTS = [(14, 2, 64), (32, 8, 128), (32, 8, 128), (28, 4, 128), (12, 2, 128), (32, 32, 96), (16, 8, 256)]


def listed():
    return [
        # One user's chat turn: a single token, where the launch and latency count.
        {"name": "norm_rope_one_f32", "kind": "norm_rope", "dtype": "f32", "hq": 14, "hkv": 2, "d": 64,
         "tokens": 1, "axes": 1},
        # A prompt with pictures or film: time, height and width positions, an odd number of tokens.
        {"name": "norm_rope_video_bf16", "kind": "norm_rope", "dtype": "bf16", "hq": 28, "hkv": 4, "d": 128,
         "tokens": 5001, "axes": 3},
        # One user's speculative step: a small tree on a short context.
        {"name": "tree_one_f32", "kind": "tree", "dtype": "f32", "hq": 14, "hkv": 2, "d": 64,
         "batch": 1, "low": 512, "high": 512, "least": 26, "most": 26},
        # A served batch of 64-token trees on contexts of a few thousand tokens.
        {"name": "tree_b16_f16", "kind": "tree", "dtype": "f16", "hq": 32, "hkv": 8, "d": 128,
         "batch": 16, "low": 1000, "high": 8000, "least": 64, "most": 64},
        # Wide heads, many users, trees of one token (no draft) to 33.
        {"name": "tree_ragged_bf16", "kind": "tree", "dtype": "bf16", "hq": 16, "hkv": 8, "d": 256,
         "batch": 61, "low": 100, "high": 2100, "least": 1, "most": 33},
        # One user's decode step with the totals kept.
        {"name": "mass_one_f32", "kind": "mass", "dtype": "f32", "hq": 14, "hkv": 2, "d": 64,
         "batch": 1, "low": 512, "high": 512},
        # A full decode batch of long contexts: the largest read.
        {"name": "mass_b64_f16", "kind": "mass", "dtype": "f16", "hq": 32, "hkv": 8, "d": 128,
         "batch": 64, "low": 1000, "high": 8000},
        # Eight prompts, each weighed by its last 32 tokens.
        {"name": "window_b8_f16", "kind": "window", "dtype": "f16", "hq": 14, "hkv": 2, "d": 64,
         "batch": 8, "low": 512, "high": 4608, "rows": 32},
        # Two long documents, weighed by their last 64 tokens.
        {"name": "window_long_bf16", "kind": "window", "dtype": "bf16", "hq": 28, "hkv": 4, "d": 128,
         "batch": 2, "low": 29000, "high": 30001, "rows": 64},
        # A batch of contexts of about 4000 tokens cut down to 1024.
        {"name": "evict_b32_f16", "kind": "evict", "dtype": "f16", "hq": 32, "hkv": 8, "d": 128,
         "batch": 32, "low": 3500, "high": 4500, "budget": 1024, "sinks": 4, "recent": 128},
        # One very long context of an odd length cut down to 16384.
        {"name": "evict_long_bf16", "kind": "evict", "dtype": "bf16", "hq": 14, "hkv": 2, "d": 64,
         "batch": 1, "low": 100001, "high": 100001, "budget": 16384, "sinks": 16, "recent": 1000},
        # The accepted branches of a batch's trees: at most 9 rows each, moved in place.
        {"name": "commit_b64_f16", "kind": "commit", "dtype": "f16", "hq": 32, "hkv": 8, "d": 128,
         "batch": 64, "low": 100, "high": 4000, "nodes": 64, "most": 9},
    ]


# What a drawn case may cost at most (the largest listed cases' work).
_MAX_KV_BYTES = 1_100_000_000
_MAX_FLOPS = {"f32": 1e10, "f16": 6e10, "bf16": 6e10}


def _log_int(rng: random.Random, low: int, high: int) -> int:
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["norm_rope", "tree", "tree", "tree", "mass", "mass", "window", "evict", "commit"])
    hq, hkv, d = rng.choice(LAYOUTS)
    c = {"kind": kind, "dtype": rng.choice(["f32", "f16", "bf16"]), "hq": hq, "hkv": hkv, "d": d}
    row_bytes = 2 * hkv * d * DTYPES[c["dtype"]].itemsize
    if kind == "norm_rope":
        c["tokens"] = _log_int(rng, 1, 5001 if c["dtype"] != "f32" else 2500)
        c["axes"] = rng.choice([1, 1, 3])
        return c
    c["batch"] = _log_int(rng, 1, 64)
    longest = {"tree": 32768, "mass": 32768, "window": 30001, "evict": 100001, "commit": 8192}[kind]
    most = max(64, min(longest, int(_MAX_KV_BYTES / (2 if kind == "evict" else 1) / (row_bytes * c["batch"]))))
    c["high"] = _log_int(rng, 64, most)
    c["low"] = max(1, c["high"] // rng.choice([1, 2, 16]))
    if kind == "tree":
        c["most"] = _log_int(rng, 1, 128)
        while 4 * d * hq * c["most"] * c["batch"] * c["high"] > _MAX_FLOPS[c["dtype"]] and c["most"] > 1:
            c["most"] //= 2
        c["least"] = rng.choice([1, c["most"]])
    elif kind == "window":
        c["rows"] = _log_int(rng, 1, 64)
        while 2 * d * hq * c["rows"] * c["batch"] * c["high"] > _MAX_FLOPS[c["dtype"]] / 2 and c["rows"] > 1:
            c["rows"] //= 2
        c["low"] = max(c["low"], c["rows"])
        c["high"] = max(c["high"], c["rows"])
    elif kind == "evict":
        c["budget"] = _log_int(rng, 16, c["high"])
        c["sinks"] = min(4, c["budget"] // 4)
        c["recent"] = c["budget"] // rng.choice([4, 8, 16])
    elif kind == "commit":
        c["nodes"] = _log_int(rng, 1, 128)
        c["most"] = min(c["nodes"], rng.randint(1, 16))
    return c


# ---------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------

def _lengths(case: dict) -> list:
    """The batch's context lengths: the case's own (its work does not depend on the seed)."""
    low, high, n = case["low"], case["high"], case["batch"]
    rng = random.Random(1000003 * n + 1009 * high + low)
    return [rng.randint(low, high) for _ in range(n)]


def _nodes(case: dict) -> list:
    """The trees' sizes, likewise."""
    rng = random.Random(7919 * case["batch"] + 31 * case["most"] + case["least"])
    return [rng.randint(case["least"], case["most"]) for _ in range(case["batch"])]


def _randn(shape, dtype, g) -> torch.Tensor:
    """N(0, 1) in `dtype`, made on the device (in pieces, so that no 32-bit copy of a pool is kept)."""
    out = torch.empty(shape, dtype=dtype, device=DEVICE)
    flat, step = out.view(-1), 1 << 26
    for i in range(0, flat.numel(), step):
        part = flat[i:i + step]
        part.copy_(torch.randn(part.numel(), generator=g, device=DEVICE))
    return out


def _tables(lens: list, seed: int, spare: int = 0):
    """Block tables [B, max pages] (-1 padded, int32, on the device), `spare` page ids that no table
    holds, and the pool's page count."""
    need = [(n + PAGE - 1) // PAGE for n in lens]
    total = sum(need)
    nb = total + spare + total // 8 + 8
    perm = torch.randperm(nb, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32)
    table[torch.arange(table.shape[1])[None, :] < torch.tensor(need)[:, None]] = perm[:total]
    return table.to(DEVICE), perm[total:total + spare].to(DEVICE), nb


def _int32(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _cumsum(values: list) -> list:
    out = [0]
    for v in values:
        out.append(out[-1] + v)
    return out


def _sections(half: int, axes: int) -> tuple:
    """The axis of each frequency: a quarter by time, three eighths each by height and width."""
    if axes == 1:
        return (0,) * half
    a, b = half // 4, half // 4 + (half - half // 4 + 1) // 2
    return (0,) * a + (1,) * (b - a) + (2,) * (half - b)


def _parents(rng: random.Random, nodes: list) -> list:
    """A drafted tree: each node hangs on one of the eight before it, or starts a branch of its own."""
    return [[rng.randint(max(-1, i - 8), i - 1) if i and rng.random() < 0.95 else -1 for i in range(n)]
            for n in nodes]


def _tree_mask(parents: list, words: int) -> torch.Tensor:
    """int32 [nodes, words]: bit j of a node's row is set where it sees node j (itself, its ancestors)."""
    rows = []
    for tree in parents:
        seen = []
        for i, p in enumerate(tree):
            seen.append((seen[p] if p >= 0 else 0) | 1 << i)
        rows += [[(s >> 32 * w) & 0xFFFFFFFF for w in range(words)] for s in seen]
    return torch.tensor(rows, dtype=torch.int64).to(torch.uint32).view(torch.int32).to(DEVICE)


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    rng = random.Random(seed)
    kind, dt, hq, hkv, d = case["kind"], DTYPES[case["dtype"]], case["hq"], case["hkv"], case["d"]
    s = {"kind": kind, "case": case}
    if kind == "norm_rope":
        # q, k and v as the fused projection leaves them: slices of one row per token
        tokens, axes, half = case["tokens"], case["axes"], d // 2
        qkv = _randn((tokens, hq + 2 * hkv, d), dt, g)
        s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        nb = (tokens + PAGE - 1) // PAGE + 8
        s["k_pool"] = torch.zeros((nb, PAGE, hkv, d), dtype=dt, device=DEVICE)
        s["v_pool"] = torch.zeros_like(s["k_pool"])
        perm = torch.randperm(nb * PAGE, generator=torch.Generator().manual_seed(seed))
        s["slots"] = perm[:tokens].to(DEVICE)
        first, i = rng.randint(0, 130000), torch.arange(tokens)
        pos = [first + i] if axes == 1 else [first + i // 1156, first + i // 34 % 34, first + i % 34]
        s["positions"] = torch.stack(pos).to(torch.int32).to(DEVICE)
        s["pair_axis"] = _sections(half, axes)
        s["inv_freq"] = (BASE ** (-torch.arange(half).double() / half)).float().to(DEVICE)
        s["q_weight"] = 1 + 0.1 * torch.randn(d, generator=g, device=DEVICE)
        s["k_weight"] = 1 + 0.1 * torch.randn(d, generator=g, device=DEVICE)
        return s
    lens = _lengths(case)
    rng.shuffle(lens)
    if kind == "tree":
        nodes = _nodes(case)
        lens = [a + b for a, b in zip(lens, nodes)]     # the drafted rows are in the cache
        words = (max(nodes) + 31) // 32
        s.update(nodes=nodes, most=max(nodes), cu=_int32(_cumsum(nodes)))
        s["parents"] = _parents(rng, nodes)
        s["mask"] = _tree_mask(s["parents"], words)
        s["q"] = _randn((sum(nodes), hq, d), dt, g)
    elif kind == "window":
        rows = [min(case["rows"], n) for n in lens]
        s.update(nodes=rows, most=max(rows), cu=_int32(_cumsum(rows)))
        s["q"] = _randn((sum(rows), hq, d), dt, g)
    elif kind == "mass":
        s["q"] = _randn((len(lens), hq, d), dt, g)
    context = lens
    if kind == "commit":
        lens = [n + case["nodes"] for n in lens]
    pages = (case["budget"] + PAGE - 1) // PAGE if kind == "evict" else 0
    s["table"], fresh, nb = _tables(lens, seed, pages * len(lens))
    s.update(lens=lens, seq_lens=_int32(lens), longest=max(lens))
    s["k_pool"] = _randn((nb, PAGE, hkv, d), dt, g)
    s["v_pool"] = _randn((nb, PAGE, hkv, d), dt, g)
    if kind in ("mass", "window", "evict"):
        width = (max(lens) + 63) // 64 * 64             # room for the next steps' keys
        # totals after the steps of a while (evict), or of the first few
        m = torch.randn((len(lens), hkv, width), generator=g, device=DEVICE).mul_(2).exp_()
        m *= 1.0 if kind == "evict" else 2.0 ** -10
        # keys that no query has looked at yet: their totals are equal
        s["mass"] = m * (torch.rand(m.shape, generator=g, device=DEVICE) > 0.1)
    if kind == "evict":
        s["fresh"] = fresh.view(len(lens), pages)
    if kind == "commit":
        accepted = [sorted(rng.sample(range(case["nodes"]), rng.randint(1, case["most"]))) for _ in lens]
        rows = [[n + a for a in acc] + [-1] * (case["most"] - len(acc)) for n, acc in zip(context, accepted)]
        s["keep"] = _int32(rows).view(len(lens), 1, case["most"])
        s["counts"], s["start"] = _int32([len(a) for a in accepted]), _int32(context)
    return s


# ---------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------

def run(s: dict):
    if own:
        return _run_own(s)
    return {"norm_rope": _plain_norm_rope, "tree": _plain_tree, "mass": _plain_mass, "window": _plain_window,
            "evict": _plain_evict, "commit": _plain_commit}[s["kind"]](s)


def _run_own(s: dict):
    from lightllm_amd import kv_cache as kc

    kind, case = s["kind"], s["case"]
    if kind == "norm_rope":
        q = kc.qk_norm_rope_append(s["q"], s["k"], s["v"], s["slots"], s["positions"], s["inv_freq"], s["k_pool"],
                                   s["v_pool"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS,
                                   pair_axis=s["pair_axis"])
        return q, s["k_pool"], s["v_pool"]
    if kind == "tree":
        return kc.paged_tree_attention(s["q"], s["k_pool"], s["v_pool"], s["table"], s["cu"], s["seq_lens"],
                                       s["mask"], s["most"], s["longest"])
    if kind == "mass":
        out = kc.paged_decode_mass(s["q"], s["k_pool"], s["v_pool"], s["table"], s["seq_lens"], s["longest"],
                                   s["mass"])
        return out, s["mass"]
    if kind == "window":
        kc.paged_window_mass(s["q"], s["k_pool"], s["table"], s["cu"], s["seq_lens"], s["most"], s["longest"],
                             s["mass"])
        return s["mass"]
    if kind == "evict":
        keep, counts, mass = kc.evict_kv(s["k_pool"], s["v_pool"], s["table"], s["seq_lens"], s["mass"],
                                         case["budget"], s["longest"], sinks=case["sinks"], recent=case["recent"],
                                         dst_table=s["fresh"])
        return keep, counts, mass, s["k_pool"], s["v_pool"]
    kc.compact_kv(s["k_pool"], s["v_pool"], s["table"], s["keep"], s["counts"], dst_start=s["start"])
    return s["k_pool"], s["v_pool"]


def _plain_norm_rope(s: dict):
    pos = s["positions"][list(s["pair_axis"])]                         # [half, T]
    angle = pos.t().double() * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]
    half = cos.shape[-1]
    turned = []
    for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
        y = x.float()
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * w
        a, b = y[..., :half], y[..., half:]
        turned.append(torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(x.dtype))
    for pool, rows in ((s["k_pool"], turned[1]), (s["v_pool"], s["v"])):
        pool.view(-1, pool.shape[2], pool.shape[3])[s["slots"]] = rows
    return turned[0], s["k_pool"], s["v_pool"]


def _padded(pool: torch.Tensor, table: torch.Tensor, n: int) -> torch.Tensor:
    """The first n positions of every sequence: 32 bits, [B, Hkv, n, D]."""
    pos = torch.arange(n, device=DEVICE)
    rows = table.clamp(min=0).long()[:, pos // PAGE] * PAGE + pos % PAGE
    return pool.view(-1, pool.shape[2], pool.shape[3])[rows].permute(0, 2, 1, 3).float().contiguous()


def _weights(q: torch.Tensor, k: torch.Tensor, seen: torch.Tensor) -> torch.Tensor:
    """softmax over the keys seen: q [B, Hkv, M, D], k [B, Hkv, L, D], seen [B, 1 or Hkv, M, L]."""
    x = torch.matmul(q, k.transpose(2, 3)) / math.sqrt(q.shape[3])
    x = torch.where(seen, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = (x - torch.where(top == -math.inf, 0.0, top)).exp()
    return p / p.sum(-1, keepdim=True).clamp(min=1e-30)


def _padded_q(s: dict):
    """The query rows of every sequence [B, Hkv, G * most, D], each padded row's node [B, most] and
    whether it is one."""
    hkv, most, cu = s["case"]["hkv"], s["most"], s["cu"].long()
    node = torch.arange(most, device=DEVICE)
    at = cu[:-1, None] + node
    real = at < cu[1:, None]
    q = s["q"][at.clamp(max=s["q"].shape[0] - 1)].float()             # [B, most, Hq, D]
    b, _, hq, d = q.shape
    q = q.view(b, most, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    return q.contiguous(), at, real


def _plain_tree(s: dict):
    q, at, real = _padded_q(s)
    b, hkv, m, d = q.shape
    g, most, n = m // s["most"], s["most"], s["longest"]
    lens, count = s["seq_lens"].long(), (s["cu"][1:] - s["cu"][:-1]).long()
    node = torch.arange(n, device=DEVICE) - (lens - count)[:, None]   # [B, L]: the key's node, below 0: context
    row = s["mask"][at.clamp(max=s["q"].shape[0] - 1)].long()         # [B, most, words]
    word = torch.gather(row, 2, (node.clamp(min=0, max=most - 1) // 32)[:, None, :].expand(b, most, n))
    bit = (word >> (node.clamp(min=0) % 32)[:, None, :]) & 1
    seen = ((node < 0)[:, None, :] | (bit == 1)) & (node < count[:, None])[:, None, :]
    seen = seen[:, None, None].expand(b, 1, g, most, n).reshape(b, 1, m, n)
    p = _weights(q, _padded(s["k_pool"], s["table"], n), seen)
    o = torch.matmul(p, _padded(s["v_pool"], s["table"], n))          # [B, Hkv, G * most, D]
    o = o.view(b, hkv, g, most, d).permute(0, 3, 1, 2, 4).reshape(b, most, hkv * g, d)
    return o[real].to(s["q"].dtype)


def _plain_mass(s: dict):
    b, hq, d = s["q"].shape
    hkv, n = s["case"]["hkv"], s["longest"]
    seen = (torch.arange(n, device=DEVICE) < s["seq_lens"][:, None])[:, None, None, :]
    p = _weights(s["q"].float().view(b, hkv, hq // hkv, d), _padded(s["k_pool"], s["table"], n), seen)
    o = torch.matmul(p, _padded(s["v_pool"], s["table"], n))
    s["mass"][:, :, :n] += p.sum(2)
    return o.reshape(b, hq, d).to(s["q"].dtype), s["mass"]


def _plain_window(s: dict):
    q, at, real = _padded_q(s)
    b, hkv, m, d = q.shape
    g, most, n = m // s["most"], s["most"], s["longest"]
    lens, count = s["seq_lens"].long(), (s["cu"][1:] - s["cu"][:-1]).long()
    place = (lens - count)[:, None] + torch.arange(most, device=DEVICE)             # [B, most]
    key = torch.arange(n, device=DEVICE)
    seen = (key <= place[:, :, None]) & (key < lens[:, None, None]) & real[:, :, None]
    seen = seen[:, None, None].expand(b, 1, g, most, n).reshape(b, 1, m, n)
    s["mass"][:, :, :n] += _weights(q, _padded(s["k_pool"], s["table"], n), seen).sum(2)
    return s["mass"]


def _moved(s: dict, keep: torch.Tensor, counts: torch.Tensor, dst: torch.Tensor, start: torch.Tensor):
    """Rows at positions keep [B, Hkv, M] moved to start + 0, 1, .. of the tables dst, all of them
    read before the first is written."""
    b, hkv, m = keep.shape
    i = torch.arange(m, device=DEVICE)
    real = (i < counts[:, None])[:, None, :].expand(b, hkv, m)

    def rows(table, pos):                                              # [B, Hkv, M] -> rows of a head's pool
        page = torch.gather(table.long(), 1, (pos // PAGE).view(b, -1)).view(b, hkv, m)
        return (page * PAGE + pos % PAGE) * hkv + torch.arange(hkv, device=DEVICE)[:, None]

    source = rows(s["table"], keep.long().clamp(min=0))[real]
    to = start.long()[:, None, None] + i.expand(b, hkv, m)
    to = rows(dst, torch.where(real, to, 0))[real]
    for pool in (s["k_pool"], s["v_pool"]):
        flat = pool.view(-1, pool.shape[3])
        flat[to] = flat[source]


def _plain_evict(s: dict):
    case, mass = s["case"], s["mass"]
    n, budget = s["longest"], min(case["budget"], s["longest"])
    lens = s["seq_lens"].long()[:, None, None]
    pos = torch.arange(n, device=DEVICE).expand(mass.shape[0], mass.shape[1], n)
    held = (pos < case["sinks"]) | (pos >= lens - case["recent"])
    rank = torch.where(held, math.inf, mass[:, :, :n])
    rank = torch.where(pos < lens, rank, -math.inf)
    first = rank.sort(stable=True, dim=-1, descending=True).indices[:, :, :budget]
    counts = s["seq_lens"].clamp(max=case["budget"])
    real = torch.arange(budget, device=DEVICE) < counts[:, None, None]
    kept = torch.where(real, first, n).sort(-1).values
    keep = torch.full((*mass.shape[:2], case["budget"]), -1, dtype=torch.int32, device=DEVICE)
    keep[:, :, :budget] = torch.where(kept < n, kept, -1)
    total = torch.zeros_like(mass)
    total[:, :, :budget] = torch.where(kept < n, torch.gather(mass, 2, kept.clamp(max=n - 1)), 0.0)
    _moved(s, keep, counts, s["fresh"], torch.zeros_like(counts))
    return keep, counts, total, s["k_pool"], s["v_pool"]


def _plain_commit(s: dict):
    keep = s["keep"].expand(-1, s["case"]["hkv"], -1)
    _moved(s, keep, s["counts"], s["table"], s["start"])
    return s["k_pool"], s["v_pool"]


# ---------------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------------

def work(case: dict) -> dict:
    es, hq, hkv, d = DTYPES[case["dtype"]].itemsize, case["hq"], case["hkv"], case["d"]
    kind, row = case["kind"], hkv * d * es                # one token's K (or V) row
    if kind == "norm_rope":
        t = case["tokens"]
        return {"bytes": t * ((2 * hq + 4 * hkv) * d * es + 4 * case["axes"] + 8) + 2 * d + 8 * d,
                "flops": 7 * t * (hq + hkv) * d}
    lens = _lengths(case)
    n = case["batch"]
    if kind == "tree":
        nodes = _nodes(case)
        keys, pairs = sum(lens) + sum(nodes), sum(a * b for a, b in zip(lens, nodes))
        return {"bytes": 2 * keys * row + 2 * sum(nodes) * hq * d * es, "flops": 4 * pairs * hq * d}
    keys = sum(lens)
    if kind == "mass":
        return {"bytes": 2 * keys * row + 2 * n * hq * d * es + 8 * keys * hkv, "flops": 4 * keys * hq * d}
    if kind == "window":
        rows = [min(case["rows"], a) for a in lens]
        return {"bytes": keys * row + sum(rows) * hq * d * es + 8 * keys * hkv,
                "flops": 2 * sum(a * b for a, b in zip(lens, rows)) * hq * d}
    if kind == "evict":
        kept = sum(min(a, case["budget"]) for a in lens)
        return {"bytes": 8 * keys * hkv + 4 * kept * hkv + 4 * kept * row, "flops": keys * hkv}
    moved = n * (1 + case["most"]) / 2
    return {"bytes": 4 * moved * row + 4 * n * case["most"], "flops": 0}


# ---------------------------------------------------------------------------------------------
# The same outputs in 64 bits, sequence by sequence
# ---------------------------------------------------------------------------------------------

def _sequence(pool: torch.Tensor, table: torch.Tensor, n: int) -> torch.Tensor:
    return pool[table[:(n + PAGE - 1) // PAGE].long()].reshape(-1, pool.shape[2], pool.shape[3])[:n]


def _attention64(q, k, seen):
    """q [P, Hq, D], k [L, Hkv, D], seen [P, L] -> weights [Hq, P, L] of each query head."""
    group = q.shape[1] // k.shape[1]
    keys = k.double().permute(1, 2, 0).contiguous()
    out = []
    for h in range(q.shape[1]):
        x = torch.mm(q[:, h].double().contiguous(), keys[h // group]) * q.shape[2] ** -0.5
        out.append(torch.softmax(x.masked_fill(~seen, -math.inf), -1))
    return torch.stack(out)


def _values64(p, v):
    """p [Hq, P, L], v [L, Hkv, D] -> [P, Hq, D]."""
    group = p.shape[0] // v.shape[1]
    vals = v.double().permute(1, 0, 2).contiguous()
    return torch.stack([torch.mm(p[h], vals[h // group]) for h in range(p.shape[0])], 1)


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    kind, hkv = case["kind"], case["hkv"]
    if kind == "norm_rope":
        axis = torch.tensor(s["pair_axis"], device=DEVICE)
        angle = s["positions"].double().t()[:, axis] * s["inv_freq"].double()[None, :]
        z = torch.polar(torch.ones_like(angle), angle)[:, None, :]
        half, outs = case["d"] // 2, []
        for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
            y = x.double()
            y = y / (y.square().mean(-1, keepdim=True) + EPS).sqrt() * w.double()
            y = torch.complex(y[..., :half], y[..., half:]) * z
            outs.append(torch.cat([y.real, y.imag], -1))
        k_pool = s["k_pool"].double()
        k_pool.view(-1, hkv, case["d"])[s["slots"]] = outs[1]
        s["v_pool"].view(-1, hkv, case["d"])[s["slots"]] = s["v"]
        return outs[0], k_pool, s["v_pool"]
    if kind in ("tree", "mass", "window"):
        mass = s["mass"].double() if kind != "tree" else None
        cum = _cumsum(s["nodes"]) if kind != "mass" else list(range(case["batch"] + 1))
        outs = []
        for b, n in enumerate(s["lens"]):
            p = cum[b + 1] - cum[b]
            seen = torch.ones((p, n), dtype=torch.bool)
            if kind == "window":
                seen = torch.arange(n)[None, :] <= torch.arange(n - p, n)[:, None]
            if kind == "tree":
                seen[:, n - p:] = False
                for i, up in enumerate(s["parents"][b]):
                    if up >= 0:
                        seen[i, n - p:] = seen[up, n - p:]
                    seen[i, n - p + i] = True
            q = s["q"][cum[b]:cum[b + 1]]
            w = _attention64(q, _sequence(s["k_pool"], s["table"][b], n), seen.to(DEVICE))
            if kind != "window":
                outs.append(_values64(w, _sequence(s["v_pool"], s["table"][b], n)))
            if kind != "tree":
                mass[b, :, :n] += w.view(hkv, -1, n).sum(1)
        if kind == "window":
            return mass
        out = torch.cat(outs)
        return out if kind == "tree" else (out, mass)
    pools = (s["k_pool"], s["v_pool"])
    if kind == "commit":
        for b in range(case["batch"]):
            count, start = int(s["counts"][b]), int(s["start"][b])
            old = [_sequence(pool, s["table"][b], s["lens"][b]) for pool in pools]
            for i in range(count):
                to, at = start + i, int(s["keep"][b, 0, i])
                for pool, rows in zip(pools, old):
                    pool[int(s["table"][b, to // PAGE]), to % PAGE] = rows[at]
        return pools
    mass = s["mass"].cpu().double()
    keep = torch.full((*mass.shape[:2], case["budget"]), -1, dtype=torch.int32)
    total = torch.zeros(mass.shape, dtype=torch.float64)
    counts = [min(n, case["budget"]) for n in s["lens"]]
    for b, n in enumerate(s["lens"]):
        old = [_sequence(pool, s["table"][b], n) for pool in pools]
        to = torch.arange(counts[b], device=DEVICE)
        page = s["fresh"][b].long()[to // PAGE]
        for h in range(hkv):
            value = mass[b, h].tolist()
            order = sorted(range(n), key=lambda j: (case["sinks"] <= j < n - case["recent"], -value[j], j))
            kept = torch.tensor(sorted(order[:counts[b]]))
            keep[b, h, :counts[b]] = kept.to(torch.int32)
            total[b, h, :counts[b]] = mass[b, h][kept]
            for pool, rows in zip(pools, old):
                pool[page, to % PAGE, h] = rows[kept.to(DEVICE), h]
    return keep.to(DEVICE), _int32(counts), total.to(DEVICE), pools[0], pools[1]

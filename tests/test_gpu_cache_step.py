"""The cache step's further operators (norm + rotation + append, drafted trees, accumulated weights,
eviction) against plain implementations in 64 bits on the CPU.

Tolerances.  u is half a step of a type: 2^-24 (fp32), 2^-11 (fp16), 2^-8 (bf16).
* Rotation: the sum of D squares, the root, the weight, the angle (2^-23 of a turn's radian) and the
  products are fp32: at most 32 steps of 2^-24 of |y1| + |y2| together, then one rounding u |out|.
* Scores: sums of at most D / 4 dependent fp32 steps over terms of total size S = scale sum |q k|
  give each weight a relative error of e = 2 ((D / 4 + 8) S + 16) 2^-24 (its own score's, and the
  normalisation's).
* Attention: with A = sum p |v|, fp32 sums and weights (e + 32 2^-24) A; 16-bit pools also round each
  weight, u A, below 2^-14 of the largest by 2^-25 in fp16, and every type rounds the output, u |out|.
"""
import random

import pytest
import torch

from lightllm_amd import kv_cache as kc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
E = 2.0 ** -24
DTYPES = [F32, F16, BF16]
IDS = ["f32", "f16", "bf16"]


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def cum(values):
    out = [0]
    for v in values:
        out.append(out[-1] + v)
    return out


class Cache:
    """A paged cache on the CPU and its copy on the GPU; sequence b's rows are k[b], v[b] [L, Hkv, D]."""

    def __init__(self, lens, hkv, d, dtype, seed, bs=16, spare=3, garbage=None):
        g = torch.Generator().manual_seed(seed)
        need = [(n + bs - 1) // bs for n in lens]
        nb = sum(need) + spare
        self.bs, self.lens = bs, lens
        self.kp = torch.randn(nb, bs, hkv, d, generator=g).to(dtype)
        self.vp = torch.randn(nb, bs, hkv, d, generator=g).to(dtype)
        perm = torch.randperm(nb, generator=g).to(torch.int32)
        self.table = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = perm[at:at + n]
            at += n
        self.spare = perm[at:]
        if garbage is not None:     # what no sequence has written
            for b, n in enumerate(lens):
                if n % bs:
                    page = int(self.table[b, n // bs])
                    self.kp[page, n % bs:] = garbage
                    self.vp[page, n % bs:] = garbage
            for page in self.spare.tolist():
                self.kp[page] = garbage
                self.vp[page] = garbage
        self.k = [self.rows(self.kp, b) for b in range(len(lens))]
        self.v = [self.rows(self.vp, b) for b in range(len(lens))]

    def rows(self, pool, b):
        n = self.lens[b]
        return pool[self.table[b, :(n + self.bs - 1) // self.bs].long()].reshape(-1, *pool.shape[2:])[:n].clone()

    def put(self, b, pos, k=None, v=None):
        page, r = int(self.table[b, pos // self.bs]), pos % self.bs
        if k is not None:
            self.kp[page, r] = k
            self.k[b][pos] = k.to(self.kp.dtype) if isinstance(k, torch.Tensor) else k
        if v is not None:
            self.vp[page, r] = v
            self.v[b][pos] = v.to(self.vp.dtype) if isinstance(v, torch.Tensor) else v

    def gpu(self):
        return self.kp.to(DEV), self.vp.to(DEV), self.table.to(DEV), i32(self.lens)


def attend64(q, k, v, seen, scale):
    """q [P, Hq, D], k, v [L, Hkv, D], seen [P, L]: (out, tolerance without rounding terms, A,
    weights [Hq, P, L], e) in 64 bits; keys that a row does not see have no part in it."""
    p_, hq, d = q.shape
    group = hq // k.shape[1]
    out = torch.zeros(p_, hq, d, dtype=torch.float64)
    mean = torch.zeros_like(out)
    weights = torch.zeros(hq, p_, k.shape[0], dtype=torch.float64)
    err = 0.0
    for h in range(hq):
        kk, vv = k[:, h // group].double(), v[:, h // group].double()
        x = q[:, h].double() @ kk.t() * scale
        size = (q[:, h].double().abs() @ kk.abs().t() * scale)[seen & torch.isfinite(x)]
        if size.numel():
            err = max(err, 2 * ((d / 4 + 8) * float(size.max()) + 16) * E)
        for i in range(p_):
            s = seen[i].nonzero()[:, 0]
            if len(s) == 0:
                continue
            w = torch.softmax(x[i, s], 0)
            weights[h, i, s] = w
            out[i, h] = (w[:, None] * vv[s]).sum(0)
            mean[i, h] = (w[:, None] * vv[s].abs()).sum(0)
    return out, mean, weights, err


def check_attention(got, want, mean, err, dtype, keys, vmax, what=""):
    got, fine = got.cpu().double(), torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine), what
    assert torch.equal(got[torch.isinf(want)], want[torch.isinf(want)]), what
    tol = (err + 32 * E) * mean + U[dtype] * want.abs() + 1e-30
    if dtype != F32:
        tol = tol + U[dtype] * mean
    if dtype == F16:
        tol = tol + keys * 2.0 ** -25 * vmax + 2.0 ** -25
    bad = (got - want).abs()[fine] / tol[fine]
    worst = float(bad.max()) if bad.numel() else 0.0
    print(what, "error / bound %.3f" % worst, flush=True)
    assert worst <= 1.0, (what, worst)


# ---------------------------------------------------------------------------------------------
# qk_norm_rope_append
# ---------------------------------------------------------------------------------------------

def norm_rope64(x, w, eps, pos, freq, axis):
    """x [T, H, D] -> (out, |y1| + |y2| per element) in 64 bits."""
    y = x.double()
    if w is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    half = len(freq)
    size = y.abs()
    if half:
        phi = pos.double()[axis].t() * freq.double()
        c, s = phi.cos()[:, None], phi.sin()[:, None]
        a, b = y[..., :half], y[..., half:2 * half]
        y = torch.cat([a * c - b * s, b * c + a * s, y[..., 2 * half:]], -1)
        both = a.abs() + b.abs()
        size = torch.cat([both, both, size[..., 2 * half:]], -1)
    return y, size


ROPE = [  # hq, hkv, d, rotary, axes, tokens
    (14, 2, 64, 64, 1, 1), (32, 8, 128, 128, 1, 37), (28, 4, 128, 128, 3, 130), (16, 8, 256, 256, 1, 5),
    (32, 32, 96, 96, 3, 9), (4, 2, 128, 64, 2, 66), (5, 1, 67, 36, 4, 7), (3, 3, 80, 20, 1, 3),
    (2, 1, 16, 8, 1, 300), (4, 4, 8, 2, 1, 2), (6, 2, 64, 0, 1, 11), (1, 1, 72, 48, 1, 65)]


@pytest.mark.parametrize("shape", ROPE, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("form", ["fused", "in_place", "plain"])
def test_norm_rope(shape, dtype, form):
    hq, hkv, d, rot, axes, t = shape
    g = torch.Generator().manual_seed(hq * d + t)
    qkv = (torch.randn(t, hq + 2 * hkv, d, generator=g) * 3).to(dtype)
    qkv[0, 0] = 0                                    # a row of zeros: eps alone
    half = rot // 2
    pos = torch.randint(0, 2 ** 20, (axes, t), generator=g, dtype=torch.int32)
    pos[0, 0] = 2 ** 31 - 1
    pos[0, -1] = -5
    freq = (1e6 ** (-torch.arange(half).double() / max(half, 1))).float()
    axis = torch.randint(0, axes, (half,), generator=g)
    qw, kw = 1 + 0.2 * torch.randn(d, generator=g), 1 + 0.2 * torch.randn(d, generator=g)
    if form == "plain":
        qw = None
    nb = t // 16 + 3
    slots = torch.randperm(nb * 16, generator=g)[:t]
    if t > 1:
        slots[t // 2] = -1
    kp0, vp0 = (torch.randn(nb, 16, hkv, d, generator=g).to(dtype) for _ in range(2))
    dev = [x.to(DEV) for x in (qkv, kp0, vp0)]
    q, k, v = dev[0][:, :hq], dev[0][:, hq:hq + hkv], dev[0][:, hq + hkv:]
    before = dev[0].clone()
    kw_args = dict(q_weight=None if qw is None else qw.to(DEV), k_weight=kw.to(DEV), eps=1e-5,
                   pair_axis=None if axes == 1 else axis.tolist())
    p = pos[0].contiguous().to(DEV) if axes == 1 and form == "plain" else pos.to(DEV)
    if form == "in_place":
        kw_args.update(q_out=q, k_out=k)
    elif form == "plain":
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
        kw_args.update(k_out=torch.zeros_like(k))
    got = kc.qk_norm_rope_append(q, k, v, slots.to(DEV), p, freq.to(DEV), dev[1], dev[2], **kw_args)
    if axes == 1:
        axis = torch.zeros(half, dtype=torch.long)
    want_q, size_q = norm_rope64(qkv[:, :hq], qw, 1e-5, pos, freq, axis)
    want_k, size_k = norm_rope64(qkv[:, hq:hq + hkv], kw, 1e-5, pos, freq, axis)

    def close(a, want, size):
        tol = 32 * E * size + U[dtype] * want.abs() + (2.0 ** -25 if dtype == F16 else 1e-38)
        worst = float(((a.cpu().double() - want).abs() / tol).max())
        assert worst <= 1.0, worst
    close(got, want_q, size_q)
    ok = slots >= 0
    close(dev[1].view(-1, hkv, d)[slots[ok].to(DEV)], want_k[ok], size_k[ok])
    assert torch.equal(dev[2].view(-1, hkv, d)[slots[ok].to(DEV)].cpu(), qkv[ok, hq + hkv:])
    rest = torch.ones(nb * 16, dtype=torch.bool)
    rest[slots[ok]] = False
    for pool, old in ((dev[1], kp0), (dev[2], vp0)):   # rows of no slot are left as they were
        assert torch.equal(pool.cpu().view(-1, hkv, d)[rest], old.view(-1, hkv, d)[rest])
    if form == "fused":
        assert torch.equal(dev[0], before)
    else:
        close(kw_args["k_out"], want_k, size_k)


def test_norm_rope_without_queries_and_tokens():
    k = torch.randn(4, 2, 64, device=DEV)
    pools = [torch.zeros(2, 16, 2, 64, device=DEV) for _ in range(2)]
    freq = torch.ones(32, device=DEV)
    slots = torch.arange(4, device=DEV)
    pos = torch.zeros(4, dtype=torch.int32, device=DEV)
    assert kc.qk_norm_rope_append(None, k, k, slots, pos, freq, *pools) is None
    assert torch.equal(pools[0].view(-1, 2, 64)[:4], k) and torch.equal(pools[1].view(-1, 2, 64)[:4], k)
    out = kc.qk_norm_rope_append(k[:0], k[:0], k[:0], slots[:0], pos[:0], freq, *pools)
    assert out.shape == (0, 2, 64)


# ---------------------------------------------------------------------------------------------
# Drafted trees
# ---------------------------------------------------------------------------------------------

def make_tree(rng, n, kind):
    """Parents of n nodes."""
    if kind == "chain":
        return [i - 1 for i in range(n)]
    if kind == "star":
        return [-1] * n
    return [rng.randint(-1, i - 1) for i in range(n)]


def ancestors(parents):
    seen = torch.zeros(len(parents), len(parents), dtype=torch.bool)
    for i, p in enumerate(parents):
        if 0 <= p < i:
            seen[i] = seen[p]
        seen[i, i] = True
    return seen


def pack_mask(masks, words):
    rows = []
    for m in masks:
        for r in m.tolist():
            bits = sum(1 << j for j, x in enumerate(r) if x)
            rows.append([(bits >> 32 * w) & 0xFFFFFFFF for w in range(words)])
    x = torch.tensor(rows, dtype=torch.int64).view(-1, words)
    return torch.where(x >= 2 ** 31, x - 2 ** 32, x).to(torch.int32)


@pytest.mark.parametrize("sizes", [[1], [5, 0, 33, 64], [257, 1, 96], [5000]], ids=str)
def test_build_tree(sizes):
    rng = random.Random(len(sizes) + sizes[0])
    kinds = ["random", "chain", "star"]
    trees = [make_tree(rng, n, kinds[(i + n) % 3]) for i, n in enumerate(sizes)]
    trees[-1][-1] = len(trees[-1]) - 1              # its own parent: a root
    flat = [p for t in trees for p in t]
    lens = [n + 17 * i for i, n in enumerate(sizes)]
    words = (max(sizes) + 31) // 32 + 1
    mask = torch.full((len(flat), words), -1, dtype=torch.int32, device=DEV)
    got, pos = kc.build_tree(i32(flat), i32(cum(sizes)), i32(lens), max(sizes), tree_mask=mask)
    masks = [ancestors(t) for t in trees]
    if max(sizes) < 1000:
        assert torch.equal(got.cpu(), pack_mask(masks, words))
    want = torch.cat([m.sum(1) - 1 + n - s for m, n, s in zip(masks, lens, sizes)]).to(torch.int32)
    assert torch.equal(pos.cpu(), want)


LAYOUTS = [(14, 2, 64, 16), (8, 2, 128, 16), (4, 4, 96, 16), (8, 4, 256, 16), (7, 1, 80, 16), (4, 2, 64, 13),
           (3, 1, 67, 16), (48, 2, 64, 16), (34, 2, 256, 16)]
TREES = {
    "one": ([1], [0]),
    "short": ([3, 1, 7], [0, 2, 13]),
    "ragged": ([26, 1, 0, 33, 64], [512, 100, 37, 5, 63]),
    "wide": ([130], [200]),
    "long": ([5, 40], [3000, 1]),
}


@pytest.mark.parametrize("layout", LAYOUTS, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("trees", list(TREES))
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_tree_attention(layout, trees, dtype):
    hq, hkv, d, bs = layout
    nodes, contexts = TREES[trees]
    if (trees == "long" and d in (67, 80)) or (trees == "wide" and hq > 16):
        contexts = [n // 4 for n in contexts]
    rng = random.Random(hq + d + len(trees))
    lens = [a + b for a, b in zip(nodes, contexts)]
    c = Cache(lens, hkv, d, dtype, hq * d, bs, garbage=float("nan"))
    g = torch.Generator().manual_seed(5)
    q = torch.randn(sum(nodes), hq, d, generator=g).to(dtype)
    masks = [ancestors(make_tree(rng, n, "random")) for n in nodes]
    words = (max(nodes) + 31) // 32
    kp, vp, table, sl = c.gpu()
    got = kc.paged_tree_attention(q.to(DEV), kp, vp, table, i32(cum(nodes)), sl, pack_mask(masks, words).to(DEV),
                                  max(nodes), max(lens))
    at = cum(nodes)
    for b, n in enumerate(nodes):
        if n == 0:
            continue
        seen = torch.cat([torch.ones(n, contexts[b], dtype=torch.bool), masks[b]], 1)
        want, mean, _, err = attend64(q[at[b]:at[b + 1]], c.k[b], c.v[b], seen, d ** -0.5)
        check_attention(got[at[b]:at[b + 1]], want, mean, err, dtype, lens[b], float(c.v[b].abs().max()), f"tree {b}")


@pytest.mark.parametrize("d", [64, 256, 67])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_tree_masks_and_values_that_are_not_finite(d, dtype):
    """Rows that see nothing give zeros; a node's K and V reach the rows that see it and no other,
    whatever they hold; nodes whose own bit is not set; bits beyond the tree."""
    hq, hkv, n, ctx = 6, 2, 40, 0
    g = torch.Generator().manual_seed(d)
    c = Cache([n], hkv, d, dtype, 9, garbage=float("inf"))
    mask = torch.rand(n, n, generator=g) < 0.3
    mask[3] = False                     # no key at all: the context is empty
    mask[:, 5] = mask[:, 6] = mask[:, 7] = mask[:, 20] = False
    mask[8, 5] = mask[9, 6] = mask[10, 7] = mask[11, 20] = True
    c.put(0, 5, v=float("inf"))
    c.put(0, 6, k=float("nan"))
    c.put(0, 7, v=torch.where(torch.arange(d) == d - 1, float("nan"), 1.0).expand(hkv, d))
    c.put(0, 20, v=torch.where(torch.arange(d) % 5 == 0, float("-inf"), 2.0).expand(hkv, d))
    q = torch.randn(n, hq, d, generator=g).to(dtype)
    words = pack_mask([mask], 2)
    words[:, 1] |= -2 ** 31             # a bit beyond the tree's 40 nodes
    kp, vp, table, sl = c.gpu()
    got = kc.paged_tree_attention(q.to(DEV), kp, vp, table, i32([0, n]), sl, words.to(DEV), n, n)
    want, mean, _, err = attend64(q, c.k[0], c.v[0], mask, d ** -0.5)
    assert torch.all(got[3] == 0)
    assert torch.isnan(got[9]).all() and torch.isnan(want[9]).all()
    check_attention(got, want, mean, err, dtype, n, 4.0, f"d {d}")
    for row in (8, 10, 11):
        assert not torch.isfinite(want[row]).all()


def test_tree_more_rows_than_the_bounds_say():
    """max_q_len and max_seq_len size the launch only."""
    nodes, lens = [70, 9], [1500, 333]
    c = Cache(lens, 2, 64, F16, 3)
    q = torch.randn(79, 8, 64, generator=torch.Generator().manual_seed(1)).half().to(DEV)
    masks = [ancestors(make_tree(random.Random(i), n, "random")) for i, n in enumerate(nodes)]
    kp, vp, table, sl = c.gpu()
    words = pack_mask(masks, 3).to(DEV)
    full = kc.paged_tree_attention(q, kp, vp, table, i32(cum(nodes)), sl, words, 70, 1500)
    less = kc.paged_tree_attention(q, kp, vp, table, i32(cum(nodes)), sl, words, 17, 64)
    assert torch.all((full.float() - less.float()).abs() <= 2.0 ** -9 * (full.float().abs() + 1))


def test_tree_of_a_chain_is_a_causal_prefill():
    """A single branch sees what a causal chunk sees."""
    nodes, ctx = [33, 64, 5], [100, 999, 0]
    lens = [a + b for a, b in zip(nodes, ctx)]
    c = Cache(lens, 2, 128, BF16, 4)
    q = torch.randn(sum(nodes), 8, 128, generator=torch.Generator().manual_seed(2)).bfloat16().to(DEV)
    kp, vp, table, sl = c.gpu()
    flat = i32([i - 1 for n in nodes for i in range(n)])
    mask, pos = kc.build_tree(flat, i32(cum(nodes)), sl, 64)
    assert pos.tolist() == [a + i for n, a in zip(nodes, ctx) for i in range(n)]
    a = kc.paged_tree_attention(q, kp, vp, table, i32(cum(nodes)), sl, mask, 64, max(lens))
    b = kc.paged_prefill(q, kp, vp, table, i32(cum(nodes)), sl, 64, max(lens))
    # both within u (A + |out|) + the score terms of the same 64-bit value, and A <= max |v| < 6
    assert torch.all((a.double() - b.double()).abs() <= 2 * (2.0 ** -8 * (6 + a.double().abs())))


def test_many_sequences():
    """More sequences than one launch's prefix sums hold."""
    n = 1500
    nodes = [1 + i % 3 for i in range(n)]
    lens = [m + i % 50 for i, m in enumerate(nodes)]
    c = Cache(lens, 1, 64, F16, 8)
    g = torch.Generator().manual_seed(6)
    q = torch.randn(sum(nodes), 2, 64, generator=g).half()
    masks = [ancestors([i - 1 for i in range(m)]) for m in nodes]
    kp, vp, table, sl = c.gpu()
    got = kc.paged_tree_attention(q.to(DEV), kp, vp, table, i32(cum(nodes)), sl, pack_mask(masks, 1).to(DEV), 3,
                                  max(lens))
    mass = torch.zeros(n, 1, 64, device=DEV)
    out = kc.paged_decode_mass(q[:n].to(DEV), kp, vp, table, sl, max(lens), mass)
    at = cum(nodes)
    for b in list(range(0, 40)) + list(range(1015, 1035)) + [n - 1]:
        m = nodes[b]
        seen = torch.cat([torch.ones(m, lens[b] - m, dtype=torch.bool), masks[b]], 1)
        want, mean, _, err = attend64(q[at[b]:at[b + 1]], c.k[b], c.v[b], seen, 0.125)
        check_attention(got[at[b]:at[b + 1]], want, mean, err, F16, 64, 5.0, f"sequence {b}")
        want, mean, w, err = attend64(q[b:b + 1], c.k[b], c.v[b], torch.ones(1, lens[b], dtype=torch.bool), 0.125)
        check_attention(out[b:b + 1], want, mean, err, F16, 64, 5.0, f"decode {b}")
        check_mass(mass[b].cpu(), torch.zeros(1, 64), w.sum(1), lens[b], err, f"mass {b}")


# ---------------------------------------------------------------------------------------------
# Accumulated weights
# ---------------------------------------------------------------------------------------------

def check_mass(got, before, weights, n, err, what):
    """got, before [Hkv, width]; weights [Hq, L] of this call."""
    hkv = got.shape[0]
    add = weights.view(hkv, -1, n).sum(1)
    want = before[:, :n].double() + add
    tol = (err + 16 * E) * add + 2 * E * want.abs() + 1e-37
    worst = float(((got[:, :n].double() - want).abs() / tol).max()) if n else 0.0
    print(what, "error / bound %.3f" % worst, flush=True)
    assert worst <= 1.0, (what, worst)
    assert torch.equal(got[:, n:], before[:, n:]), what     # behind the last key: untouched


MASS_LAYOUTS = [(14, 2, 64, 16), (8, 2, 128, 16), (4, 4, 96, 16), (8, 4, 256, 16), (7, 1, 80, 16), (4, 2, 64, 13),
                (20, 1, 64, 16), (34, 2, 256, 16), (64, 1, 128, 16)]


@pytest.mark.parametrize("layout", MASS_LAYOUTS, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_decode_mass(layout, dtype):
    hq, hkv, d, bs = layout
    lens = [1, 16, 0, 517, 63, 2050, 64]
    c = Cache(lens, hkv, d, dtype, hq + d, bs, garbage=float("nan"))
    g = torch.Generator().manual_seed(3)
    q = torch.randn(len(lens), hq, d, generator=g).to(dtype)
    before = torch.rand(len(lens), hkv, 2300, generator=g)
    big = torch.zeros(len(lens), hkv + 1, 2300, device=DEV)       # a view with a stride of its own
    mass = big[:, :hkv]
    mass.copy_(before)
    kp, vp, table, sl = c.gpu()
    got = kc.paged_decode_mass(q.to(DEV), kp, vp, table, sl, 2050, mass)
    for b, n in enumerate(lens):
        if n == 0:
            assert torch.all(got[b] == 0)
            assert torch.equal(mass[b].cpu(), before[b])
            continue
        want, mean, w, err = attend64(q[b:b + 1], c.k[b], c.v[b], torch.ones(1, n, dtype=torch.bool), d ** -0.5)
        check_attention(got[b:b + 1], want, mean, err, dtype, n, float(c.v[b].abs().max()), f"out {b}")
        check_mass(mass[b].cpu(), before[b], w[:, 0], n, err, f"mass {b}")
    assert torch.all(big[:, hkv] == 0)


WINDOWS = {"one": ([1, 1], [1, 700]), "ragged": ([32, 5, 0, 64, 17], [1200, 5, 9, 64, 257]), "wide": ([150], [400])}


@pytest.mark.parametrize("layout", LAYOUTS, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("window", list(WINDOWS))
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_window_mass(layout, window, dtype):
    hq, hkv, d, bs = layout
    rows, lens = WINDOWS[window]
    c = Cache(lens, hkv, d, dtype, hq + d, bs, garbage=float("nan"))
    g = torch.Generator().manual_seed(3)
    q = torch.randn(sum(rows), hq, d, generator=g).to(dtype)
    before = torch.rand(len(lens), hkv, 1300, generator=g)
    mass = before.to(DEV)
    kp, vp, table, sl = c.gpu()
    kc.paged_window_mass(q.to(DEV), kp, table, i32(cum(rows)), sl, max(rows), max(lens), mass)
    at = cum(rows)
    for b, n in enumerate(lens):
        p = rows[b]
        seen = torch.arange(n)[None, :] <= torch.arange(n - p, n)[:, None]
        _, _, w, err = attend64(q[at[b]:at[b + 1]], c.k[b], c.v[b], seen, d ** -0.5)
        # sums of p G terms: (p G) 2^-24 at most
        check_mass(mass[b].cpu(), before[b], w.sum(1), n, err + p * hq // hkv * E, f"mass {b}")


def test_window_of_one_row_is_the_decode():
    lens = [300, 31]
    c = Cache(lens, 2, 64, F32, 7)
    q = torch.randn(2, 8, 64, generator=torch.Generator().manual_seed(1)).to(DEV)
    kp, vp, table, sl = c.gpu()
    a, b = torch.zeros(2, 2, 320, device=DEV), torch.zeros(2, 2, 320, device=DEV)
    kc.paged_decode_mass(q, kp, vp, table, sl, 300, a)
    kc.paged_window_mass(q, kp, table, i32([0, 1, 2]), sl, 1, 300, b)
    assert torch.all((a - b).abs() <= 1e-5 * a + 1e-12)
    assert torch.all((a.sum(2) - 4).abs() <= 1e-4)      # four heads' weights add up to four


# ---------------------------------------------------------------------------------------------
# Eviction
# ---------------------------------------------------------------------------------------------

def select64(mass, lens, budget, sinks, recent):
    n, hkv, width = mass.shape
    keep = torch.full((n, hkv, budget), -1, dtype=torch.int32)
    out = torch.zeros(n, hkv, width)
    for b in range(n):
        for h in range(hkv):
            m, size = mass[b, h].tolist(), lens[b]
            val = [float("-inf") if x != x else x for x in m]
            nan = [x != x for x in m]
            order = sorted(range(size), key=lambda j: (sinks <= j < size - recent, nan[j], -val[j], j))
            kept = sorted(order[:min(size, budget)])
            keep[b, h, :len(kept)] = torch.tensor(kept, dtype=torch.int32)
            out[b, h, :len(kept)] = mass[b, h, kept]
    return keep, [min(x, budget) for x in lens], out


def totals(g, n, hkv, width, kind):
    m = torch.randn(n, hkv, width, generator=g)
    if kind == "heavy":
        return (2 * m).exp() * (torch.rand(m.shape, generator=g) > 0.3)
    if kind == "ties":
        return (m * 2).round()
    if kind == "equal":
        return torch.full_like(m, 0.25)
    if kind == "odd":       # zeros of both signs, infinities, NaN, denormals, negative values
        pick = torch.tensor([0.0, -0.0, float("inf"), float("-inf"), float("nan"), 1e-40, -1e-40, 3.0, -3.0])
        return pick[torch.randint(0, 9, m.shape, generator=g)]
    return m


@pytest.mark.parametrize("kind", ["heavy", "ties", "equal", "odd", "normal"])
@pytest.mark.parametrize("budget,sinks,recent", [(1, 0, 0), (1, 1, 0), (40, 4, 9), (64, 0, 64), (500, 17, 100),
                                                 (1024, 4, 0), (4000, 4, 128)])
def test_evict_select(kind, budget, sinks, recent):
    g = torch.Generator().manual_seed(budget)
    lens = [1, budget, budget + 1, 3000, 0, 1025]
    lens = [min(n, 4100) for n in lens]
    width = 4160
    mass = totals(g, len(lens), 3, width, kind)
    keep, counts, out = kc.evict_select(mass.to(DEV), i32(lens), budget, 4100, sinks, recent)
    wk, wc, wo = select64(mass, lens, budget, sinks, recent)
    assert counts.tolist() == wc
    assert torch.equal(keep.cpu(), wk)
    assert torch.equal(out.cpu().view(torch.int32), wo.view(torch.int32))   # bit for bit, NaN too


@pytest.mark.parametrize("n", [4095, 16384, 16385, 40000, 70001, 131072])
@pytest.mark.parametrize("kind", ["heavy", "equal"])
def test_evict_select_long(n, kind):
    g = torch.Generator().manual_seed(n)
    mass = totals(g, 2, 1, n, kind)
    lens, budget = [n, n - 1000], n // 3
    keep, counts, out = kc.evict_select(mass.to(DEV), i32(lens), budget, n, 4, 700)
    wk, wc, wo = select64(mass, lens, budget, 4, 700)
    assert counts.tolist() == wc and torch.equal(keep.cpu(), wk) and torch.equal(out.cpu(), wo)


def moved(c, keep, counts, start, dst):
    """The CPU pools after the move, and the tables' row lookup."""
    kp, vp = c.kp.clone(), c.vp.clone()
    for b, count in enumerate(counts):
        for h in range(kp.shape[2]):
            src = keep[b, h if keep.shape[1] > 1 else 0]
            for i in range(count):
                s, t = int(src[i]), start[b] + i
                if not 0 <= s < c.table.shape[1] * c.bs or not 0 <= t < dst.shape[1] * c.bs:
                    continue
                sp, tp = int(c.table[b, s // c.bs]), int(dst[b, t // c.bs])
                if sp < 0 or tp < 0:
                    continue
                kp[tp, t % c.bs, h] = c.kp[sp, s % c.bs, h]
                vp[tp, t % c.bs, h] = c.vp[sp, s % c.bs, h]
    return kp, vp


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("layout", [(2, 64, 16), (8, 128, 16), (3, 67, 16), (4, 256, 13), (1, 96, 16), (5, 2, 16)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("heads", ["all", "each"])
def test_compact(in_place, layout, dtype, heads):
    hkv, d, bs = layout
    lens = [1, 700, 40, 16]
    c = Cache(lens, hkv, d, dtype, d, bs, spare=200)
    rng = random.Random(d)
    counts, start = [1, 511, 0, 16], [0, 30, 0, 0]
    m = 520
    keep = torch.full((4, hkv if heads == "each" else 1, m), -1, dtype=torch.int32)
    for b, n in enumerate(counts):
        for h in range(keep.shape[1]):
            if n:
                keep[b, h, :n] = torch.tensor(sorted(rng.sample(range(start[b], lens[b]), n)), dtype=torch.int32)
    pages = (m + 30 + bs - 1) // bs
    dst = None if in_place else c.spare[:4 * pages].view(4, pages).clone()
    if dst is not None:
        dst[1, 3] = -1          # a hole: its rows are not written
    wk, wv = moved(c, keep, counts, start, c.table if in_place else dst)
    kp, vp, table, _ = c.gpu()
    kc.compact_kv(kp, vp, table, keep.to(DEV), i32(counts), dst_table=None if in_place else dst.to(DEV),
                  dst_start=i32(start))
    assert torch.equal(kp.cpu(), wk) and torch.equal(vp.cpu(), wv)


def test_compact_positions_outside_the_tables():
    c = Cache([64, 64], 2, 64, F16, 1, spare=8)
    keep = torch.tensor([[[0, 63, 64, -1, 2 ** 31 - 1, 5]], [[1, 2, 3, 4, 5, 6]]], dtype=torch.int32)
    dst = c.spare[:2].view(2, 1).clone()
    start = [0, 13]             # the second sequence's rows run over its one page
    wk, wv = moved(c, keep, [6, 6], start, dst)
    kp, vp, table, _ = c.gpu()
    kc.compact_kv(kp, vp, table, keep.to(DEV), i32([6, 6]), dst_table=dst.to(DEV), dst_start=i32(start))
    assert torch.equal(kp.cpu(), wk) and torch.equal(vp.cpu(), wv)


@pytest.mark.parametrize("in_place", [False, True])
def test_evict_kv_then_decode(in_place):
    """After an eviction the decode attends exactly the kept rows, each head its own."""
    hq, hkv, d, budget = 8, 2, 64, 100
    lens = [700, 90, 333]
    c = Cache(lens, hkv, d, F32, 2, spare=30)
    g = torch.Generator().manual_seed(4)
    mass = totals(g, 3, hkv, 704, "heavy")
    wk, wc, wo = select64(mass, lens, budget, 2, 10)
    kp, vp, table, sl = c.gpu()
    dst = None if in_place else c.spare[:21].view(3, 7).contiguous().to(DEV)
    keep, counts, totals_ = kc.evict_kv(kp, vp, table, sl, mass.to(DEV), budget, 700, sinks=2, recent=10,
                                        dst_table=dst)
    assert torch.equal(keep.cpu(), wk) and counts.tolist() == wc and torch.equal(totals_.cpu(), wo)
    q = torch.randn(3, hq, d, generator=g)
    got = kc.paged_decode(q.to(DEV), kp, vp, table if in_place else dst, counts, budget)
    for b in range(3):
        rows = wk[b, :, :wc[b]].long()
        k = torch.stack([c.k[b][rows[h], h] for h in range(hkv)], 1)
        v = torch.stack([c.v[b][rows[h], h] for h in range(hkv)], 1)
        want, mean, _, err = attend64(q[b:b + 1], k, v, torch.ones(1, wc[b], dtype=torch.bool), d ** -0.5)
        check_attention(got[b:b + 1], want, mean, err, F32, wc[b], 5.0, f"sequence {b}")


# ---------------------------------------------------------------------------------------------
# Together
# ---------------------------------------------------------------------------------------------

def test_speculative_step_and_eviction():
    """One layer's life: a prompt's rows normed, rotated and appended; its keys weighed by the last
    rows; a tree drafted, read and its accepted branch committed; a decode step on the result that
    keeps its weights; the cache cut down; and a last decode.  Checked at every stage."""
    hq, hkv, d, dtype = 8, 2, 128, F16
    g = torch.Generator().manual_seed(11)
    prompt, tree = [130, 61], [-1, 0, 0, 1, 3, 2, -1, 4]
    P = len(tree)
    room = [n + P + 1 for n in prompt]
    c = Cache(room, hkv, d, dtype, 12, spare=20)
    kp, vp, table, _ = c.gpu()
    freq = (1e4 ** (-torch.arange(d // 2).double() / (d // 2))).float()
    qw, kw = 1 + 0.1 * torch.randn(d, generator=g), 1 + 0.1 * torch.randn(d, generator=g)

    def put_rows(counts, starts, positions):
        """Rows of a fused projection into the cache at positions starts + 0 .."""
        t = sum(counts)
        qkv = torch.randn(t, hq + 2 * hkv, d, generator=g).to(dtype).to(DEV)
        slots = kc.build_slots(table, i32(cum(counts)), i32(starts), t)
        return kc.qk_norm_rope_append(qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:], slots, positions,
                                      freq.to(DEV), kp, vp, q_weight=qw.to(DEV), k_weight=kw.to(DEV)).cpu()

    def rows(pool, b, n):
        return pool.cpu()[c.table[b, :(n + 15) // 16].long()].reshape(-1, hkv, d)[:n]

    pos = i32([p for n in prompt for p in range(n)])
    q = put_rows(prompt, [0, 0], pos)
    mass = torch.zeros(2, hkv, 160, device=DEV)
    last = [32, 32]
    qs = torch.cat([q[:130][-32:], q[130:][-32:]])
    kc.paged_window_mass(qs.to(DEV), kp, table, i32(cum(last)), i32(prompt), 32, 130, mass)
    for b, n in enumerate(prompt):
        seen = torch.arange(n)[None] <= torch.arange(n - 32, n)[:, None]
        _, _, w, err = attend64(qs[32 * b:32 * b + 32], rows(kp, b, n), rows(vp, b, n), seen, d ** -0.5)
        check_mass(mass[b].cpu(), torch.zeros(hkv, 160), w.sum(1), n, err + 128 * E, f"window {b}")

    lens = [n + P for n in prompt]
    mask, pos = kc.build_tree(i32(tree * 2), i32([0, P, 2 * P]), i32(lens), P)
    q = put_rows([P, P], prompt, pos)
    out = kc.paged_tree_attention(q.to(DEV), kp, vp, table, i32([0, P, 2 * P]), i32(lens), mask, P, max(lens))
    for b, n in enumerate(lens):
        seen = torch.cat([torch.ones(P, n - P, dtype=torch.bool), ancestors(tree)], 1)
        want, mean, _, err = attend64(q[b * P:b * P + P], rows(kp, b, n), rows(vp, b, n), seen, d ** -0.5)
        check_attention(out[b * P:b * P + P], want, mean, err, dtype, n, 5.0, f"tree {b}")

    accepted = [[0, 1, 3, 4, 7], [6]]
    old = [(rows(kp, b, n), rows(vp, b, n)) for b, n in enumerate(lens)]
    keep = torch.full((2, 1, 5), -1, dtype=torch.int32)
    for b, acc in enumerate(accepted):
        keep[b, 0, :len(acc)] = torch.tensor([prompt[b] + a for a in acc])
    kc.compact_kv(kp, vp, table, keep.to(DEV), i32([5, 1]), dst_start=i32(prompt))
    lens = [n + len(a) for n, a in zip(prompt, accepted)]
    for b, acc in enumerate(accepted):
        index = list(range(prompt[b])) + [prompt[b] + a for a in acc]
        assert torch.equal(rows(kp, b, lens[b]), old[b][0][index]) and torch.equal(rows(vp, b, lens[b]), old[b][1][index])

    q = put_rows([1, 1], lens, i32(lens))
    lens = [n + 1 for n in lens]
    before = mass.cpu().clone()
    out = kc.paged_decode_mass(q.to(DEV), kp, vp, table, i32(lens), max(lens), mass)
    for b, n in enumerate(lens):
        want, mean, w, err = attend64(q[b:b + 1], rows(kp, b, n), rows(vp, b, n), torch.ones(1, n, dtype=torch.bool),
                                      d ** -0.5)
        check_attention(out[b:b + 1], want, mean, err, dtype, n, 5.0, f"decode {b}")
        check_mass(mass[b].cpu(), before[b], w[:, 0], n, err, f"mass {b}")

    now = mass.cpu()
    wk, wc, wo = select64(now, lens, 64, 4, 16)
    old = [(rows(kp, b, n), rows(vp, b, n)) for b, n in enumerate(lens)]
    dst = c.spare[:8].view(2, 4).contiguous().to(DEV)
    got, counts, mass = kc.evict_kv(kp, vp, table, i32(lens), mass, 64, max(lens), 4, 16, dst_table=dst)
    assert torch.equal(got.cpu(), wk) and counts.tolist() == wc and torch.equal(mass.cpu(), wo)
    q = torch.randn(2, hq, d, generator=g).to(dtype)
    out = kc.paged_decode(q.to(DEV), kp, vp, dst, counts, 64)
    for b, n in enumerate(wc):
        index = wk[b, :, :n].long()
        k = torch.stack([old[b][0][index[h], h] for h in range(hkv)], 1)
        v = torch.stack([old[b][1][index[h], h] for h in range(hkv)], 1)
        want, mean, _, err = attend64(q[b:b + 1], k, v, torch.ones(1, n, dtype=torch.bool), d ** -0.5)
        check_attention(out[b:b + 1], want, mean, err, dtype, n, 5.0, f"after {b}")

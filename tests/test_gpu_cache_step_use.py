"""The cache step's further operators as a program uses them: captured and replayed, on streams, with the
caller's workspaces, beside cached prefixes, on large pools and long contexts.  Tolerances are those of
test_gpu_cache_step."""
import random

import pytest
import torch

from lightllm_amd import kv_cache as kc
from lightllm_amd._lib import LLKVError
from test_gpu_cache_step import (BF16, DEV, DTYPES, E, F16, F32, IDS, Cache, ancestors, attend64, check_attention,
                                 check_mass, cum, i32, make_tree, pack_mask)

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------
# A whole step, eager, captured, on streams
# ---------------------------------------------------------------------------------------------

class Step:
    """Buffers of one layer's step over every operator, and the step.  Lengths stay within the bounds that
    the calls are given."""
    HQ, HKV, D, P, MOST, BUDGET = 8, 2, 64, 7, 300, 64

    def __init__(self, seed):
        g = torch.Generator().manual_seed(seed)
        self.c = c = Cache([self.MOST] * 3, self.HKV, self.D, F16, seed, spare=12)
        self.kp0, self.vp0, self.table, _ = c.gpu()
        self.kp, self.vp = self.kp0.clone(), self.vp0.clone()
        self.dst = c.spare[:12].view(3, 4).contiguous().to(DEV)
        self.freq = (1e4 ** (-torch.arange(32).double() / 32)).float().to(DEV)
        self.w = (1 + 0.1 * torch.randn(self.D, generator=g)).to(DEV)
        self.cu = i32([0, 7, 14, 21])
        self.qkv = torch.empty(21, self.HQ + 2 * self.HKV, self.D, dtype=F16, device=DEV)
        self.parents, self.lens, self.start = (torch.zeros(n, dtype=torch.int32, device=DEV) for n in (21, 3, 3))
        self.keep = torch.zeros(3, 1, 3, dtype=torch.int32, device=DEV)
        self.counts = torch.zeros(3, dtype=torch.int32, device=DEV)
        self.mass = torch.zeros(3, self.HKV, self.MOST, device=DEV)

    def fill(self, seed):
        g = torch.Generator().manual_seed(seed)
        rng = random.Random(seed)
        lens = [rng.randint(self.P, self.MOST) for _ in range(3)]
        self.kp.copy_(self.kp0)
        self.vp.copy_(self.vp0)
        self.qkv.copy_(torch.randn(self.qkv.shape, generator=g).half())
        self.parents.copy_(torch.tensor([rng.randint(-1, i - 1) for _ in range(3) for i in range(self.P)]))
        self.lens.copy_(torch.tensor(lens))
        self.start.copy_(torch.tensor([n - self.P for n in lens]))
        self.keep.copy_(torch.tensor([[sorted(rng.sample(range(n - self.P, n), 3))] for n in lens]))
        self.counts.copy_(torch.tensor([rng.randint(0, 3) for _ in lens]))
        self.mass.copy_(torch.rand(self.mass.shape, generator=g))

    def run(self, stream=None):
        s = dict(stream=stream)
        q = self.qkv[:, :self.HQ]
        mask, pos = kc.build_tree(self.parents, self.cu, self.lens, self.P, **s)
        slots = kc.build_slots(self.table, self.cu, self.start, 21, **s)
        q = kc.qk_norm_rope_append(q, self.qkv[:, self.HQ:self.HQ + 2], self.qkv[:, self.HQ + 2:], slots, pos, self.freq,
                                   self.kp, self.vp, q_weight=self.w, k_weight=self.w, **s)
        tree = kc.paged_tree_attention(q, self.kp, self.vp, self.table, self.cu, self.lens, mask, self.P, self.MOST, **s)
        kc.paged_window_mass(q, self.kp, self.table, self.cu, self.lens, self.P, self.MOST, self.mass, **s)
        kc.compact_kv(self.kp, self.vp, self.table, self.keep, self.counts, dst_start=self.start, **s)
        dec = kc.paged_decode_mass(q[:3], self.kp, self.vp, self.table, self.lens, self.MOST, self.mass, **s)
        keep, counts, totals = kc.evict_kv(self.kp, self.vp, self.table, self.lens, self.mass, self.BUDGET, self.MOST, 4,
                                           16, dst_table=self.dst, **s)
        return [mask, pos, q, tree, self.mass, dec, keep, counts, totals, self.kp, self.vp]

    def eager(self, seed):
        self.fill(seed)
        out = [x.clone() for x in self.run()]
        torch.cuda.synchronize()
        return out


def same(got, want, what):
    for i, (a, b) in enumerate(zip(got, want)):
        assert torch.equal(a, b), (what, i)


def test_two_graphs_replayed_with_eager_work_between():
    """Every replay gives what the eager step gives, whatever ran since; two captured steps share nothing."""
    a, b = Step(1), Step(2)
    want = [[s.eager(seed) for seed in range(4)] for s in (a, b)]
    graphs, outs = [], []
    for s in (a, b):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            s.run()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(s.run())
        graphs.append(graph)
    for seed in (0, 3, 1, 2, 0):
        a.fill(seed)
        b.fill(seed)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            same(outs[i], want[i][seed], f"graph {i}, inputs {seed}")
        other = Step(3)             # eager work that uses the allocator
        other.eager(seed)


@pytest.mark.parametrize("form", ["argument", "context"])
def test_two_streams_at_once(form):
    steps = [Step(4), Step(5)]
    want = [s.eager(9) for s in steps]
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(3):
        outs = []
        for s in steps:
            s.fill(9)
        torch.cuda.synchronize()
        for s, st in zip(steps, streams):
            if form == "argument":
                outs.append(s.run(st))
            else:
                with torch.cuda.stream(st):
                    outs.append(s.run())
        torch.cuda.synchronize()
        for i in range(2):
            same(outs[i], want[i], f"stream {i}")


# ---------------------------------------------------------------------------------------------
# Workspaces, scales, bounds, addresses
# ---------------------------------------------------------------------------------------------

def small(dtype, d=64, hq=8, hkv=2, lens=(130, 17, 400), nodes=(5, 1, 20), seed=3, garbage=float("nan")):
    c = Cache(list(lens), hkv, d, dtype, seed, garbage=garbage)
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(sum(nodes), hq, d, generator=g).to(dtype)
    masks = [ancestors(make_tree(random.Random(seed + i), n, "random")) for i, n in enumerate(nodes)]
    return c, q, masks, pack_mask(masks, (max(nodes) + 31) // 32)


def test_workspaces_of_the_caller():
    """A workspace of the needed size serves call after call; a smaller one is refused."""
    c, q, _, words = small(F16)
    kp, vp, table, sl = c.gpu()
    cu, q, words = i32([0, 5, 6, 26]), q.to(DEV), words.to(DEV)
    mass = [torch.zeros(3, 2, 400, device=DEV) for _ in range(4)]
    L = kc.lib()
    sizes = [L.llkv_paged_tree_attention_workspace_size(3, 20, 8, 2, 64, 16, 400, 1),
             L.llkv_paged_decode_mass_workspace_size(3, 8, 2, 64, 16, 400, 1),
             L.llkv_paged_window_mass_workspace_size(26, 8, 400, 1), L.llkv_evict_select_workspace_size(3, 2, 20000)]
    ws = torch.full((max(sizes),), 255, dtype=torch.uint8, device=DEV)
    long = torch.rand(3, 2, 20000, device=DEV)
    calls = [lambda m, w: kc.paged_tree_attention(q, kp, vp, table, cu, sl, words, 20, 400, workspace=w),
             lambda m, w: (kc.paged_decode_mass(q[:3], kp, vp, table, sl, 400, m, workspace=w), m),
             lambda m, w: (kc.paged_window_mass(q, kp, table, cu, sl, 20, 400, m, workspace=w), m)[1],
             lambda m, w: kc.evict_select(long, i32([20000, 3, 16400]), 700, 20000, 4, 8, workspace=w)]
    flat = lambda x: [x] if isinstance(x, torch.Tensor) else list(x)
    for i, call in enumerate(calls):
        want = [x.clone() for x in flat(call(mass[0].zero_(), None))]
        for _ in range(2):
            same(flat(call(mass[1].zero_(), ws)), want, f"call {i}")
        with pytest.raises(LLKVError, match="workspace"):
            call(mass[2], ws[:sizes[i] - 1])


@pytest.mark.parametrize("scale", [-0.2, 0.0, 0.9])
@pytest.mark.parametrize("d", [64, 256, 67])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_scales(scale, d, dtype):
    c, q, masks, words = small(dtype, d)
    kp, vp, table, sl = c.gpu()
    cu = i32([0, 5, 6, 26])
    q64 = q if scale > 0 else -q if scale < 0 else torch.zeros_like(q)     # the same problem
    s64 = abs(scale) if scale else 1.0
    got = kc.paged_tree_attention(q.to(DEV), kp, vp, table, cu, sl, words.to(DEV), 20, 400, scale=scale)
    mass, win = (torch.zeros(3, 2, 400, device=DEV) for _ in range(2))
    dec = kc.paged_decode_mass(q[:3].to(DEV), kp, vp, table, sl, 400, mass, scale=scale)
    kc.paged_window_mass(q.to(DEV), kp, table, cu, sl, 20, 400, win, scale=scale)
    at = [0, 5, 6, 26]
    for b, n in enumerate(c.lens):
        rows, p, vmax = slice(at[b], at[b + 1]), at[b + 1] - at[b], float(c.v[b].abs().max())
        seen = torch.cat([torch.ones(p, n - p, dtype=torch.bool), masks[b]], 1)
        want, mean, _, err = attend64(q64[rows], c.k[b], c.v[b], seen, s64)
        check_attention(got[rows], want, mean, err, dtype, n, vmax, f"tree {b}")
        want, mean, w, err = attend64(q64[b:b + 1], c.k[b], c.v[b], torch.ones(1, n, dtype=torch.bool), s64)
        check_attention(dec[b:b + 1], want, mean, err, dtype, n, vmax, f"decode {b}")
        check_mass(mass[b].cpu(), torch.zeros(2, 400), w[:, 0], n, err, f"mass {b}")
        seen = torch.arange(n)[None] <= torch.arange(n - p, n)[:, None]
        _, _, w, err = attend64(q64[rows], c.k[b], c.v[b], seen, s64)
        check_mass(win[b].cpu(), torch.zeros(2, 400), w.sum(1), n, err + p * 4 * E, f"window {b}")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_totals_stop_at_the_bound(dtype):
    """Lengths beyond max_seq_len: as if they ended there."""
    c, q, _, _ = small(dtype)
    kp, vp, table, sl = c.gpu()
    q, cu = q.to(DEV), i32([0, 5, 6, 26])
    cut = sl.clamp(max=100)
    got = []
    for lens in (sl, cut):
        m = torch.zeros(3, 2, 100, device=DEV)
        out = kc.paged_decode_mass(q[:3], kp, vp, table, lens, 100, m)
        w = torch.zeros(3, 2, 100, device=DEV)
        kc.paged_window_mass(q, kp, table, cu, lens, 20, 100, w)
        got.append([out, m, w, *kc.evict_select(m, lens, 40, 100, 2, 5)])
    same(got[0], got[1], "bound")


def shifted(t):
    """The same values one element further than an aligned address."""
    raw = torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)
    out = raw[1:].view(t.shape)
    out.copy_(t)
    assert out.data_ptr() % 16 != 0
    return out


@pytest.mark.parametrize("dtype", [F32, F16], ids=["f32", "f16"])
def test_addresses_that_are_not_aligned(dtype):
    c, q, masks, words = small(dtype, 128)
    kp, vp, table, sl = c.gpu()
    cu, at = i32([0, 5, 6, 26]), [0, 5, 6, 26]
    out = shifted(torch.zeros(26, 8, 128, dtype=dtype))
    got = kc.paged_tree_attention(q.to(DEV), shifted(kp), shifted(vp), table, cu, sl, words.to(DEV), 20, 400, out=out)
    assert got is out
    mass, win = (shifted(torch.zeros(3, 2, 400)) for _ in range(2))
    dec = kc.paged_decode_mass(shifted(q[:3]), kp, vp, table, sl, 400, mass)
    kc.paged_window_mass(shifted(q), kp, table, cu, sl, 20, 400, win)
    for b, n in enumerate(c.lens):
        rows, p, vmax = slice(at[b], at[b + 1]), at[b + 1] - at[b], float(c.v[b].abs().max())
        seen = torch.cat([torch.ones(p, n - p, dtype=torch.bool), masks[b]], 1)
        want, mean, _, err = attend64(q[rows], c.k[b], c.v[b], seen, 128 ** -0.5)
        check_attention(got[rows], want, mean, err, dtype, n, vmax, f"tree {b}")
        want, mean, w, err = attend64(q[b:b + 1], c.k[b], c.v[b], torch.ones(1, n, dtype=torch.bool), 128 ** -0.5)
        check_attention(dec[b:b + 1], want, mean, err, dtype, n, vmax, f"decode {b}")
        check_mass(mass[b].cpu(), torch.zeros(2, 400), w[:, 0], n, err, f"mass {b}")
        seen = torch.arange(n)[None] <= torch.arange(n - p, n)[:, None]
        _, _, w, err = attend64(q[rows], c.k[b], c.v[b], seen, 128 ** -0.5)
        check_mass(win[b].cpu(), torch.zeros(2, 400), w.sum(1), n, err + p * 4 * E, f"window {b}")
    # moves and the norm, bit for bit what aligned tensors give
    pools = [[kp.clone(), vp.clone()], [shifted(kp), shifted(vp)]]
    keep = i32([[[3, 9, 16]], [[0, 1, 2]], [[7, 200, 399]]])
    freq, w = torch.rand(64, device=DEV), torch.rand(128, device=DEV)
    qs = []
    for i, (a, b) in enumerate(pools):
        kc.compact_kv(a, b, table, keep, i32([3, 2, 3]))
        x = q.to(DEV) if i == 0 else shifted(q)
        qs.append(kc.qk_norm_rope_append(x, x[:, :2], x[:, 2:4], torch.arange(26, device=DEV), i32(list(range(26))),
                                         freq, a, b, q_weight=w, k_weight=w if i == 0 else shifted(w)))
    for i in range(2):
        live = ~torch.isnan(pools[0][i])
        assert torch.equal(live, ~torch.isnan(pools[1][i]))
    assert torch.equal(pools[0][1][live], pools[1][1][live])
    # rotated rows: two orders of the same fp32 sum of squares, then one rounding
    u = E if dtype == F32 else 2.0 ** -11
    assert torch.all((qs[0].double() - qs[1].double()).abs() <= (64 * E + 2 * u) * 2 * qs[0].double().abs().amax(-1, True))


@pytest.mark.parametrize("layout", [(8, 2, 64, 16), (4, 2, 64, 13)], ids=lambda s: "x".join(map(str, s)))
def test_rows_behind_the_last_sequence(layout):
    """A padded batch: rows that no sequence has stay as they were."""
    hq, hkv, d, bs = layout
    c = Cache([40, 90], hkv, d, F32, 1, bs)
    q = torch.randn(20, hq, d, device=DEV)
    kp, vp, table, sl = c.gpu()
    cu = i32([0, 3, 11])
    mask, pos = torch.full((20, 1), 77, dtype=torch.int32, device=DEV), torch.full((20,), 78, dtype=torch.int32, device=DEV)
    kc.build_tree(i32([0] * 20), cu, sl, 8, tree_mask=mask, positions=pos)
    assert torch.all(mask[11:] == 77) and torch.all(pos[11:] == 78)
    out = torch.full((20, hq, d), 5.0, device=DEV)
    kc.paged_tree_attention(q, kp, vp, table, cu, sl, mask, 8, 90, out=out)
    assert torch.all(out[11:] == 5) and not torch.any(out[:11] == 5)
    a, b = torch.zeros(2, hkv, 96, device=DEV), torch.zeros(2, hkv, 96, device=DEV)
    kc.paged_window_mass(q, kp, table, cu, sl, 8, 90, a)
    kc.paged_window_mass(q[:11], kp, table, cu, sl, 8, 90, b)
    assert torch.equal(a, b)


# ---------------------------------------------------------------------------------------------
# Wide trees, large batches, shared prefixes, long contexts, large pools
# ---------------------------------------------------------------------------------------------

class Big:
    """A cache on the GPU whose tables may share a prefix; rows come to the CPU as they are checked."""

    def __init__(self, lens, hkv, d, dtype, shared=0, base=0, seed=1):
        g = torch.Generator(device=DEV).manual_seed(seed)
        need = [(n + 15) // 16 for n in lens]
        nb = shared + sum(m - shared for m in need)
        shape = (base + nb, 16, hkv, d)
        self.kp, self.vp = (torch.empty(shape, dtype=dtype, device=DEV) for _ in range(2))
        for pool in (self.kp, self.vp):
            pool[base:].normal_(generator=g)
        order = torch.randperm(nb, generator=torch.Generator().manual_seed(seed)) + base
        self.table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
        at = shared
        for b, m in enumerate(need):
            self.table[b, :shared] = order[:shared]
            self.table[b, shared:m] = order[at:at + m - shared]
            at += m - shared
        self.lens, self.dev_table, self.dev_lens = lens, self.table.to(DEV), i32(lens)

    def rows(self, pool, b, heads):
        n = self.lens[b]
        index = self.table[b, :(n + 15) // 16].long().to(DEV)
        return pool[index][:, :, heads].reshape(-1, len(heads), pool.shape[3])[:n].cpu()


def check_tree_rows(c, got, q, masks, nodes, hkv, dtype, seqs, heads, what):
    """Some rows and heads of some sequences against 64 bits."""
    at, group = cum(nodes), q.shape[1] // hkv
    for b in seqs:
        n, p = c.lens[b], nodes[b]
        k, v = c.rows(c.kp, b, heads), c.rows(c.vp, b, heads)
        pick = sorted({0, p // 3, p - 1})
        cols = [h * group + i for h in heads for i in (0, group - 1)]
        seen = torch.cat([torch.ones(p, n - p, dtype=torch.bool), masks[b]], 1)[pick]
        rows = torch.tensor([at[b] + i for i in pick])
        kk, vv = k.repeat_interleave(2, 1), v.repeat_interleave(2, 1)
        want, mean, _, err = attend64(q[rows][:, cols].cpu(), kk, vv, seen, q.shape[2] ** -0.5)
        check_attention(got[rows.to(DEV)][:, cols], want, mean, err, dtype, n, 6.0, f"{what}, sequence {b}")


WIDE = [  # dtype, hq, hkv, d, nodes, contexts
    (F16, 32, 8, 128, [64, 64, 62, 64, 64, 64, 64, 64], [4200, 4230, 4100, 4160, 4400, 4200, 4090, 4111]),   # 256 columns
    (BF16, 16, 4, 64, [61, 64, 64, 17], [17000, 16000, 17007, 16500]),
    (BF16, 8, 2, 96, [50, 60, 55], [900, 2000, 31]),        # units of 64
    (F16, 12, 2, 256, [40, 1, 33], [1500, 700, 2100]),      # two units of 128
    (F16, 4, 2, 256, [40, 20], [333, 2000]),                # one
    (F32, 16, 8, 64, [24, 20, 31, 9], [2100] * 4),
    (F32, 28, 4, 128, [64, 70], [2500, 3000]),
    (BF16, 14, 2, 64, [300, 2, 129], [500, 4000, 1]),
]


@pytest.mark.parametrize("case", WIDE, ids=lambda c: "x".join(map(str, c[1:4])))
def test_wide_trees(case):
    dtype, hq, hkv, d, nodes, contexts = case
    lens = [a + b for a, b in zip(nodes, contexts)]
    c = Big(lens, hkv, d, dtype)
    q = torch.randn(sum(nodes), hq, d, generator=torch.Generator().manual_seed(2)).to(dtype).to(DEV)
    masks = [ancestors(make_tree(random.Random(i), n, "random")) for i, n in enumerate(nodes)]
    words = pack_mask(masks, (max(nodes) + 31) // 32).to(DEV)
    got = kc.paged_tree_attention(q, c.kp, c.vp, c.dev_table, i32(cum(nodes)), c.dev_lens, words, max(nodes), max(lens))
    check_tree_rows(c, got, q, masks, nodes, hkv, dtype, range(min(len(nodes), 3)), [0, hkv - 1], "wide")


@pytest.mark.parametrize("shared", [0, 100], ids=["own", "prefix"])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
def test_batches_beyond_the_caches(shared, dtype):
    """More than 192 MB of keys and values, with and without a prefix that all sequences share."""
    hq, hkv, d, n = 16, 8, 128, 16
    nodes = [3 + i % 5 for i in range(n)]
    lens = [3300 + 37 * i for i in range(n)]
    c = Big(lens, hkv, d, dtype, shared)
    q = torch.randn(sum(nodes), hq, d, generator=torch.Generator().manual_seed(2)).to(dtype).to(DEV)
    masks = [ancestors(make_tree(random.Random(i), m, "random")) for i, m in enumerate(nodes)]
    got = kc.paged_tree_attention(q, c.kp, c.vp, c.dev_table, i32(cum(nodes)), c.dev_lens, pack_mask(masks, 1).to(DEV),
                                  max(nodes), max(lens))
    check_tree_rows(c, got, q, masks, nodes, hkv, dtype, (0, 7, 15), [0, 5], "tree")
    mass = torch.zeros(n, hkv, max(lens), device=DEV)
    out = kc.paged_decode_mass(q[:n], c.kp, c.vp, c.dev_table, c.dev_lens, max(lens), mass)
    check_decode_rows(c, out, mass, q[:n], hkv, dtype, (0, 15), 3, "decode")


def check_decode_rows(c, out, mass, q, hkv, dtype, seqs, head, what):
    group = q.shape[1] // hkv
    for b in seqs:
        n, cols = c.lens[b], slice(head * group, (head + 1) * group)
        k, v = c.rows(c.kp, b, [head]), c.rows(c.vp, b, [head])
        want, mean, w, err = attend64(q[b:b + 1, cols].cpu(), k, v, torch.ones(1, n, dtype=torch.bool), q.shape[2] ** -0.5)
        check_attention(out[b:b + 1, cols], want, mean, err, dtype, n, 6.0, f"{what}, sequence {b}")
        check_mass(mass[b, head:head + 1].cpu(), torch.zeros(1, mass.shape[2]), w[:, 0], n, err, f"{what}, sequence {b}")


@pytest.mark.parametrize("dtype,d", [(F16, 128), (F32, 64), (BF16, 96), (F32, 256)], ids=str)
def test_one_long_context(dtype, d):
    """One sequence over every work-group, its parts joined."""
    n, hq, p = 131077, 3, 5
    c = Big([n], 1, d, dtype)
    q = torch.randn(p, hq, d, generator=torch.Generator().manual_seed(2)).to(dtype).to(DEV)
    masks = [ancestors([-1, 0, 0, 1, -1])]
    got = kc.paged_tree_attention(q, c.kp, c.vp, c.dev_table, i32([0, p]), c.dev_lens, pack_mask(masks, 1).to(DEV), p, n)
    check_tree_rows(c, got, q, masks, [p], 1, dtype, [0], [0], "tree")
    mass = torch.zeros(1, 1, n, device=DEV)
    out = kc.paged_decode_mass(q[:1], c.kp, c.vp, c.dev_table, c.dev_lens, n, mass)
    check_decode_rows(c, out, mass, q[:1], 1, dtype, [0], 0, "decode")
    win = torch.zeros(1, 1, n, device=DEV)
    kc.paged_window_mass(q, c.kp, c.dev_table, i32([0, p]), c.dev_lens, p, n, win)
    seen = torch.arange(n)[None] <= torch.arange(n - p, n)[:, None]
    _, _, w, err = attend64(q.cpu(), c.rows(c.kp, 0, [0]), c.rows(c.vp, 0, [0]), seen, d ** -0.5)
    check_mass(win[0].cpu(), torch.zeros(1, n), w.sum(1), n, err + p * hq * E, "window")


@pytest.mark.parametrize("n", [40, 9000])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_queries_that_are_no_numbers(dtype, n):
    """Rows of NaN give NaN, and no other row does, whether or not their keys are cut into parts."""
    c = Big([n], 1, 64, dtype)
    q = torch.randn(3, 2, 64, generator=torch.Generator().manual_seed(2)).to(dtype).to(DEV)
    q[1] = float("nan")
    words = pack_mask([ancestors([-1, -1, -1])], 1).to(DEV)
    got = kc.paged_tree_attention(q, c.kp, c.vp, c.dev_table, i32([0, 3]), c.dev_lens, words, 3, n)
    assert torch.isnan(got[1]).all() and torch.isfinite(got[[0, 2]]).all()
    mass = torch.zeros(1, 1, n, device=DEV)
    out = kc.paged_decode_mass(q[1:2], c.kp, c.vp, c.dev_table, c.dev_lens, n, mass)
    assert torch.isnan(out).all() and torch.isnan(mass).all()
    win = torch.zeros(1, 1, n, device=DEV)
    kc.paged_window_mass(q[1:2], c.kp, c.dev_table, i32([0, 1]), c.dev_lens, 1, n, win)
    assert torch.isnan(win).all()


def test_pools_of_more_than_2_to_32_elements():
    """Rows whose offsets do not fit 32 bits."""
    hq, hkv, d, lens, nodes = 8, 8, 128, [700, 90], [9, 4]
    c = Big(lens, hkv, d, BF16, base=2 ** 32 // (16 * hkv * d) + 1)
    assert c.kp.numel() > 2 ** 32
    q = torch.randn(13, hq, d, generator=torch.Generator().manual_seed(2)).to(BF16).to(DEV)
    masks = [ancestors(make_tree(random.Random(i), n, "random")) for i, n in enumerate(nodes)]
    cu = i32(cum(nodes))
    # the nodes' rows by the append itself
    slots = kc.build_slots(c.dev_table, cu, i32([691, 86]), 13)
    assert int(slots.min()) * hkv * d > 2 ** 32
    new = torch.randn(13, 2 * hkv, d, generator=torch.Generator().manual_seed(3)).to(BF16).to(DEV)
    freq = torch.zeros(64, device=DEV)          # angles of zero: the rows as they are
    kc.qk_norm_rope_append(None, new[:, :hkv], new[:, hkv:], slots, i32(list(range(13))), freq, c.kp, c.vp)
    assert torch.equal(c.rows(c.kp, 0, list(range(8)))[691:], new[:9, :hkv].cpu())
    assert torch.equal(c.rows(c.vp, 1, list(range(8)))[86:], new[9:, hkv:].cpu())
    got = kc.paged_tree_attention(q, c.kp, c.vp, c.dev_table, cu, c.dev_lens, pack_mask(masks, 1).to(DEV), 9, 700)
    check_tree_rows(c, got, q, masks, nodes, hkv, BF16, (0, 1), [0, 7], "tree")
    mass = torch.zeros(2, hkv, 700, device=DEV)
    out = kc.paged_decode_mass(q[:2], c.kp, c.vp, c.dev_table, c.dev_lens, 700, mass)
    check_decode_rows(c, out, mass, q[:2], hkv, BF16, (0, 1), 7, "decode")
    win = torch.zeros(2, hkv, 700, device=DEV)
    kc.paged_window_mass(q, c.kp, c.dev_table, cu, c.dev_lens, 9, 700, win)
    seen = torch.arange(700)[None] <= torch.arange(691, 700)[:, None]
    _, _, w, err = attend64(q[:9, 7:].cpu(), c.rows(c.kp, 0, [7]), c.rows(c.vp, 0, [7]), seen, d ** -0.5)
    check_mass(win[0, 7:].cpu(), torch.zeros(1, 700), w.sum(1), 700, err + 9 * E, "window")
    # a move to the sequence's own pages and one to others
    old = [c.rows(p, 0, list(range(8))) for p in (c.kp, c.vp)]
    kc.compact_kv(c.kp, c.vp, c.dev_table[:1], i32([[[690, 692, 699]]]), i32([3]), dst_start=i32([690]))
    for p, o in zip((c.kp, c.vp), old):
        assert torch.equal(c.rows(p, 0, list(range(8)))[690:693], o[[690, 692, 699]])
    kc.compact_kv(c.kp, c.vp, c.dev_table[:1], i32([[[5, 5, 600]]]), i32([3]), dst_table=c.dev_table[1:])   # one row twice
    for p, o in zip((c.kp, c.vp), old):
        assert torch.equal(c.rows(p, 1, list(range(8)))[:3], o[[5, 5, 600]])

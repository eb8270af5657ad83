"""What the cache step's further operators refuse, on the CPU: the C calls before they touch a device
(addresses that are never read), the Python calls before they reach the library."""
import ctypes

import pytest
import torch

from lightllm_amd import _lib as L
from lightllm_amd import kv_cache as kc

P = ctypes.c_void_p(0x1000)      # never dereferenced: the checks fail first
N = None


def err(rc):
    return rc, L.last_error()


def norm_rope(q_out=P, k_out=N, q=P, k=P, v=P, strides=(512, 128, 512, 128, 128), slots=P, pos=P, axes=1,
              pair_axis=N, freq=P, qw=P, kw=P, eps=1e-6, t=4, hq=8, hkv=2, d=64, rot=64, dt=0, kp=P, vp=P):
    return err(L.lib().llkv_qk_norm_rope_append(q_out, k_out, q, k, v, *strides, kp, vp, slots, pos, axes, pair_axis,
                                                freq, qw, kw, eps, t, hq, hkv, d, rot, dt, N))


@pytest.mark.parametrize("args,status,word", [
    (dict(t=-1), 1, "shape"), (dict(hkv=0), 1, "shape"), (dict(hq=0), 1, "shape"), (dict(d=257, rot=64), 2, "256"),
    (dict(rot=63), 1, "rotary_dim"), (dict(rot=66), 1, "rotary_dim"), (dict(rot=-2), 1, "rotary_dim"),
    (dict(dt=3), 1, "dtype"), (dict(k=N), 1, "null"), (dict(v=N), 1, "null"), (dict(kp=N), 1, "null"),
    (dict(vp=N), 1, "null"), (dict(slots=N), 1, "null"), (dict(q_out=N), 1, "null"), (dict(pos=N), 1, "null"),
    (dict(freq=N), 1, "null"), (dict(axes=0), 1, "num_axes"), (dict(axes=5), 1, "num_axes"),
    (dict(axes=2), 1, "pair_axis"), (dict(axes=2, pair_axis=bytes([0] * 31 + [2])), 1, "pair_axis[31]"),
    (dict(eps=-1.0), 1, "eps"), (dict(eps=float("nan")), 1, "eps"),
    (dict(strides=(500, 128, 512, 128, 128)), 1, "strides"), (dict(strides=(512, 128, 512, -1, 128)), 1, "strides"),
    (dict(strides=(512, 100, 512, 128, 128), k_out=P), 1, "strides"), (dict(t=2 ** 30), 2, "rows"),
], ids=str)
def test_norm_rope(args, status, word):
    rc, msg = norm_rope(**args)
    assert rc == status and word in msg, (rc, msg)


def tree(out=P, q=P, k=P, v=P, table=P, blocks=8, cu=P, lens=P, mask=P, words=2, n=2, total=9, most=40, longest=100,
         hq=8, hkv=2, d=64, bs=16, dt=0, ws=P, nbytes=1 << 40):
    return err(L.lib().llkv_paged_tree_attention(out, q, k, v, table, blocks, cu, lens, mask, words, n, total, most,
                                                 longest, hq, hkv, d, bs, 0.1, dt, ws, nbytes, N))


ATTENTION = [(dict(n=-1), 1, "shape"), (dict(hq=0), 1, "shape"), (dict(bs=0), 1, "shape"), (dict(blocks=0), 1, "shape"),
             (dict(longest=-1), 1, "shape"), (dict(d=300), 2, "256"), (dict(hq=7), 1, "multiple"), (dict(dt=3), 1, "dtype"),
             (dict(blocks=1 << 28), 2, "too large"), (dict(q=N), 1, "null"), (dict(k=N), 1, "null"),
             (dict(table=N), 1, "null"), (dict(lens=N), 1, "null")]


@pytest.mark.parametrize("args,status,word", ATTENTION + [
    (dict(words=1), 1, "mask"), (dict(words=0), 1, "mask"), (dict(most=0), 1, "mask"), (dict(total=-1), 1, "mask"),
    (dict(out=N), 1, "null"), (dict(v=N), 1, "null"), (dict(cu=N), 1, "null"), (dict(mask=N), 1, "null"),
    (dict(total=2 ** 31 - 1), 2, "too many"), (dict(nbytes=0), 3, "workspace"), (dict(ws=N), 3, "workspace"),
    (dict(ws=ctypes.c_void_p(0x1008)), 1, "aligned"),
], ids=str)
def test_tree_attention(args, status, word):
    rc, msg = tree(**args)
    assert rc == status and word in msg, (rc, msg)


def decode_mass(out=P, mass=P, strides=(200, 100), q=P, k=P, v=P, table=P, lens=P, n=2, hq=8, hkv=2, d=64, bs=16, blocks=8,
                longest=100, dt=0, ws=P, nbytes=1 << 40):
    return err(L.lib().llkv_paged_decode_mass(out, mass, *strides, q, k, v, table, lens, n, hq, hkv, d, bs, blocks,
                                              longest, 0.1, dt, ws, nbytes, N))


@pytest.mark.parametrize("args,status,word", ATTENTION + [
    (dict(out=N), 1, "null"), (dict(mass=N), 1, "null"), (dict(v=N), 1, "null"), (dict(strides=(200, 99)), 1, "totals"),
    (dict(strides=(199, 100)), 1, "totals"), (dict(hq=130), 2, "64 query heads"), (dict(nbytes=0), 3, "workspace"),
    (dict(ws=N), 3, "workspace"),
], ids=str)
def test_decode_mass(args, status, word):
    rc, msg = decode_mass(**args)
    assert rc == status and word in msg, (rc, msg)


def window(mass=P, strides=(200, 100), q=P, k=P, table=P, blocks=8, cu=P, lens=P, n=2, total=9, most=5, longest=100, hq=8,
           hkv=2, d=64, bs=16, dt=0, ws=P, nbytes=1 << 40):
    return err(L.lib().llkv_paged_window_mass(mass, *strides, q, k, table, blocks, cu, lens, n, total, most, longest, hq,
                                              hkv, d, bs, 0.1, dt, ws, nbytes, N))


@pytest.mark.parametrize("args,status,word", ATTENTION + [
    (dict(mass=N), 1, "null"), (dict(cu=N), 1, "null"), (dict(strides=(200, 99)), 1, "totals"),
    (dict(strides=(199, 100)), 1, "totals"), (dict(most=0), 1, "shape"), (dict(nbytes=0), 3, "workspace"),
    (dict(ws=N), 3, "workspace"), (dict(ws=ctypes.c_void_p(0x1008)), 1, "aligned"),
], ids=str)
def test_window_mass(args, status, word):
    rc, msg = window(**args)
    assert rc == status and word in msg, (rc, msg)


def select(keep=P, counts=P, out=P, out_strides=(200, 100), width=100, mass=P, strides=(200, 100), lens=P, n=2, hkv=2,
           longest=100, budget=50, sinks=4, recent=16, ws=P, nbytes=1 << 40):
    return err(L.lib().llkv_evict_select(keep, counts, out, *out_strides, width, mass, *strides, lens, n, hkv, longest,
                                         budget, sinks, recent, ws, nbytes, N))


@pytest.mark.parametrize("args,status,word", [
    (dict(n=-1), 1, "shape"), (dict(hkv=0), 1, "shape"), (dict(longest=-1), 1, "shape"), (dict(budget=0), 1, "budget"),
    (dict(sinks=-1), 1, "budget"), (dict(recent=-1), 1, "budget"), (dict(sinks=40), 1, "budget"),
    (dict(keep=N), 1, "null"), (dict(counts=N), 1, "null"), (dict(out=N), 1, "null"), (dict(mass=N), 1, "null"),
    (dict(lens=N), 1, "null"), (dict(strides=(200, 99)), 1, "totals"), (dict(strides=(199, 100)), 1, "totals"),
    (dict(width=49), 1, "totals"), (dict(width=101), 1, "totals"), (dict(out_strides=(199, 100)), 1, "totals"),
    (dict(n=65536), 2, "too many"), (dict(longest=20000, strides=(40000, 20000), ws=N), 3, "workspace"),
    (dict(longest=20000, strides=(40000, 20000), nbytes=100), 3, "workspace"),
    (dict(ws=ctypes.c_void_p(0x1004)), 1, "aligned"),
], ids=str)
def test_evict_select(args, status, word):
    rc, msg = select(**args)
    assert rc == status and word in msg, (rc, msg)


def compact(k=P, v=P, src=P, src_blocks=8, dst=P, dst_blocks=4, keep=P, heads=2, most=50, counts=P, start=N, n=2, hkv=2,
            d=64, bs=16, dt=0):
    return err(L.lib().llkv_compact(k, v, src, src_blocks, dst, dst_blocks, keep, heads, most, counts, start, n, hkv, d,
                                    bs, dt, N))


@pytest.mark.parametrize("args,status,word", [
    (dict(n=-1), 1, "shape"), (dict(most=-1), 1, "shape"), (dict(hkv=0), 1, "shape"), (dict(d=0), 1, "shape"),
    (dict(bs=0), 1, "shape"), (dict(src_blocks=0), 1, "shape"), (dict(dst_blocks=0), 1, "shape"), (dict(heads=3), 1, "heads"),
    (dict(heads=0), 1, "heads"), (dict(dt=3), 1, "dtype"), (dict(k=N), 1, "null"), (dict(v=N), 1, "null"),
    (dict(src=N), 1, "null"), (dict(keep=N), 1, "null"), (dict(counts=N), 1, "null"),
    (dict(src_blocks=1 << 27), 2, "too large"),
], ids=str)
def test_compact(args, status, word):
    rc, msg = compact(**args)
    assert rc == status and word in msg, (rc, msg)


def test_build_tree():
    f = L.lib().llkv_build_tree
    assert err(f(P, 1, P, P, P, P, 2, 9, 33, N))[0] == 1
    assert err(f(P, 0, P, P, P, P, 2, 9, 1, N))[0] == 1
    for bad in range(4):
        a = [P, P, P, P]
        a[bad] = N
        mask, positions, parents, cu = a[0], P, a[1], a[2]
        rc = f(mask, 2, positions, parents, cu, a[3], 2, 9, 40, N)
        assert rc == 1 and "null" in L.last_error()


def test_nothing_to_do():
    """Empty batches are no error, as for the other operators, whatever the pointers."""
    assert norm_rope(t=0, k=N)[0] == 0
    assert tree(n=0, q=N)[0] == 0 and tree(total=0, q=N)[0] == 0
    assert decode_mass(n=0, q=N)[0] == 0
    assert window(n=0, q=N)[0] == 0 and window(total=0, q=N)[0] == 0
    assert select(n=0, mass=N)[0] == 0
    assert compact(n=0, k=N)[0] == 0 and compact(most=0, k=N)[0] == 0
    assert L.lib().llkv_build_tree(N, 1, N, N, N, N, 0, 0, 1, N) == 0


def test_workspace_sizes_of_bad_shapes():
    lib = L.lib()
    assert lib.llkv_paged_tree_attention_workspace_size(0, 4, 8, 2, 64, 16, 100, 0) == 0
    assert lib.llkv_paged_tree_attention_workspace_size(2, 4, 7, 2, 64, 16, 100, 0) == 0
    assert lib.llkv_paged_tree_attention_workspace_size(2, 4, 8, 2, 64, 16, 100, 3) == 0
    assert lib.llkv_paged_decode_mass_workspace_size(2, 7, 2, 64, 16, 100, 0) == 0
    assert lib.llkv_paged_window_mass_workspace_size(0, 8, 100, 0) == 0
    # scores: four bytes for every query head and key, in whole tiles
    assert lib.llkv_paged_decode_mass_workspace_size(2, 8, 2, 67, 16, 100, 0) == 2 * 8 * 128 * 4


def cpu(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def test_python_calls_refuse_tensors_of_the_host():
    """An address of host memory never reaches a kernel."""
    pool, i = cpu(4, 16, 2, 64), cpu(2, dtype=torch.int32)
    table, cu, mass = cpu(2, 4, dtype=torch.int32), cpu(3, dtype=torch.int32), cpu(2, 2, 64)
    q = cpu(2, 8, 64)
    for call in (
            lambda: kc.qk_norm_rope_append(q, cpu(2, 2, 64), cpu(2, 2, 64), cpu(2, dtype=torch.int64), i, cpu(32), pool, pool),
            lambda: kc.build_tree(i, cu, i, 2),
            lambda: kc.paged_tree_attention(q, pool, pool, table, cu, i, cpu(2, 1, dtype=torch.int32), 1, 64),
            lambda: kc.paged_decode_mass(q, pool, pool, table, i, 64, mass),
            lambda: kc.paged_window_mass(q, pool, table, cu, i, 1, 64, mass),
            lambda: kc.evict_select(mass, i, 8, 64),
            lambda: kc.compact_kv(pool, pool, table, cpu(2, 1, 4, dtype=torch.int32), i),
            lambda: kc.evict_kv(pool, pool, table, i, mass, 8, 64)):
        with pytest.raises(ValueError, match="GPU"):
            call()

"""Python mirror of the reference's paged KV-cache operator API
(include/lightllm/kv_cache/paged_attention.h:31-145 and
block_allocator.h:37-186 of wjb554/lightllm), over the C ABI.

Torch provides device memory and the stream; every computation runs in the
gfx950 kernels of liblightllm_kv.so.  Device index arrays are int32 (block
tables, lengths, offsets) except slot mappings (int64).
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import Optional, Sequence, Union

import torch

from ._lib import DTYPE_BF16, DTYPE_F16, DTYPE_F32, check, lib

_TORCH_TO_DT = {torch.float32: DTYPE_F32, torch.float16: DTYPE_F16, torch.bfloat16: DTYPE_BF16}
_DT_TO_TORCH = {v: k for k, v in _TORCH_TO_DT.items()}

POLICY_HASH, POLICY_RADIX = 0, 1
STORAGE_DEVICE, STORAGE_HOST, STORAGE_NONE = 0, 1, 2


def dtype_code(t: torch.dtype) -> int:
    try:
        return _TORCH_TO_DT[t]
    except KeyError:
        raise ValueError(f"unsupported dtype {t}") from None


# The smallest calls are bound by the host, so a call passes addresses as plain
# integers (the argument types of _lib.py convert them) and asks for the raw
# current stream: a one-sequence append + decode 15.0 -> 10.3 .. 12.0 us a call, also with
# max_seq_len growing by one from call to call.
def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _stream(stream=None):
    if stream is not None:
        return stream.cuda_stream
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _require(t: torch.Tensor, dtype: torch.dtype, name: str):
    if t.dtype != dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: must be contiguous")


class BlockAllocator:
    """Block pool + prefix cache (reference BlockAllocator semantics, implemented in
    C++).  K/V pools are torch tensors [num_blocks, block_size, Hkv, D] on `device`
    (or none with device=None, metadata only)."""

    def __init__(self, num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int,
                 policy: int = POLICY_HASH, kv_dtype: torch.dtype = torch.float32,
                 device: Optional[str] = "cuda"):
        self.num_blocks, self.block_size = num_blocks, block_size
        self.num_kv_heads, self.head_dim = num_kv_heads, head_dim
        self.kv_dtype, self.policy = kv_dtype, policy
        h = ctypes.c_void_p()
        check(lib().llkv_allocator_create(num_blocks, block_size, num_kv_heads, head_dim, policy,
                                          dtype_code(kv_dtype), STORAGE_NONE, ctypes.byref(h)))
        self._h = h
        if device is not None:
            shape = (num_blocks, block_size, num_kv_heads, head_dim)
            self.k_storage = torch.zeros(shape, dtype=kv_dtype, device=device)
            self.v_storage = torch.zeros(shape, dtype=kv_dtype, device=device)
        else:
            self.k_storage = self.v_storage = None

    @staticmethod
    def blocks_for_budget(budget_bytes: int, block_size: int, num_kv_heads: int, head_dim: int,
                          kv_dtype: torch.dtype) -> int:
        """Pages (K and V) that fit `budget_bytes` in the pool's element type."""
        n = lib().llkv_blocks_for_budget(budget_bytes, block_size, num_kv_heads, head_dim,
                                         dtype_code(kv_dtype))
        if n < 0:
            raise ValueError("blocks_for_budget: bad arguments")
        return n

    def __del__(self):
        h = getattr(self, "_h", None)
        if h is not None and h.value:
            lib().llkv_allocator_destroy(h)
            self._h = None

    # ---- allocation --------------------------------------------------------
    def allocate(self, token_hash: int = 0) -> int:
        return lib().llkv_allocator_allocate(self._h, token_hash)

    def allocate_tokens(self, tokens: Sequence[int], start_pos: int):
        """Returns (n_new, all_block_ids)."""
        arr = (ctypes.c_int * max(1, len(tokens)))(*tokens)
        cap = len(tokens) // self.block_size + 2
        out = (ctypes.c_int * cap)()
        cnt = ctypes.c_int(0)
        n_new = lib().llkv_allocator_allocate_tokens(self._h, arr, len(tokens), start_pos, out, cap,
                                                     ctypes.byref(cnt))
        return n_new, list(out[: cnt.value])

    def release(self, block_id: int) -> None:
        lib().llkv_allocator_release(self._h, block_id)

    def find_by_hash(self, token_hash: int) -> int:
        return lib().llkv_allocator_find_by_hash(self._h, token_hash)

    def find_cached_prefix(self, tokens: Sequence[int], start_pos: int):
        """Returns (matched_tokens, block_ids)."""
        arr = (ctypes.c_int * max(1, len(tokens)))(*tokens)
        cap = len(tokens) // self.block_size + 2
        out = (ctypes.c_int * cap)()
        n = ctypes.c_int(0)
        matched = lib().llkv_allocator_find_cached_prefix(self._h, arr, len(tokens), start_pos, out,
                                                          cap, ctypes.byref(n))
        return matched, list(out[: n.value])

    def insert_cached_blocks(self, tokens: Sequence[int], start_pos: int,
                             block_ids: Sequence[int]) -> None:
        arr = (ctypes.c_int * max(1, len(tokens)))(*tokens)
        ids = (ctypes.c_int * max(1, len(block_ids)))(*block_ids)
        lib().llkv_allocator_insert_cached_blocks(self._h, arr, len(tokens), start_pos, ids,
                                                  len(block_ids))

    def evict_lru(self) -> int:
        return lib().llkv_allocator_evict_lru(self._h)

    def increment_ref(self, block_id: int) -> None:
        lib().llkv_allocator_increment_ref(self._h, block_id)

    def reset(self) -> None:
        check(lib().llkv_allocator_reset(self._h))
        if self.k_storage is not None:
            self.k_storage.zero_()
            self.v_storage.zero_()

    # ---- inspection --------------------------------------------------------
    def num_free(self) -> int:
        return lib().llkv_allocator_num_free(self._h)

    def ref_count(self, block_id: int) -> int:
        return lib().llkv_allocator_ref_count(self._h, block_id)

    def token_hash(self, block_id: int) -> int:
        return lib().llkv_allocator_token_hash(self._h, block_id)

    def prefix_cache_size(self) -> int:
        return lib().llkv_allocator_prefix_cache_size(self._h)


def hash_tokens(tokens: Sequence[int]) -> int:
    arr = (ctypes.c_int * max(1, len(tokens)))(*tokens)
    return lib().llkv_hash_tokens(arr, len(tokens))


# ---------------------------------------------------------------------------
# Operators
# ---------------------------------------------------------------------------

def append_kv(k: torch.Tensor, v: torch.Tensor, slot_mapping: torch.Tensor,
              k_pool: torch.Tensor, v_pool: torch.Tensor, stream=None) -> None:
    """KV append by slot mapping: row i of k/v -> pool row slot_mapping[i] (int64, <0 skips)."""
    _require(slot_mapping, torch.int64, "slot_mapping")
    _require(k, k_pool.dtype, "k")
    _require(v, k_pool.dtype, "v")
    hkv, d = k_pool.shape[2], k_pool.shape[3]
    check(lib().llkv_append(_ptr(k_pool), _ptr(v_pool), _ptr(k), _ptr(v), _ptr(slot_mapping),
                            k.shape[0], hkv, d, dtype_code(k_pool.dtype), _stream(stream)))


def build_slots(block_table: torch.Tensor, cu_tokens: torch.Tensor, start_pos: torch.Tensor,
                num_tokens: int, block_size: int = 16, out: Optional[torch.Tensor] = None,
                stream=None) -> torch.Tensor:
    """Device slot mapping: token t of sequence n (rows cu_tokens[n]..) sits at position
    start_pos[n] + t - cu_tokens[n]; slot = table[n][pos // bs] * bs + pos % bs, or -1 outside
    the table (the reference's write_decode_kv / scatter_prefill_kv host loops)."""
    for name, t in (("block_table", block_table), ("cu_tokens", cu_tokens), ("start_pos", start_pos)):
        _require(t, torch.int32, name)
    if out is None:
        out = torch.empty(num_tokens, dtype=torch.int64, device=block_table.device)
    _require(out, torch.int64, "out")
    check(lib().llkv_build_slots(_ptr(out), _ptr(block_table), block_table.shape[1], _ptr(cu_tokens),
                                 _ptr(start_pos), start_pos.shape[0], num_tokens, block_size,
                                 _stream(stream)))
    return out


def rope_append(q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, slot_mapping: torch.Tensor,
                cos: torch.Tensor, sin: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                stream=None) -> None:
    """Fused RoPE + KV append: q [T, Hq, D] (or None) and k [T, Hkv, D] rotated in place over the
    first 2 * cos.shape[1] dims (Neox halves), then the k and v rows written to pool rows
    slot_mapping[t] (<0 skips).  cos / sin: fp32 [T, rotary_dim / 2]."""
    _require(slot_mapping, torch.int64, "slot_mapping")
    _require(k, k_pool.dtype, "k")
    _require(v, k_pool.dtype, "v")
    if q is not None:
        _require(q, k_pool.dtype, "q")
    _require(cos, torch.float32, "cos")
    _require(sin, torch.float32, "sin")
    t, hkv, d = k.shape
    hq = q.shape[1] if q is not None else 0
    check(lib().llkv_rope_append(_ptr(q), _ptr(k), _ptr(v), _ptr(k_pool), _ptr(v_pool),
                                 _ptr(slot_mapping), _ptr(cos), _ptr(sin), t, hq, hkv, d,
                                 2 * cos.shape[1], dtype_code(k_pool.dtype), _stream(stream)))


def scatter_prefill_kv(k: torch.Tensor, v: torch.Tensor, start_pos: int, n_tokens: int,
                       block_table: torch.Tensor, max_blocks: int, allocator: BlockAllocator,
                       stream=None) -> None:
    """Reference scatter_prefill_kv_gpu (paged_attention.h:95-102)."""
    _require(block_table, torch.int32, "block_table")
    _require(k, allocator.kv_dtype, "k")
    _require(v, allocator.kv_dtype, "v")
    check(lib().llkv_scatter_prefill(_ptr(allocator.k_storage), _ptr(allocator.v_storage), _ptr(k),
                                     _ptr(v), start_pos, n_tokens, _ptr(block_table), max_blocks,
                                     allocator.num_kv_heads, allocator.head_dim, allocator.block_size,
                                     dtype_code(allocator.kv_dtype), _stream(stream)))


def scatter_prefill_kv_batched(k_flat: torch.Tensor, v_flat: torch.Tensor, kv_offsets, num_tokens,
                               start_poss, token_cumsum, flat_bt, max_blocks: int, n: int,
                               p_total: int, allocator: BlockAllocator, stream=None) -> None:
    """Reference scatter_prefill_kv_batched_gpu_dispatch (paged_attention.h:116-124)."""
    for name, t in (("kv_offsets", kv_offsets), ("num_tokens", num_tokens),
                    ("start_poss", start_poss), ("token_cumsum", token_cumsum), ("flat_bt", flat_bt)):
        _require(t, torch.int32, name)
    check(lib().llkv_scatter_prefill_batched(
        _ptr(allocator.k_storage), _ptr(allocator.v_storage), _ptr(k_flat), _ptr(v_flat),
        allocator.num_kv_heads, allocator.head_dim, _ptr(kv_offsets), _ptr(num_tokens),
        _ptr(start_poss), _ptr(token_cumsum), _ptr(flat_bt), max_blocks, n, p_total,
        allocator.block_size, dtype_code(allocator.kv_dtype), _stream(stream)))


def gather_kv(k_pool: torch.Tensor, v_pool: torch.Tensor, block_table: torch.Tensor,
              cu_seqlens: torch.Tensor, total_tokens: int, stream=None):
    """Block-table gather into contiguous [total_tokens, Hkv, D] (reconstruct_kv on device)."""
    _require(block_table, torch.int32, "block_table")
    _require(cu_seqlens, torch.int32, "cu_seqlens")
    nb, bs, hkv, d = k_pool.shape
    kd = torch.empty((total_tokens, hkv, d), dtype=k_pool.dtype, device=k_pool.device)
    vd = torch.empty_like(kd)
    check(lib().llkv_gather(_ptr(kd), _ptr(vd), _ptr(k_pool), _ptr(v_pool), _ptr(block_table),
                            block_table.shape[1], _ptr(cu_seqlens), cu_seqlens.shape[0] - 1,
                            total_tokens, hkv, d, bs, dtype_code(k_pool.dtype), _stream(stream)))
    return kd, vd


def decode_workspace_bytes(num_seqs: int, hq: int, hkv: int, d: int, block_size: int,
                           max_seq_len: int, num_splits: int = 0) -> int:
    return lib().llkv_paged_decode_workspace_size(num_seqs, hq, hkv, d, block_size, max_seq_len,
                                                  num_splits)


# Sizes remembered by shape, for plain integers alone: tensors and arrays, which the C call takes
# as well, may change in place.
@functools.lru_cache(maxsize=256)
def _decode_size(*shape: int) -> int:
    return lib().llkv_paged_decode_workspace_size(*shape)


def _decode_workspace_bytes(num_seqs: int, hq: int, hkv: int, d: int, block_size: int, max_seq_len,
                            num_splits) -> int:
    if type(max_seq_len) is not int or type(num_splits) is not int:
        return decode_workspace_bytes(num_seqs, hq, hkv, d, block_size, max_seq_len, num_splits)
    if max_seq_len > 0 and block_size > 0:   # the size depends on the number of pages
        max_seq_len -= (max_seq_len - 1) % block_size
    return _decode_size(num_seqs, hq, hkv, d, block_size, max_seq_len, num_splits)


DECODE_SCHEDULES = ("one_split", "unit", "splits", "balanced", "generic")


def decode_schedule(num_seqs: int, hq: int, hkv: int, d: int, max_seq_len: int, dtype: torch.dtype,
                    num_splits: int = 0, block_size: int = 16, with_append: bool = False):
    """(schedule name, key splits) that paged_decode / paged_decode_append take for this shape on
    the current device (llkv_paged_decode_schedule): one_split runs one kernel, unit one kernel
    (splits == 1) or 16-wave splits and a merge kernel, splits and balanced a merge kernel after
    the split kernel."""
    kind, splits = ctypes.c_int(), ctypes.c_int()
    check(lib().llkv_paged_decode_schedule(num_seqs, hq, hkv, d, block_size, max_seq_len, num_splits,
                                           dtype_code(dtype), int(with_append), ctypes.byref(kind),
                                           ctypes.byref(splits)))
    return DECODE_SCHEDULES[kind.value], splits.value


_WS: dict = {}


def _workspace(nbytes: int, device) -> torch.Tensor:
    """Workspace for the split partials of decode and prefill, cached per device and grown
    on demand.  Calls that share it must be ordered on one stream."""
    ws = _WS.get(device)
    if ws is None or ws.numel() < nbytes:
        ws = torch.zeros(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
        _WS[device] = ws
    return ws


def paged_decode(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                 block_table: torch.Tensor, seq_lens: torch.Tensor, max_seq_len: int,
                 num_splits: int = 0, scale: Optional[float] = None,
                 out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None,
                 stream=None) -> torch.Tensor:
    """Paged decode attention over pools [nb, bs, Hkv, D]; q [B, Hq, D]."""
    _require(q, k_pool.dtype, "q")
    _require(block_table, torch.int32, "block_table")
    _require(seq_lens, torch.int32, "seq_lens")
    b, hq, d = q.shape
    nb, bs, hkv, _ = k_pool.shape
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    if out is None:
        out = torch.empty_like(q)
    ws = _decode_workspace_bytes(b, hq, hkv, d, bs, max_seq_len, num_splits)
    if ws and (workspace is None or workspace.numel() * workspace.element_size() < ws):
        workspace = _workspace(ws, q.device)
    check(lib().llkv_paged_decode(_ptr(out), _ptr(q), _ptr(k_pool), _ptr(v_pool), _ptr(block_table),
                                  _ptr(seq_lens), b, hq, hkv, d, bs, block_table.shape[1],
                                  max_seq_len, num_splits, scale, dtype_code(q.dtype),
                                  _ptr(workspace) if ws else None, ws, _stream(stream)))
    return out


def paged_decode_append(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor,
                        k_pool: torch.Tensor, v_pool: torch.Tensor, block_table: torch.Tensor,
                        seq_lens: torch.Tensor, max_seq_len: int, num_splits: int = 0,
                        scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                        workspace: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """Fused KV append + paged decode: the new rows k_new / v_new [B, Hkv, D] go to position
    seq_lens[b] - 1 of each sequence (seq_lens count the new token), then decode attention over
    [0, seq_lens[b]); equal to append_kv followed by paged_decode."""
    _require(q, k_pool.dtype, "q")
    _require(k_new, k_pool.dtype, "k_new")
    _require(v_new, k_pool.dtype, "v_new")
    _require(block_table, torch.int32, "block_table")
    _require(seq_lens, torch.int32, "seq_lens")
    b, hq, d = q.shape
    nb, bs, hkv, _ = k_pool.shape
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    if out is None:
        out = torch.empty_like(q)
    ws = _decode_workspace_bytes(b, hq, hkv, d, bs, max_seq_len, num_splits)
    if ws and (workspace is None or workspace.numel() * workspace.element_size() < ws):
        workspace = _workspace(ws, q.device)
    check(lib().llkv_paged_decode_append(_ptr(out), _ptr(q), _ptr(k_new), _ptr(v_new), _ptr(k_pool),
                                         _ptr(v_pool), _ptr(block_table), _ptr(seq_lens), b, hq, hkv,
                                         d, bs, block_table.shape[1], max_seq_len, num_splits, scale,
                                         dtype_code(q.dtype), _ptr(workspace) if ws else None, ws,
                                         _stream(stream)))
    return out


def paged_attention(q: torch.Tensor, block_table: torch.Tensor, max_blocks_per_seq: int,
                    seq_lens: torch.Tensor, allocator: BlockAllocator,
                    max_seq_len: Optional[int] = None) -> torch.Tensor:
    """Reference paged_attention (paged_attention.h:31-36).  Like the reference, reads
    seq_lens back to size the launch unless max_seq_len is given."""
    if max_seq_len is None:
        max_seq_len = int(seq_lens.max().item()) if seq_lens.numel() else 0
    bt = block_table.view(-1, max_blocks_per_seq)
    return paged_decode(q, allocator.k_storage, allocator.v_storage, bt, seq_lens, max_seq_len)


@functools.lru_cache(maxsize=256)
def _prefill_size(*shape: int) -> int:
    return lib().llkv_paged_prefill_workspace_size(*shape)


def _prefill_workspace_bytes(num_seqs: int, total_q: int, max_q_len, max_seq_len, hq: int, d: int, block_size: int,
                             dtype: int) -> int:
    plain = type(max_q_len) is int and type(max_seq_len) is int
    size = _prefill_size if plain else lib().llkv_paged_prefill_workspace_size
    return size(num_seqs, total_q, max_q_len, max_seq_len, hq, d, block_size, dtype)


def paged_prefill(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                  block_table: torch.Tensor, cu_q: torch.Tensor, seq_lens: torch.Tensor,
                  max_q_len: int, max_seq_len: int, causal: bool = True,
                  scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                  stream=None, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Varlen paged prefill: q [total_q, Hq, D], sequence n owns rows cu_q[n]:cu_q[n+1].
    workspace: uint8 device buffer for the key-chunk partials (default: a cached one);
    pass an empty tensor to run every key range unsplit."""
    _require(q, k_pool.dtype, "q")
    for name, t in (("block_table", block_table), ("cu_q", cu_q), ("seq_lens", seq_lens)):
        _require(t, torch.int32, name)
    tq, hq, d = q.shape
    nb, bs, hkv, _ = k_pool.shape
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    if out is None:
        out = torch.empty_like(q)
    n = seq_lens.shape[0]
    ws_bytes = _prefill_workspace_bytes(n, tq, max_q_len, max_seq_len, hq, d, bs, dtype_code(q.dtype))
    if workspace is None and ws_bytes:
        workspace = _workspace(ws_bytes, q.device)
    ws_ptr = _ptr(workspace) if workspace is not None else None
    ws_len = workspace.numel() if workspace is not None else 0
    check(lib().llkv_paged_prefill(_ptr(out), _ptr(q), _ptr(k_pool), _ptr(v_pool), _ptr(block_table),
                                   block_table.shape[1], _ptr(cu_q), _ptr(seq_lens),
                                   n, tq, max_q_len, max_seq_len, hq, hkv, d, bs,
                                   1 if causal else 0, scale, dtype_code(q.dtype), ws_ptr, ws_len,
                                   _stream(stream)))
    return out


def prefill_paged_attention(q: torch.Tensor, block_table: torch.Tensor, max_blocks: int,
                            seq_len: torch.Tensor, allocator: BlockAllocator,
                            causal: bool = False) -> torch.Tensor:
    """Reference prefill_paged_attention (paged_attention.h:71-77): one sequence, seq_len is a
    device int32 [1] holding history + P."""
    p = q.shape[0]
    total = int(seq_len.reshape(-1)[0].item())
    cu = torch.tensor([0, p], dtype=torch.int32, device=q.device)
    bt = block_table.reshape(1, -1)[:, :max_blocks].contiguous()
    return paged_prefill(q, allocator.k_storage, allocator.v_storage, bt, cu,
                         seq_len.reshape(-1)[:1].contiguous(), p, total, causal)


def first_prefill_attn_batched(out: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                               hq: int, hkv: int, d: int, offsets, kv_offsets, num_tokens,
                               token_cumsum, start_poss, n: int, p_total: int, scale: float,
                               stream=None, max_tokens: int = 0) -> None:
    """Reference first_prefill_attn_batched_gpu_dispatch (paged_attention.h:138-145).
    offsets / kv_offsets are element offsets of row starts; max_tokens is a host upper bound
    of num_tokens (0: p_total)."""
    for name, t in (("offsets", offsets), ("kv_offsets", kv_offsets), ("num_tokens", num_tokens),
                    ("token_cumsum", token_cumsum), ("start_poss", start_poss)):
        _require(t, torch.int32, name)
    check(lib().llkv_first_prefill_batched(_ptr(out), _ptr(q), _ptr(k), _ptr(v), hq, hkv, d,
                                           _ptr(offsets), _ptr(kv_offsets), _ptr(num_tokens),
                                           _ptr(token_cumsum), _ptr(start_poss), n, p_total, max_tokens,
                                           scale, dtype_code(q.dtype), _stream(stream)))


# ---------------------------------------------------------------------------
# The cache step's further operators: norm + rotation + append, drafted trees, accumulated weights
# and eviction.  Their arguments are checked in full (device, type, shape), before anything is
# launched.  Workspaces and outputs come from torch's allocator on the stream of the call, so that
# calls on different streams share none, and a captured call owns its own.
# ---------------------------------------------------------------------------

# One expression for what a call almost always finds; the reasons are looked for afterwards (a
# one-token qk_norm_rope_append checks ten tensors: 18.1 us a call with a test per property).
def _device_of(t: torch.Tensor, what: str = "the pools") -> int:
    """The device of a call: the pools', which has to be the current one."""
    device = t.get_device()
    if device < 0:
        raise ValueError(f"{what} must be on a GPU")
    if device != torch._C._cuda_getDevice():
        raise ValueError(f"{what} must be on the current device, not on cuda:{device}")
    return device


def _check(t: torch.Tensor, dtype: torch.dtype, shape: tuple, device: int, name: str):
    """`t` is contiguous, of this type and shape, on this device."""
    if t.dtype is dtype and t.shape == shape and t.get_device() == device and t.is_contiguous():
        return
    _require(t, dtype, name)
    if t.shape != shape:
        raise ValueError(f"{name}: expected shape {shape}, got {tuple(t.shape)}")
    raise ValueError(f"{name}: must be on cuda:{device}")


def _check_table(t: torch.Tensor, n: int, device: int, name: str) -> int:
    """An int32 table of n rows; returns their width."""
    width = t.shape[-1] if t.dim() == 2 else None
    _check(t, torch.int32, (n, width), device, name)
    return width


def _check_pools(k_pool: torch.Tensor, v_pool: Optional[torch.Tensor]):
    """(device, type, block size, kv heads, head_dim) of the pools."""
    device = _device_of(k_pool)
    dtype, shape = k_pool.dtype, k_pool.shape
    if len(shape) != 4 or not k_pool.is_contiguous():
        raise ValueError("k_pool: expected contiguous [pages, block size, kv heads, head_dim]")
    if v_pool is not None:
        _check(v_pool, dtype, shape, device, "v_pool")
    return device, dtype, shape[1], shape[2], shape[3]


def _check_rows(t: torch.Tensor, dtype: torch.dtype, shape: tuple, device: int, name: str) -> int:
    """Rows [T, heads, D] whose heads are contiguous; returns the elements between tokens."""
    strides = t.stride()
    if (t.dtype is dtype and t.shape == shape and t.get_device() == device and strides[2] == 1
            and strides[1] == shape[2]):
        return strides[0]
    if t.dtype != dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name}: expected shape {shape}, got {tuple(t.shape)}")
    if t.get_device() != device:
        raise ValueError(f"{name}: must be on cuda:{device}")
    if t.numel() and (strides[2] != 1 and shape[2] > 1 or strides[1] != shape[2] and shape[1] > 1):
        raise ValueError(f"{name}: the heads of a token must be contiguous")
    return strides[0]


def _check_mass(mass: torch.Tensor, n: int, hkv: int, least: int, device: int):
    """Totals [N, Hkv, at least `least` keys] with contiguous rows of keys; returns their strides."""
    if mass.dtype != torch.float32:
        raise TypeError(f"mass: expected torch.float32, got {mass.dtype}")
    if mass.dim() != 3 or mass.shape[0] != n or mass.shape[1] != hkv:
        raise ValueError(f"mass: expected shape ({n}, {hkv}, keys), got {tuple(mass.shape)}")
    if mass.get_device() != device:
        raise ValueError(f"mass: must be on cuda:{device}")
    width = mass.shape[2]
    if width < least:
        raise ValueError(f"mass: rows of {width} keys for up to {least}")
    bs, hs, ks = mass.stride()
    if hkv == 1:
        hs = width
    if n == 1:
        bs = hkv * hs
    if ks != 1 and width > 1 or hs < width or bs < hkv * hs:
        raise ValueError("mass: rows of keys must be contiguous and must not overlap")
    return bs, hs


def _empty(shape: tuple, dtype: torch.dtype, device: int, stream) -> torch.Tensor:
    """A tensor of the call's stream (memory that another stream still uses is not handed out)."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device="cuda")      # the current device (_device_of)
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device="cuda")


def _scratch(nbytes: int, given: Optional[torch.Tensor], device: int, stream):
    """(address, bytes) of a workspace: the caller's, or one from torch's allocator, returned as the
    third value to be held until the call is enqueued."""
    if given is not None:
        if given.get_device() != device:
            raise ValueError(f"workspace: must be on cuda:{device}")
        if not given.is_contiguous():
            raise ValueError("workspace: must be contiguous")
        return given.data_ptr(), given.numel() * given.element_size(), given
    if nbytes == 0:
        return None, 0, None
    ws = _empty((nbytes,), torch.uint8, device, stream)
    return ws.data_ptr(), nbytes, ws


def _scale(scale: Optional[float], d: int) -> float:
    return 1.0 / math.sqrt(d) if scale is None else scale


def qk_norm_rope_append(q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, slot_mapping: torch.Tensor,
                        positions: torch.Tensor, inv_freq: torch.Tensor, k_pool: torch.Tensor,
                        v_pool: torch.Tensor, q_weight: Optional[torch.Tensor] = None,
                        k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                        pair_axis: Optional[Union[bytes, Sequence[int]]] = None,
                        q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None,
                        stream=None) -> Optional[torch.Tensor]:
    """RMS norm of every query and key head (fp32 weights [D], or None), rotation of the first
    2 * len(inv_freq) dims (Neox halves) and KV append, in one pass; returns q_out.

    q [T, Hq, D] (or None), k and v [T, Hkv, D]: heads contiguous, any distance between tokens (slices
    of a fused projection).  positions: int32 [T] or [axes, T], up to four axes; pair_axis: the axis of
    each rotated pair, len(inv_freq) small integers (host; not needed with one axis).  inv_freq: fp32.
    q_out: a new tensor by default; q itself rotates in place.  k_out: None writes the k rows to the
    pool only.  The k and v rows go to pool rows slot_mapping[t] (<0 skips)."""
    device, dt, _, hkv, d = _check_pools(k_pool, v_pool)
    t = k.shape[0]
    ks = _check_rows(k, dt, (t, hkv, d), device, "k")
    vs = _check_rows(v, dt, (t, hkv, d), device, "v")
    _check(slot_mapping, torch.int64, (t,), device, "slot_mapping")
    axes, half = positions.shape[0] if positions.dim() == 2 else 1, inv_freq.shape[0]
    _check(positions, torch.int32, (axes, t) if positions.dim() == 2 else (t,), device, "positions")
    _check(inv_freq, torch.float32, (half,), device, "inv_freq")
    if q_weight is not None:
        _check(q_weight, torch.float32, (d,), device, "q_weight")
    if k_weight is not None:
        _check(k_weight, torch.float32, (d,), device, "k_weight")
    if pair_axis is not None:
        if not isinstance(pair_axis, bytes):
            pair_axis = bytes(pair_axis)
        if len(pair_axis) != half:
            raise ValueError(f"pair_axis: {len(pair_axis)} axes for {half} pairs")
        if half and max(pair_axis) >= axes:
            raise ValueError(f"pair_axis: axis {max(pair_axis)} of {axes}")
    hq = qs = qos = kos = 0
    if q is not None:
        hq = q.shape[1] if q.dim() == 3 else 0
        qs = _check_rows(q, dt, (t, hq, d), device, "q")
        if q_out is None:
            q_out, qos = _empty((t, hq, d), dt, device, stream), hq * d
        else:
            qos = _check_rows(q_out, dt, (t, hq, d), device, "q_out")
    elif q_out is not None:
        raise ValueError("q_out: there is no q")
    if k_out is not None:
        kos = _check_rows(k_out, dt, (t, hkv, d), device, "k_out")
    check(lib().llkv_qk_norm_rope_append(
        _ptr(q_out), _ptr(k_out), _ptr(q), _ptr(k), _ptr(v), qos, kos, qs, ks, vs, _ptr(k_pool), _ptr(v_pool),
        _ptr(slot_mapping), _ptr(positions), axes, pair_axis, _ptr(inv_freq), _ptr(q_weight), _ptr(k_weight), eps,
        t, hq, hkv, d, 2 * half, dtype_code(dt), _stream(stream)))
    return q_out


def build_tree(parents: torch.Tensor, cu_q: torch.Tensor, seq_lens: torch.Tensor, max_q_len: int,
               tree_mask: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None, stream=None):
    """(tree_mask int32 [total_q, words], positions int32 [total_q]) of drafted trees: parents int32
    [total_q] within each sequence's rows cu_q[n]:cu_q[n+1], anything outside [0, i) a root; the mask has
    node i itself and its ancestors, the position is the context's length plus the depth."""
    device = _device_of(parents, "parents")
    n, total = seq_lens.shape[0], parents.shape[0]
    _check(parents, torch.int32, (total,), device, "parents")
    _check(seq_lens, torch.int32, (n,), device, "seq_lens")
    _check(cu_q, torch.int32, (n + 1,), device, "cu_q")
    if tree_mask is None:
        tree_mask = _empty((total, (max_q_len + 31) // 32), torch.int32, device, stream)
    if positions is None:
        positions = _empty((total,), torch.int32, device, stream)
    words = _check_table(tree_mask, total, device, "tree_mask")
    _check(positions, torch.int32, (total,), device, "positions")
    check(lib().llkv_build_tree(_ptr(tree_mask), words, _ptr(positions), _ptr(parents), _ptr(cu_q),
                                _ptr(seq_lens), n, total, max_q_len, _stream(stream)))
    return tree_mask, positions


# By the device, too: a launch is as large as the device's compute units hold.
@functools.lru_cache(maxsize=256)
def _tree_size(device: int, *shape: int) -> int:
    return lib().llkv_paged_tree_attention_workspace_size(*shape)


@functools.lru_cache(maxsize=256)
def _mass_size(device: int, *shape: int) -> int:
    return lib().llkv_paged_decode_mass_workspace_size(*shape)


def paged_tree_attention(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, block_table: torch.Tensor,
                         cu_q: torch.Tensor, seq_lens: torch.Tensor, tree_mask: torch.Tensor, max_q_len: int,
                         max_seq_len: int, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                         workspace: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """Attention of drafted trees: q [total_q, Hq, D], sequence n owning rows cu_q[n]:cu_q[n+1], whose K
    and V are its last cached positions.  A row sees the whole context and the nodes j of its sequence
    whose bit is set in its row of tree_mask (int32 [total_q, words]; build_tree)."""
    device, dtype, bs, hkv, d = _check_pools(k_pool, v_pool)
    tq, hq = q.shape[0], q.shape[1]
    n = seq_lens.shape[0]
    _check(q, dtype, (tq, hq, d), device, "q")
    _check(seq_lens, torch.int32, (n,), device, "seq_lens")
    blocks = _check_table(block_table, n, device, "block_table")
    _check(cu_q, torch.int32, (n + 1,), device, "cu_q")
    words = _check_table(tree_mask, tq, device, "tree_mask")
    if out is None:
        out = _empty((tq, hq, d), dtype, device, stream)
    else:
        _check(out, dtype, (tq, hq, d), device, "out")
    max_q_len, max_seq_len, dt = int(max_q_len), int(max_seq_len), dtype_code(dtype)
    need = _tree_size(device, n, max_q_len, hq, hkv, d, bs, max_seq_len, dt)
    ws, nbytes, held = _scratch(need, workspace, device, stream)
    check(lib().llkv_paged_tree_attention(_ptr(out), _ptr(q), _ptr(k_pool), _ptr(v_pool), _ptr(block_table),
                                          blocks, _ptr(cu_q), _ptr(seq_lens), _ptr(tree_mask), words, n, tq, max_q_len,
                                          max_seq_len, hq, hkv, d, bs, _scale(scale, d), dt, ws, nbytes, _stream(stream)))
    return out


def paged_decode_mass(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, block_table: torch.Tensor,
                      seq_lens: torch.Tensor, max_seq_len: int, mass: torch.Tensor, scale: Optional[float] = None,
                      out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None,
                      stream=None) -> torch.Tensor:
    """paged_decode that also adds each key's weight, summed over the query heads of its kv head, to
    mass: fp32 [B, Hkv, keys >= max_seq_len]."""
    device, dtype, bs, hkv, d = _check_pools(k_pool, v_pool)
    b, hq = q.shape[0], q.shape[1]
    _check(q, dtype, (b, hq, d), device, "q")
    _check(seq_lens, torch.int32, (b,), device, "seq_lens")
    blocks = _check_table(block_table, b, device, "block_table")
    max_seq_len, dt = int(max_seq_len), dtype_code(dtype)
    mass_bs, mass_hs = _check_mass(mass, b, hkv, max_seq_len, device)
    if out is None:
        out = _empty((b, hq, d), dtype, device, stream)
    else:
        _check(out, dtype, (b, hq, d), device, "out")
    ws, nbytes, held = _scratch(_mass_size(device, b, hq, hkv, d, bs, max_seq_len, dt), workspace, device, stream)
    check(lib().llkv_paged_decode_mass(_ptr(out), _ptr(mass), mass_bs, mass_hs, _ptr(q), _ptr(k_pool), _ptr(v_pool),
                                       _ptr(block_table), _ptr(seq_lens), b, hq, hkv, d, bs, blocks, max_seq_len,
                                       _scale(scale, d), dt, ws, nbytes, _stream(stream)))
    return out


def paged_window_mass(q: torch.Tensor, k_pool: torch.Tensor, block_table: torch.Tensor, cu_q: torch.Tensor,
                      seq_lens: torch.Tensor, max_q_len: int, max_seq_len: int, mass: torch.Tensor,
                      scale: Optional[float] = None, workspace: Optional[torch.Tensor] = None, stream=None) -> None:
    """Adds the weights that the last rows of each sequence (q [total_q, Hq, D], rows
    cu_q[n]:cu_q[n+1] its last tokens, causal) give to each of its keys to mass, fp32 [N, Hkv,
    keys >= max_seq_len]."""
    device, dtype, bs, hkv, d = _check_pools(k_pool, None)
    tq, hq = q.shape[0], q.shape[1]
    n = seq_lens.shape[0]
    _check(q, dtype, (tq, hq, d), device, "q")
    _check(seq_lens, torch.int32, (n,), device, "seq_lens")
    blocks = _check_table(block_table, n, device, "block_table")
    _check(cu_q, torch.int32, (n + 1,), device, "cu_q")
    max_q_len, max_seq_len, dt = int(max_q_len), int(max_seq_len), dtype_code(dtype)
    mass_bs, mass_hs = _check_mass(mass, n, hkv, max_seq_len, device)
    need = lib().llkv_paged_window_mass_workspace_size(tq, hq, max_seq_len, dt)
    ws, nbytes, held = _scratch(need, workspace, device, stream)
    check(lib().llkv_paged_window_mass(_ptr(mass), mass_bs, mass_hs, _ptr(q), _ptr(k_pool), _ptr(block_table),
                                       blocks, _ptr(cu_q), _ptr(seq_lens), n, tq, max_q_len, max_seq_len, hq, hkv, d, bs,
                                       _scale(scale, d), dt, ws, nbytes, _stream(stream)))


def evict_select(mass: torch.Tensor, seq_lens: torch.Tensor, budget: int, max_seq_len: int, sinks: int = 0,
                 recent: int = 0, workspace: Optional[torch.Tensor] = None, stream=None):
    """(keep int32 [N, Hkv, budget], counts int32 [N], totals like mass): for every kv head the positions to
    keep, rising, -1 behind the last: the first `sinks`, the last `recent`, and the largest totals of the rest
    (ties: the lower position); the kept totals in the same order, zeros behind them."""
    device, max_seq_len = _device_of(mass, "mass"), int(max_seq_len)
    n, hkv, width = mass.shape
    mass_bs, mass_hs = _check_mass(mass, n, hkv, max_seq_len, device)
    _check(seq_lens, torch.int32, (n,), device, "seq_lens")
    if budget <= 0 or sinks < 0 or recent < 0 or sinks + recent > budget:
        raise ValueError(f"a budget of {budget} for {sinks} sinks and {recent} recent keys")
    keep = _empty((n, hkv, budget), torch.int32, device, stream)
    counts = _empty((n,), torch.int32, device, stream)
    out = _empty((n, hkv, width), torch.float32, device, stream)
    need = lib().llkv_evict_select_workspace_size(n, hkv, max_seq_len)
    ws, nbytes, held = _scratch(need, workspace, device, stream)
    check(lib().llkv_evict_select(_ptr(keep), _ptr(counts), _ptr(out), hkv * width, width, width, _ptr(mass), mass_bs,
                                  mass_hs, _ptr(seq_lens), n, hkv, max_seq_len, budget, sinks, recent, ws, nbytes,
                                  _stream(stream)))
    return keep, counts, out


def compact_kv(k_pool: torch.Tensor, v_pool: torch.Tensor, block_table: torch.Tensor, keep: torch.Tensor,
               counts: torch.Tensor, dst_table: Optional[torch.Tensor] = None,
               dst_start: Optional[torch.Tensor] = None, stream=None) -> None:
    """Moves the K and V rows at positions keep[n, h, i], i < counts[n] (keep int32 [N, Hkv or 1, M]; 1: all
    heads alike) to positions dst_start[n] + i (0 + i): of dst_table's pages, which hold none of the rows
    read, or in place (dst_table None; keep rising, keep[i] >= dst_start + i, and pages that no other
    sequence shares)."""
    device, dtype, bs, hkv, d = _check_pools(k_pool, v_pool)
    n = block_table.shape[0]
    blocks, dst_blocks = _check_table(block_table, n, device, "block_table"), 0
    _check(counts, torch.int32, (n,), device, "counts")
    heads, most = keep.shape[1:] if keep.dim() == 3 else (0, 0)
    if heads != hkv and heads != 1:
        raise ValueError(f"keep: expected shape ({n}, {hkv} or 1, positions), got {tuple(keep.shape)}")
    _check(keep, torch.int32, (n, heads, most), device, "keep")
    if dst_table is not None:
        dst_blocks = _check_table(dst_table, n, device, "dst_table")
    if dst_start is not None:
        _check(dst_start, torch.int32, (n,), device, "dst_start")
    check(lib().llkv_compact(_ptr(k_pool), _ptr(v_pool), _ptr(block_table), blocks, _ptr(dst_table), dst_blocks,
                             _ptr(keep), heads, most, _ptr(counts), _ptr(dst_start), n, hkv, d, bs,
                             dtype_code(dtype), _stream(stream)))


def evict_kv(k_pool: torch.Tensor, v_pool: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
             mass: torch.Tensor, budget: int, max_seq_len: int, sinks: int = 0, recent: int = 0,
             dst_table: Optional[torch.Tensor] = None, stream=None):
    """Cuts every sequence down to at most `budget` keys per kv head by their totals (evict_select) and moves
    their rows (compact_kv) to positions 0 .. of dst_table's pages, or of its own with dst_table None.
    Returns (keep, counts, totals): counts are the new lengths.  The rows keep the rotation of their old
    positions, and new tokens go on with theirs; the caller frees what the tables no longer need."""
    device, _, bs, hkv, _ = _check_pools(k_pool, v_pool)
    n = seq_lens.shape[0]
    if mass.shape[:2] != (n, hkv):
        raise ValueError(f"mass: expected shape ({n}, {hkv}, keys), got {tuple(mass.shape)}")
    _check_table(block_table, n, device, "block_table")     # before the totals are read
    if dst_table is not None:
        blocks = _check_table(dst_table, n, device, "dst_table")
        if blocks * bs < min(budget, int(max_seq_len)):
            raise ValueError(f"dst_table: {blocks} pages for {budget} keys")
    keep, counts, totals = evict_select(mass, seq_lens, budget, max_seq_len, sinks, recent, stream=stream)
    compact_kv(k_pool, v_pool, block_table, keep, counts, dst_table, stream=stream)
    return keep, counts, totals

"""PyTorch-facing wrappers of the liblitekern C ABI.

Every function validates dtype / device / layout, then calls one C entry
point on the current CUDA stream of the tensors' device. Nothing here
computes on the host: a CPU tensor or a missing library raises.
"""

from __future__ import annotations

import contextlib
import ctypes
import math
from typing import NamedTuple, Optional, Union

import torch

from ._lib import (LK_DTYPE_BF16, LK_DTYPE_F16, LK_DTYPE_F32, LK_KV_16BIT, LK_KV_E4M3, LK_KV_INT8,
                   check, lib)

_DTYPES = {torch.float32: LK_DTYPE_F32, torch.float16: LK_DTYPE_F16, torch.bfloat16: LK_DTYPE_BF16}


def _dtype_code(t: torch.Tensor, allowed=(torch.float16, torch.bfloat16)) -> int:
    if t.dtype not in allowed:
        raise TypeError(f"dtype {t.dtype} not supported here (allowed: {allowed})")
    return _DTYPES[t.dtype]


def _cuda(*ts: Optional[torch.Tensor]) -> torch.device:
    dev, index = None, -1
    for t in ts:
        if t is None:
            continue
        i = t.get_device()
        if i < 0:
            raise RuntimeError("litevllm_b200 kernels run on CUDA tensors only (no CPU fallback)")
        if dev is None:
            dev, index = t.device, i
        elif i != index:
            raise RuntimeError(f"tensors on different devices: {dev} vs {t.device}")
    assert dev is not None
    return dev


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _stream(dev: torch.device) -> int:
    # the handle alone: building a torch.cuda.Stream object costs 2.5 us a call
    return torch._C._cuda_getCurrentRawStream(
        torch.cuda.current_device() if dev.index is None else dev.index)


_NULL = contextlib.nullcontext()


def _on(dev: torch.device):
    """Make dev current for the call (a no-op when it already is)."""
    return _NULL if dev.index == torch.cuda.current_device() else torch.cuda.device(dev)


class _Workspaces:
    """Zero-initialised scratch buffers, one per (device, purpose, stream).

    The kernels leave their counter regions zero after every call, so a
    buffer is reused across calls on one stream without re-clearing; calls on
    different streams may run at the same time, so each stream has its own.
    """

    def __init__(self) -> None:
        self._bufs: dict[tuple, torch.Tensor] = {}

    def get(self, dev: torch.device, name: str, nbytes: int) -> torch.Tensor:
        key = (dev.index, name)
        buf = self._bufs.get(key)
        if buf is None or buf.numel() < nbytes:
            size = max(nbytes, 1 << 16)
            if buf is not None:
                size = max(size, buf.numel() * 2)
            buf = torch.zeros(size, dtype=torch.uint8, device=dev)
            self._bufs[key] = buf
        return buf


WORKSPACES = _Workspaces()


# --------------------------------------------------------------- KV store ---
def store_kvcache(
    key: torch.Tensor,
    value: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    slot_mapping: torch.Tensor,
    status: Optional[torch.Tensor] = None,
) -> None:
    """key_cache[slot // bs, slot % bs] = key[t] (and value), for every t.

    key/value: [T, H_kv, D]; caches [num_blocks, bs, H_kv, D] contiguous;
    slot_mapping int64 [T]. Mirrors litevllm/layers/attention.py:79-84.
    """
    dev = _cuda(key, value, key_cache, value_cache, slot_mapping, status)
    if key.dim() != 3 or value.shape != key.shape:
        raise ValueError("key/value must be [T, H_kv, D] with equal shapes")
    T, H_kv, D = key.shape
    if key_cache.dim() != 4 or key_cache.shape[2:] != (H_kv, D) or value_cache.shape != key_cache.shape:
        raise ValueError("caches must be [num_blocks, block_size, H_kv, D]")
    if not (key_cache.is_contiguous() and value_cache.is_contiguous()):
        raise ValueError("caches must be contiguous")
    for t in (key, value):
        if t.stride(2) != 1 or t.stride(1) != D:
            raise ValueError("key/value must have unit d-stride and head stride D")
    if key.dtype != key_cache.dtype or value.dtype != key_cache.dtype:
        raise TypeError("key/value dtype must match the cache dtype")
    if slot_mapping.dtype != torch.int64 or slot_mapping.numel() != T:
        raise TypeError("slot_mapping must be int64 [T]")
    slot_mapping = slot_mapping.contiguous()
    code = _dtype_code(key_cache, (torch.float32, torch.float16, torch.bfloat16))
    num_slots = key_cache.shape[0] * key_cache.shape[1]
    with _on(dev):
        check(
            lib().lk_store_kv(
                key.data_ptr(), value.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(),
                slot_mapping.data_ptr(), T, H_kv, D, key.stride(0), value.stride(0), num_slots,
                code, _ptr(status), _stream(dev),
            )
        )


# ------------------------------------------------------------ 8-bit cache ---
_KV_FORMATS = {torch.int8: LK_KV_INT8, torch.float8_e4m3fn: LK_KV_E4M3}


class QuantizedCache(NamedTuple):
    """The key or the value cache of one layer in 8 bits: data int8 or
    float8_e4m3fn [num_blocks, block_size, H_kv, D] and scale fp32 [num_blocks,
    H_kv, block_size], one scale per (token, KV head) row; a row's values are
    data * scale. Block copies and swaps take (data, data) and (scale, scale)
    pairs of the K and V caches like any other block-major tensors."""

    data: torch.Tensor
    scale: torch.Tensor


def new_quantized_cache(num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int,
                        dtype: torch.dtype = torch.int8, device="cuda") -> QuantizedCache:
    """A zeroed 8-bit key or value cache (dtype torch.int8 or torch.float8_e4m3fn)."""
    if dtype not in _KV_FORMATS:
        raise TypeError("8-bit caches are torch.int8 or torch.float8_e4m3fn")
    return QuantizedCache(
        torch.zeros((num_blocks, block_size, num_kv_heads, head_dim), dtype=dtype, device=device),
        torch.zeros((num_blocks, num_kv_heads, block_size), dtype=torch.float32, device=device))


def _check_q8(key_cache: QuantizedCache, value_cache: QuantizedCache) -> int:
    """Checks a pair of 8-bit caches; the LK_KV_* code."""
    if not isinstance(key_cache, QuantizedCache) or not isinstance(value_cache, QuantizedCache):
        raise TypeError("key_cache and value_cache must both be QuantizedCache")
    kd, ks = key_cache
    vd, vs = value_cache
    if kd.dtype not in _KV_FORMATS or vd.dtype != kd.dtype:
        raise TypeError("8-bit caches are both torch.int8 or both torch.float8_e4m3fn")
    if ks.dtype != torch.float32 or vs.dtype != torch.float32:
        raise TypeError("scales must be fp32")
    if kd.dim() != 4 or vd.shape != kd.shape:
        raise ValueError("cache data must be [num_blocks, block_size, H_kv, D] of equal shapes")
    nb, bs, H_kv, _ = kd.shape
    if ks.shape != (nb, H_kv, bs) or vs.shape != ks.shape:
        raise ValueError("scales must be [num_blocks, H_kv, block_size]")
    if not (kd.is_contiguous() and vd.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
        raise ValueError("caches and scales must be contiguous")
    return _KV_FORMATS[kd.dtype]


def _check_status(status: Optional[torch.Tensor]) -> None:
    if status is not None and (status.dtype != torch.int32 or status.numel() < 1):
        raise TypeError("status must be an int32 tensor")


def store_kvcache_q8(
    key: torch.Tensor,
    value: torch.Tensor,
    key_cache: QuantizedCache,
    value_cache: QuantizedCache,
    slot_mapping: torch.Tensor,
    status: Optional[torch.Tensor] = None,
) -> None:
    """store_kvcache into 8-bit caches: each (token, KV head) row is quantised
    as it is written (lk_store_kv_q8 has the formula).

    key/value: fp16 / bf16 [T, H_kv, D], D 64 or 128; slot_mapping int64 [T],
    -1 skips a token.
    """
    fmt = _check_q8(key_cache, value_cache)
    dev = _cuda(key, value, *key_cache, *value_cache, slot_mapping, status)
    if key.dim() != 3 or value.shape != key.shape:
        raise ValueError("key/value must be [T, H_kv, D] with equal shapes")
    T, H_kv, D = key.shape
    nb, bs, Hc, Dc = key_cache.data.shape
    if (Hc, Dc) != (H_kv, D):
        raise ValueError("caches must be [num_blocks, block_size, H_kv, D]")
    for t in (key, value):
        if t.stride(2) != 1 or t.stride(1) != D:
            raise ValueError("key/value must have unit d-stride and head stride D")
    code = _dtype_code(key)
    if value.dtype != key.dtype:
        raise TypeError("key and value must share a dtype")
    if slot_mapping.dtype != torch.int64 or slot_mapping.numel() != T:
        raise TypeError("slot_mapping must be int64 [T]")
    _check_status(status)
    slot_mapping = slot_mapping.contiguous()
    with _on(dev):
        check(
            lib().lk_store_kv_q8(
                key.data_ptr(), value.data_ptr(), key_cache.data.data_ptr(),
                key_cache.scale.data_ptr(), value_cache.data.data_ptr(),
                value_cache.scale.data_ptr(), slot_mapping.data_ptr(), T, H_kv, D, key.stride(0),
                value.stride(0), nb, bs, code, fmt, _ptr(status), _stream(dev),
            )
        )


def load_kvcache_q8(
    key_cache: QuantizedCache,
    value_cache: QuantizedCache,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    cu_rows: torch.Tensor,
    num_rows: int,
    dtype: torch.dtype = torch.bfloat16,
    key_out: Optional[torch.Tensor] = None,
    value_out: Optional[torch.Tensor] = None,
    status: Optional[torch.Tensor] = None,
) -> tuple:
    """Read 8-bit caches back: (keys, values) [num_rows, H_kv, D] of `dtype`
    (fp32, fp16 or bf16). Row cu_rows[b] + p is position p of sequence b;
    a sequence's rows past its context are zero, rows that belong to no sequence
    are left as they were. cu_rows int32 [B + 1]."""
    fmt = _check_q8(key_cache, value_cache)
    dev = _cuda(*key_cache, *value_cache, block_tables, context_lens, cu_rows, key_out, value_out,
                status)
    nb, bs, H_kv, D = key_cache.data.shape
    if block_tables.dtype != torch.int32 or block_tables.dim() != 2:
        raise TypeError("block_tables must be int32 [B, max_blocks]")
    B, max_blocks = block_tables.shape
    if max_blocks > 0 and block_tables.stride(1) != 1:
        block_tables = block_tables.contiguous()
    if context_lens.dtype != torch.int32 or context_lens.numel() != B:
        raise TypeError("context_lens must be int32 [B]")
    if cu_rows.dtype != torch.int32 or cu_rows.numel() != B + 1:
        raise TypeError("cu_rows must be int32 [B + 1]")
    _check_status(status)
    context_lens, cu_rows = context_lens.contiguous(), cu_rows.contiguous()
    num_rows = int(num_rows)
    if num_rows < 0:
        raise ValueError("num_rows must not be negative")
    outs = []
    for out in (key_out, value_out):
        if out is None:
            out = torch.empty((num_rows, H_kv, D), dtype=dtype, device=dev)
        elif out.shape != (num_rows, H_kv, D) or out.dtype != dtype or not out.is_contiguous():
            raise ValueError("key_out/value_out must be contiguous [num_rows, H_kv, D] of dtype")
        outs.append(out)
    code = _dtype_code(outs[0], (torch.float32, torch.float16, torch.bfloat16))
    with _on(dev):
        check(
            lib().lk_load_kv_q8(
                outs[0].data_ptr(), outs[1].data_ptr(), key_cache.data.data_ptr(),
                key_cache.scale.data_ptr(), value_cache.data.data_ptr(),
                value_cache.scale.data_ptr(), block_tables.data_ptr(), block_tables.stride(0),
                context_lens.data_ptr(), cu_rows.data_ptr(), B, num_rows, H_kv, D, nb, bs,
                max_blocks, code, fmt, _ptr(status), _stream(dev),
            )
        )
    return tuple(outs)


def _tree_workspace(dev, workspace, T, B, max_q, H, H_kv, D, bs, max_blocks, fmt):
    """(pointer, bytes, tensor to keep alive). Without a caller's workspace the
    partials of split contexts live in a buffer of this call's own, from torch's
    allocator: calls on other streams and captured graphs never share it."""
    key = (dev.index, T, B, max_q, H, H_kv, D, bs, max_blocks, fmt)
    need = _TREE_WS.get(key)
    if need is None:
        if len(_TREE_WS) > 65536:  # token counts vary from step to step
            _TREE_WS.clear()
        need = _TREE_WS[key] = int(lib().lk_paged_tree_workspace_bytes(
            T, B, max_q, H, H_kv, D, bs, max_blocks, fmt))
    if workspace is None:
        if need == 0:
            return None, 0, None
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    nbytes = workspace.numel() * workspace.element_size()
    if nbytes < need:
        raise ValueError(f"workspace too small: need {need} bytes")
    return workspace.data_ptr(), nbytes, workspace


_TREE_WS: dict = {}  # shape -> lk_paged_tree_workspace_bytes, asked once per shape


def tree_workspace_bytes(num_tokens: int, num_seqs: int, max_q_len: int, H: int, H_kv: int,
                         D: int, block_size: int, max_blocks: int,
                         cache_dtype: torch.dtype = torch.bfloat16) -> int:
    """Bytes of a caller-owned workspace for paged_tree_attention (decode:
    num_tokens = num_seqs and max_q_len = 1), of the current device."""
    return int(lib().lk_paged_tree_workspace_bytes(
        num_tokens, num_seqs, max_q_len, H, H_kv, D, block_size, max_blocks,
        _KV_FORMATS.get(cache_dtype, LK_KV_16BIT)))


def paged_decode_q8(
    query: torch.Tensor,
    key_cache: QuantizedCache,
    value_cache: QuantizedCache,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    scale: float,
    out: Optional[torch.Tensor] = None,
    workspace: Optional[torch.Tensor] = None,
    status: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """paged_decode over 8-bit caches: query fp16 / bf16 [B, H, D] -> [B, H, D],
    D 64 or 128, any block size and G = H / H_kv. A context of 0 gives NaN rows."""
    fmt = _check_q8(key_cache, value_cache)
    dev = _cuda(query, *key_cache, *value_cache, block_tables, context_lens, out, workspace, status)
    return _tree(dev, query, key_cache.data, key_cache.scale, value_cache.data, value_cache.scale,
                 fmt, block_tables, context_lens, None, None, 1, scale, out, workspace, status)


def paged_tree_attention(
    query: torch.Tensor,
    key_cache: Union[torch.Tensor, QuantizedCache],
    value_cache: Union[torch.Tensor, QuantizedCache],
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    max_q_len: int,
    scale: float,
    tree_mask: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    workspace: Optional[torch.Tensor] = None,
    status: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Attention of a tree of drafted tokens over the paged cache.

    query fp16 / bf16 [T, H, D] packed by cu_seqlens_q (int32 [B + 1]); the n
    tokens of sequence b, n <= max_q_len, are the last n of its context_lens[b]
    tokens, already stored (store_kvcache / store_kvcache_q8). Token i sees the
    keys before them and the d-th of them where bit d of its row of tree_mask
    (int64 [T, words], word d // 64; tree_mask_from_parents) is set; without a
    mask the tokens are a chain (d <= i). A token that sees nothing is NaN.
    Caches: 16-bit tensors of the query's dtype or QuantizedCache pairs.
    """
    if isinstance(key_cache, QuantizedCache) or isinstance(value_cache, QuantizedCache):
        fmt = _check_q8(key_cache, value_cache)
        (kd, ks), (vd, vs) = key_cache, value_cache
    else:
        fmt, kd, ks, vd, vs = LK_KV_16BIT, key_cache, None, value_cache, None
    dev = _cuda(query, kd, ks, vd, vs, block_tables, context_lens, cu_seqlens_q, tree_mask, out,
                workspace, status)
    if fmt == LK_KV_16BIT:
        if kd.dim() != 4 or vd.shape != kd.shape:
            raise ValueError("cache shape mismatch")
        if kd.dtype != query.dtype or vd.dtype != query.dtype:
            raise TypeError("query dtype must match the cache dtype")
        if not (kd.is_contiguous() and vd.is_contiguous()):
            raise ValueError("caches must be contiguous")
    if cu_seqlens_q.dtype != torch.int32 or cu_seqlens_q.numel() != block_tables.shape[0] + 1:
        raise TypeError("cu_seqlens_q must be int32 [B + 1]")
    max_q_len = int(max_q_len)
    if max_q_len < 0:
        raise ValueError("max_q_len must not be negative")
    if tree_mask is not None:
        if tree_mask.dtype != torch.int64 or tree_mask.dim() != 2 or tree_mask.shape[0] != query.shape[0]:
            raise TypeError("tree_mask must be int64 [T, words]")
        if tree_mask.shape[1] * 64 < max_q_len:
            raise ValueError("tree_mask must have a bit for each of max_q_len tokens")
        if tree_mask.stride(1) != 1:
            tree_mask = tree_mask.contiguous()
    return _tree(dev, query, kd, ks, vd, vs, fmt, block_tables, context_lens,
                 cu_seqlens_q.contiguous(), tree_mask, max_q_len, scale, out, workspace, status)


def _tree(dev, query, kd, ks, vd, vs, fmt, block_tables, context_lens, cu, mask, max_q, scale, out,
          workspace, status):
    if query.dim() != 3:
        raise ValueError("query must be [T, H, D]")
    T, H, D = query.shape
    nb, bs, H_kv, Dk = kd.shape
    if Dk != D:
        raise ValueError("cache shape mismatch")
    if query.stride(2) != 1 or query.stride(1) != D:
        raise ValueError("query must have unit d-stride and head stride D")
    if block_tables.dtype != torch.int32 or block_tables.dim() != 2:
        raise TypeError("block_tables must be int32 [B, max_blocks]")
    B, max_blocks = block_tables.shape
    if cu is None and B != T:
        raise ValueError("decode takes one query per row of block_tables")
    if block_tables.stride(1) != 1 and max_blocks > 0:
        block_tables = block_tables.contiguous()
    if context_lens.dtype != torch.int32 or context_lens.numel() != B:
        raise TypeError("context_lens must be int32 [B]")
    context_lens = context_lens.contiguous()
    code = _dtype_code(query)
    _check_status(status)
    if out is None:
        out = torch.empty((T, H, D), dtype=query.dtype, device=dev)
    elif out.shape != (T, H, D) or out.dtype != query.dtype or out.stride(2) != 1 or out.stride(1) != D:
        raise ValueError("bad out tensor")
    if T == 0 or B == 0 or max_q == 0:
        return out
    with _on(dev):
        ws, ws_bytes, keep = _tree_workspace(dev, workspace, T, B, max_q, H, H_kv, D, bs,
                                             max_blocks, fmt)
        args = (B, H, H_kv, D, bs, max_blocks, float(scale), code, fmt, ws, ws_bytes, _ptr(status),
                _stream(dev))
        head = (out.data_ptr(), out.stride(0), query.data_ptr(), query.stride(0), kd.data_ptr(),
                _ptr(ks), vd.data_ptr(), _ptr(vs), nb, block_tables.data_ptr(),
                block_tables.stride(0))
        if cu is None:
            check(lib().lk_paged_decode_q8(*head, context_lens.data_ptr(), *args))
        else:
            check(
                lib().lk_paged_tree_attention(
                    *head, cu.data_ptr(), context_lens.data_ptr(), _ptr(mask),
                    0 if mask is None else mask.stride(0), 0 if mask is None else mask.shape[1], T,
                    B, max_q, *args[1:],
                )
            )
    return out


def tree_mask_from_parents(parents, device=None) -> torch.Tensor:
    """The int64 [T, words] mask of paged_tree_attention from each sequence's
    list of parent indices: parents[b][i] < i is the drafted token that token i
    of sequence b continues, -1 for one that continues the context. Built on
    the host."""
    words = max(1, -(-max((len(p) for p in parents), default=0) // 64))
    rows = []
    for p in parents:
        sees = []
        for i, parent in enumerate(p):
            if not -1 <= parent < i:
                raise ValueError(f"token {i}: parent {parent} is not an earlier token or -1")
            sees.append((sees[parent] if parent >= 0 else 0) | (1 << i))
        rows += sees
    out = []
    for bits in rows:
        w = [(bits >> (64 * k)) & (2**64 - 1) for k in range(words)]
        out.append([x - 2**64 if x >> 63 else x for x in w])
    return torch.tensor(out, dtype=torch.int64).view(len(rows), words).to(device or "cpu")


# ----------------------------------------------------------- paged decode ---
def decode_num_splits(B: int, H_kv: int, max_blocks: int, block_size: int) -> int:
    return int(lib().lk_paged_decode_num_splits(B, H_kv, max_blocks, block_size))


def decode_workspace_bytes(B: int, H: int, H_kv: int, D: int, num_splits: int) -> int:
    return int(lib().lk_paged_decode_workspace_bytes(B, H, H_kv, D, num_splits))


def paged_decode(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    scale: float,
    num_splits: int = 0,
    out: Optional[torch.Tensor] = None,
    workspace: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Single-token paged attention; mirrors Attention._decode_fast
    (litevllm/layers/attention.py:91-139). query [B, H, D] -> [B, H, D]."""
    dev = _cuda(query, key_cache, value_cache, block_tables, context_lens, out, workspace)
    if query.dim() != 3:
        raise ValueError("query must be [B, H, D]")
    B, H, D = query.shape
    nb, bs, H_kv, Dk = key_cache.shape
    if Dk != D or value_cache.shape != key_cache.shape:
        raise ValueError("cache shape mismatch")
    if not (key_cache.is_contiguous() and value_cache.is_contiguous()):
        raise ValueError("caches must be contiguous")
    if query.dtype != key_cache.dtype:
        raise TypeError("query dtype must match the cache dtype")
    if query.stride(2) != 1 or query.stride(1) != D:
        raise ValueError("query must have unit d-stride and head stride D")
    if block_tables.dtype != torch.int32 or block_tables.dim() != 2 or block_tables.shape[0] != B:
        raise TypeError("block_tables must be int32 [B, max_blocks]")
    if block_tables.stride(1) != 1:
        block_tables = block_tables.contiguous()
    if context_lens.dtype != torch.int32 or context_lens.numel() != B:
        raise TypeError("context_lens must be int32 [B]")
    context_lens = context_lens.contiguous()
    code = _dtype_code(query, (torch.float32, torch.float16, torch.bfloat16))
    if out is None:
        out = torch.empty((B, H, D), dtype=query.dtype, device=dev)
    elif out.shape != (B, H, D) or out.dtype != query.dtype or out.stride(2) != 1 or out.stride(1) != D:
        raise ValueError("bad out tensor")
    if B == 0:
        return out
    max_blocks = block_tables.shape[1]
    plan_key = (B, H, H_kv, D, bs, max_blocks, query.dtype, int(num_splits))
    plan = _DECODE_PLANS.get(plan_key)
    if plan is None:
        num_splits = int(num_splits)
        if num_splits == 0:  # auto split count; -1 selects the persistent kernel
            num_splits = decode_num_splits(B, H_kv, max_blocks, bs)
        need = decode_workspace_bytes(B, H, H_kv, D, num_splits)
        want = need
        if not _decode_takes_split_kernel(query.dtype, D, bs, H // H_kv):
            # room for the generic kernel's split-KV partials (less only means fewer splits)
            want = max(need, int(lib().lk_paged_attention_generic_workspace_bytes(
                B, H, D, max_blocks, bs)))
        plan = _DECODE_PLANS[plan_key] = (num_splits, need, want)
    num_splits, need, want = plan
    stream = _stream(dev)
    if workspace is None:
        workspace = WORKSPACES.get(dev, f"decode:{stream}", want)
    elif workspace.numel() * workspace.element_size() < need:
        raise ValueError(f"workspace too small: need {need} bytes")
    with _on(dev):
        check(
            lib().lk_paged_decode(
                out.data_ptr(), out.stride(0), query.data_ptr(), query.stride(0),
                key_cache.data_ptr(), value_cache.data_ptr(), nb, block_tables.data_ptr(),
                block_tables.stride(0), context_lens.data_ptr(), B, H, H_kv, D, bs, max_blocks,
                float(scale), num_splits, workspace.data_ptr(),
                workspace.numel() * workspace.element_size(), code, stream,
            )
        )
    return out


# (B, H, H_kv, D, block_size, max_blocks, dtype, num_splits argument) ->
# (split count, workspace bytes the kernel needs, bytes to allocate): the
# library's answers for a shape, asked once per shape instead of per call.
_DECODE_PLANS: dict = {}


def paged_decode_shared_prefix(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    scale: float,
    prefix_tokens: int,
    out: Optional[torch.Tensor] = None,
    workspace: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """paged_decode for a batch whose rows share their first prefix_tokens
    tokens (the same physical blocks at the start of every block-table row):
    the shared part runs once, on the tensor cores, for all rows. Same result
    as paged_decode (Attention._decode_fast, litevllm/layers/attention.py:91-139)."""
    dev = _cuda(query, key_cache, value_cache, block_tables, context_lens, out, workspace)
    if query.dim() != 3:
        raise ValueError("query must be [B, H, D]")
    B, H, D = query.shape
    nb, bs, H_kv, Dk = key_cache.shape
    if Dk != D or value_cache.shape != key_cache.shape:
        raise ValueError("cache shape mismatch")
    if not (key_cache.is_contiguous() and value_cache.is_contiguous()):
        raise ValueError("caches must be contiguous")
    if query.dtype != key_cache.dtype:
        raise TypeError("query dtype must match the cache dtype")
    if query.stride(2) != 1 or query.stride(1) != D:
        raise ValueError("query must have unit d-stride and head stride D")
    if block_tables.dtype != torch.int32 or block_tables.dim() != 2 or block_tables.shape[0] != B:
        raise TypeError("block_tables must be int32 [B, max_blocks]")
    block_tables = block_tables.contiguous()
    if context_lens.dtype != torch.int32 or context_lens.numel() != B:
        raise TypeError("context_lens must be int32 [B]")
    context_lens = context_lens.contiguous()
    code = _dtype_code(query)
    if out is None:
        out = torch.empty((B, H, D), dtype=query.dtype, device=dev)
    if B == 0:
        return out
    max_blocks = block_tables.shape[1]
    need = int(lib().lk_paged_decode_shared_prefix_workspace_bytes(B, H, H_kv, D, max_blocks, bs,
                                                                    int(prefix_tokens)))
    if need == 0:
        raise ValueError("invalid shared-prefix decode shape")
    if workspace is None:
        workspace = WORKSPACES.get(dev, f"decode:{_stream(dev)}", need)
    elif workspace.numel() * workspace.element_size() < need:
        raise ValueError(f"workspace too small: need {need} bytes")
    with _on(dev):
        check(
            lib().lk_paged_decode_shared_prefix(
                out.data_ptr(), out.stride(0), query.data_ptr(), query.stride(0),
                key_cache.data_ptr(), value_cache.data_ptr(), nb, block_tables.data_ptr(),
                block_tables.stride(0), context_lens.data_ptr(), B, H, H_kv, D, bs, max_blocks,
                float(scale), int(prefix_tokens), workspace.data_ptr(),
                workspace.numel() * workspace.element_size(), code, _stream(dev),
            )
        )
    return out


def decode_status(workspace: Optional[torch.Tensor] = None, device=None) -> int:
    """Read (and clear) the LK_STATUS_* bits the decode kernels left in their
    workspace (by default the current stream's). Synchronises the current stream."""
    if workspace is None:
        dev = torch.device("cuda", torch.cuda.current_device() if device is None else device)
        workspace = WORKSPACES.get(dev, f"decode:{_stream(dev)}", 256)
    v = int(workspace[:4].view(torch.int32).item())
    workspace[:4].zero_()
    return v


# --------------------------------------------------------- paged prefill ---
def paged_prefill(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    max_q_len: int,
    scale: float,
    block_tables: Optional[torch.Tensor] = None,
    context_lens: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    status: Optional[torch.Tensor] = None,
    workspace: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Causal attention for prefill chunks over prior paged context.

    query [T, H, D] packed by cu_seqlens_q (int32 [S+1]). Paged mode
    (block_tables given): caches [num_blocks, bs, H_kv, D], context_lens =
    prior + chunk length per sequence. Contiguous mode (block_tables None):
    key_cache/value_cache are the chunk's own [T, H_kv, D] keys/values and
    every sequence starts at position 0 (Attention._prefill,
    litevllm/layers/attention.py:141-151).
    """
    dev = _cuda(query, key_cache, value_cache, cu_seqlens_q, block_tables, context_lens, out, status, workspace)
    if query.dim() != 3:
        raise ValueError("query must be [T, H, D]")
    T, H, D = query.shape
    if query.stride(2) != 1 or query.stride(1) != D:
        raise ValueError("query must have unit d-stride and head stride D")
    if block_tables is not None:
        nb, bs, H_kv, Dk = key_cache.shape
        if not (key_cache.is_contiguous() and value_cache.is_contiguous()):
            raise ValueError("caches must be contiguous")
        if block_tables.dtype != torch.int32 or block_tables.stride(1) != 1:
            raise TypeError("block_tables must be int32 with unit column stride")
        if context_lens is None or context_lens.dtype != torch.int32:
            raise TypeError("context_lens must be int32 in paged mode")
        context_lens = context_lens.contiguous()
        bt_stride = block_tables.stride(0)
        num = nb
    else:
        if key_cache.dim() != 3:
            raise ValueError("contiguous mode wants key/value [T, H_kv, D]")
        key_cache = key_cache.contiguous()
        value_cache = value_cache.contiguous()
        Tk, H_kv, Dk = key_cache.shape
        bs, bt_stride, num = 16, 0, Tk
        context_lens = None
    if Dk != D or value_cache.shape != key_cache.shape:
        raise ValueError("key/value shape mismatch")
    if query.dtype != key_cache.dtype:
        raise TypeError("query dtype must match the cache dtype")
    if cu_seqlens_q.dtype != torch.int32:
        raise TypeError("cu_seqlens_q must be int32")
    cu_seqlens_q = cu_seqlens_q.contiguous()
    S = cu_seqlens_q.numel() - 1
    code = _dtype_code(query, (torch.float32, torch.float16, torch.bfloat16))
    if out is None:
        out = torch.empty((T, H, D), dtype=query.dtype, device=dev)
    elif out.shape != (T, H, D) or not out.is_contiguous():
        raise ValueError("bad out tensor")
    if S <= 0 or T == 0:
        return out
    need = int(lib().lk_paged_prefill_workspace_bytes())
    if workspace is None:
        # one per stream: the plan and the split partials belong to one launch at a time
        workspace = WORKSPACES.get(dev, f"prefill:{_stream(dev)}", need)
    elif workspace.numel() * workspace.element_size() < need:
        raise ValueError(f"workspace too small: need {need} bytes")
    with _on(dev):
        check(
            lib().lk_paged_prefill_ws(
                out.data_ptr(), query.data_ptr(), query.stride(0), key_cache.data_ptr(),
                value_cache.data_ptr(), num, _ptr(block_tables), bt_stride,
                cu_seqlens_q.data_ptr(), _ptr(context_lens), S, int(max_q_len), H, H_kv, D, bs,
                float(scale), code, workspace.data_ptr(),
                workspace.numel() * workspace.element_size(), _ptr(status), _stream(dev),
            )
        )
    return out


def _decode_takes_split_kernel(dtype: torch.dtype, head_dim: int, block_size: int, G: int) -> bool:
    """lk_paged_decode's own routing: 16-bit caches, head_dim 128, block sizes
    that are multiples of 16 and G <= 8 run the split kernel (G need not be a
    power of two there); everything else the generic kernel, whose split-KV
    partials want a larger workspace."""
    return (dtype in (torch.float16, torch.bfloat16) and head_dim == 128
            and block_size % 16 == 0 and G <= 8)


def tuned_attention_shape(dtype: torch.dtype, head_dim: int, block_size: int, G: int) -> bool:
    """True when the tuned prefill and shared-prefix kernels take this shape
    (their tensor-core tiles hold 128 / G positions, so G is 1, 2, 4 or 8);
    other shapes run the generic CUDA-core kernel (fp32 caches, head dims
    other than 128, block sizes not a multiple of 16, other G). The decode
    split kernel takes every G <= 8 (_decode_takes_split_kernel)."""
    return (dtype in (torch.float16, torch.bfloat16) and head_dim == 128
            and block_size % 16 == 0 and G in (1, 2, 4, 8))


def paged_attention_generic(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    scale: float,
    block_tables: Optional[torch.Tensor] = None,
    context_lens: Optional[torch.Tensor] = None,
    cu_seqlens_q: Optional[torch.Tensor] = None,
    max_q_len: Optional[int] = None,
    status: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """The generic CUDA-core kernel called directly (lk_paged_attention_generic).

    cu_seqlens_q None: decode, one query per row at position
    context_lens[b] - 1 (Attention._decode_fast). Otherwise prefill chunks as in
    paged_prefill: paged when block_tables is given, else key_cache /
    value_cache are the chunk's own [T, H_kv, D] keys / values.
    """
    dev = _cuda(query, key_cache, value_cache, block_tables, context_lens, cu_seqlens_q, status)
    T, H, D = query.shape
    if query.stride(2) != 1 or query.stride(1) != D:
        raise ValueError("query must have unit d-stride and head stride D")
    if query.dtype != key_cache.dtype or value_cache.shape != key_cache.shape:
        raise TypeError("query / cache dtype or shape mismatch")
    key_cache, value_cache = key_cache.contiguous(), value_cache.contiguous()
    if block_tables is not None:
        nb, bs, H_kv, _ = key_cache.shape
        if block_tables.dtype != torch.int32 or block_tables.stride(1) != 1:
            raise TypeError("block_tables must be int32 with unit column stride")
        bt_stride, max_blocks = block_tables.stride(0), block_tables.shape[1]
    else:
        nb, H_kv, _ = key_cache.shape
        bs, bt_stride, max_blocks = 16, 0, 0
    if context_lens is not None:
        context_lens = context_lens.contiguous()
    if cu_seqlens_q is None:
        S, mq = T, 1
    else:
        cu_seqlens_q = cu_seqlens_q.contiguous()
        S = cu_seqlens_q.numel() - 1
        # without max_q_len, the row count bounds every chunk (no device read)
        mq = int(max_q_len) if max_q_len is not None else T
    code = _dtype_code(query, (torch.float32, torch.float16, torch.bfloat16))
    out = torch.empty((T, H, D), dtype=query.dtype, device=dev)
    with _on(dev):
        check(
            lib().lk_paged_attention_generic(
                out.data_ptr(), out.stride(0), query.data_ptr(), query.stride(0),
                key_cache.data_ptr(), value_cache.data_ptr(), nb, _ptr(block_tables), bt_stride,
                _ptr(cu_seqlens_q), _ptr(context_lens), S, mq, H, H_kv, D, bs, max_blocks,
                float(scale), code, _ptr(status), _stream(dev),
            )
        )
    return out


# ---------------------------------------------------------------- sampler ---
def sample(
    logits: torch.Tensor,
    temperatures: Optional[torch.Tensor] = None,
    noise: Optional[torch.Tensor] = None,
    seed: int = 0,
    offset: int = 0,
    noise_dump: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    workspace: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Greedy / Gumbel-max token ids, int64 [B].

    temperatures: fp32 [B] (0 = greedy row) or None (all greedy).
    noise: fp32 [B, >=V] Gumbel noise, or None for in-kernel Philox noise
    keyed by (seed, offset); noise_dump (fp32 [B, V]) receives that noise.
    """
    if logits.dim() == 1:
        logits = logits.unsqueeze(0)
    dev = _cuda(logits, temperatures, noise, noise_dump, out, workspace)
    B, V = logits.shape
    if logits.stride(1) != 1:
        logits = logits.contiguous()
    code = _dtype_code(logits, (torch.float32, torch.float16, torch.bfloat16))
    if temperatures is not None:
        if temperatures.dtype != torch.float32 or temperatures.numel() != B:
            raise TypeError("temperatures must be fp32 [B]")
        temperatures = temperatures.contiguous()
    noise_ld = 0
    if noise is not None:
        if noise.dtype != torch.float32 or noise.shape[0] != B or noise.shape[1] < V or noise.stride(1) != 1:
            raise TypeError("noise must be fp32 [B, >=V] with unit column stride")
        noise_ld = noise.stride(0)
    if noise_dump is not None:
        if noise_dump.dtype != torch.float32 or noise_dump.shape != (B, V) or not noise_dump.is_contiguous():
            raise TypeError("noise_dump must be contiguous fp32 [B, V]")
    if out is None:
        out = torch.empty(B, dtype=torch.int64, device=dev)
    if B == 0:
        return out
    need = _SAMPLE_WS.get((B, V))
    if need is None:
        need = _SAMPLE_WS[(B, V)] = int(lib().lk_sample_workspace_bytes(B, V))
    stream = _stream(dev)
    if workspace is None:
        workspace = WORKSPACES.get(dev, f"sample:{stream}", need)
    with _on(dev):
        check(
            lib().lk_sample(
                out.data_ptr(), logits.data_ptr(), B, V, logits.stride(0), _ptr(temperatures),
                _ptr(noise), noise_ld, seed & (2**64 - 1), offset & (2**64 - 1), _ptr(noise_dump),
                workspace.data_ptr(), workspace.numel() * workspace.element_size(), code, stream,
            )
        )
    return out


_SAMPLE_WS: dict = {}  # (B, V) -> lk_sample_workspace_bytes, asked once per shape


def sample_filtered(
    logits: torch.Tensor,
    temperatures: torch.Tensor,
    top_k: Optional[torch.Tensor] = None,
    top_p: Optional[torch.Tensor] = None,
    noise: Optional[torch.Tensor] = None,
    seed: int = 0,
    offset: int = 0,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Top-k / top-p filtered Gumbel-max sampling (fp32 / f16 / bf16 logits), int64 [B].
    Mirrors Sampler.sample's filtered branch (litevllm/layers/sampler.py:178-225)."""
    if logits.dim() == 1:
        logits = logits.unsqueeze(0)
    dev = _cuda(logits, temperatures, top_k, top_p, noise, out)
    B, V = logits.shape
    if logits.stride(1) != 1:
        logits = logits.contiguous()
    code = _dtype_code(logits, (torch.float32, torch.float16, torch.bfloat16))
    temperatures = temperatures.to(torch.float32).contiguous()
    if top_k is not None:
        top_k = top_k.to(torch.int32).contiguous()
    if top_p is not None:
        top_p = top_p.to(torch.float32).contiguous()
    noise_ld = 0
    if noise is not None:
        if noise.dtype != torch.float32 or noise.shape[0] != B or noise.shape[1] < V or noise.stride(1) != 1:
            raise TypeError("noise must be fp32 [B, >=V]")
        noise_ld = noise.stride(0)
    if out is None:
        out = torch.empty(B, dtype=torch.int64, device=dev)
    if B == 0:
        return out
    with _on(dev):
        check(
            lib().lk_sample_filtered(
                out.data_ptr(), logits.data_ptr(), B, V, logits.stride(0), temperatures.data_ptr(),
                _ptr(top_k), _ptr(top_p), _ptr(noise), noise_ld, seed & (2**64 - 1),
                offset & (2**64 - 1), code, _stream(dev),
            )
        )
    return out


def softmax_temp(logits: torch.Tensor, temperatures: torch.Tensor) -> torch.Tensor:
    """fp32 softmax(logits / T) per row (the top-k / top-p path)."""
    if logits.dim() == 1:
        logits = logits.unsqueeze(0)
    dev = _cuda(logits, temperatures)
    B, V = logits.shape
    logits = logits.contiguous()
    code = _dtype_code(logits, (torch.float32, torch.float16, torch.bfloat16))
    temperatures = temperatures.to(torch.float32).contiguous()
    probs = torch.empty((B, V), dtype=torch.float32, device=dev)
    with _on(dev):
        check(
            lib().lk_softmax_temp(
                probs.data_ptr(), V, logits.data_ptr(), B, V, V, temperatures.data_ptr(), code,
                _stream(dev),
            )
        )
    return probs


def repetition_penalty_(
    logits: torch.Tensor,
    past_token_ids: torch.Tensor,
    penalty,
    status: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """In place: each distinct id of past_token_ids[b] gets s / p if s > 0 else
    s * p on row b of logits, p = penalty (a float, or fp32 [B] per row; 1.0
    leaves the row alone). The reference's _apply_repetition_penalty
    (litevllm/layers/sampler.py:190-201) on a caller-owned tensor."""
    if logits.dim() == 1:
        logits = logits.unsqueeze(0)
    if past_token_ids.dim() == 1:
        past_token_ids = past_token_ids.unsqueeze(0)
    dev = _cuda(logits, past_token_ids, status)
    B, V = logits.shape
    if logits.stride(1) != 1:
        raise ValueError("logits must have unit column stride")
    code = _dtype_code(logits, (torch.float32, torch.float16, torch.bfloat16))
    past = past_token_ids.to(device=dev, dtype=torch.int64)
    if past.shape[0] != B:
        raise ValueError("past_token_ids must have one row per logits row")
    if past.shape[1] > 0 and past.stride(1) != 1:
        past = past.contiguous()
    if isinstance(penalty, torch.Tensor):
        pens = penalty.to(device=dev, dtype=torch.float32).contiguous()
        if pens.numel() != B:
            raise ValueError("per-row penalties must have B entries")
    else:
        pens = torch.full((B,), float(penalty), dtype=torch.float32, device=dev)
    with _on(dev):
        check(
            lib().lk_repetition_penalty(
                logits.data_ptr(), B, V, logits.stride(0), past.data_ptr(),
                past.stride(0) if past.shape[1] > 0 else 0, past.shape[1], pens.data_ptr(),
                _ptr(status), code, _stream(dev),
            )
        )
    return logits


def process_logits(
    logits: torch.Tensor,
    prompt_ids: Optional[torch.Tensor] = None,
    prompt_lens: Optional[torch.Tensor] = None,
    output_ids: Optional[torch.Tensor] = None,
    output_lens: Optional[torch.Tensor] = None,
    repetition: Optional[torch.Tensor] = None,
    presence: Optional[torch.Tensor] = None,
    frequency: Optional[torch.Tensor] = None,
    bias_ids: Optional[torch.Tensor] = None,
    bias: Optional[torch.Tensor] = None,
    allowed: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    status: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Penalties, biases and a grammar mask on a step's logits [B, V] (fp32,
    fp16, bf16), in one pass (lk_process_logits has the formula).

    prompt_ids / output_ids: int64 [B, L], the first *_lens[b] (int32, all if
    None) of a row count, negative ids are padding. repetition (prompt and
    output tokens), presence, frequency (output tokens): fp32 [B]. bias_ids
    int64 / bias fp32 [B, n], n <= 1024: biases of one id add up. allowed:
    int32 [B, >= ceil(V / 32)], a 0 in bit v % 32 of word v // 32 makes token v
    -inf. Returns a new tensor, or out (which may be logits: in place).
    """
    if logits.dim() == 1:
        logits = logits.unsqueeze(0)
        out = out.unsqueeze(0) if out is not None and out.dim() == 1 else out
    dev = _cuda(logits, prompt_ids, prompt_lens, output_ids, output_lens, repetition, presence,
                frequency, bias_ids, bias, allowed, out, status)
    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError("logits must be [B, V]")
    B, V = logits.shape
    code = _dtype_code(logits, (torch.float32, torch.float16, torch.bfloat16))
    if logits.stride(1) != 1 or (B > 1 and logits.stride(0) < V):
        if out is not None and out.data_ptr() == logits.data_ptr():
            raise ValueError("in place, logits must have unit column stride and rows of their own")
        logits = logits.contiguous()
    ids_args = []
    for name, ids, lens in (("prompt", prompt_ids, prompt_lens), ("output", output_ids, output_lens)):
        if ids is None:
            ids_args += [None, 0, None, 0]
            continue
        if ids.dtype != torch.int64 or ids.dim() != 2 or ids.shape[0] != B:
            raise TypeError(f"{name}_ids must be int64 [B, L]")
        if ids.shape[1] > 0 and (ids.stride(1) != 1 or (B > 1 and ids.stride(0) < ids.shape[1])):
            ids = ids.contiguous()
        if lens is not None:
            if lens.dtype != torch.int32 or lens.numel() != B:
                raise TypeError(f"{name}_lens must be int32 [B]")
            lens = lens.contiguous()
        ids_args += [ids, max(ids.stride(0), ids.shape[1]), lens, ids.shape[1]]
    rows = []
    for name, x in (("repetition", repetition), ("presence", presence), ("frequency", frequency)):
        if x is not None:
            if x.dtype != torch.float32 or x.numel() != B:
                raise TypeError(f"{name} must be fp32 [B]")
            x = x.contiguous()
        rows.append(x)
    nbias = 0
    if (bias_ids is None) != (bias is None):
        raise ValueError("bias_ids and bias go together")
    if bias_ids is not None:
        if bias_ids.dtype != torch.int64 or bias_ids.dim() != 2 or bias_ids.shape[0] != B:
            raise TypeError("bias_ids must be int64 [B, n]")
        if bias.dtype != torch.float32 or bias.shape != bias_ids.shape:
            raise TypeError("bias must be fp32 [B, n]")
        bias_ids, bias = bias_ids.contiguous(), bias.contiguous()
        nbias = bias_ids.shape[1]
    allowed_ld = 0
    if allowed is not None:
        if allowed.dtype != torch.int32 or allowed.dim() != 2 or allowed.shape[0] != B or allowed.shape[1] * 32 < V:
            raise TypeError("allowed must be int32 [B, >= ceil(V / 32)]")
        if allowed.stride(1) != 1 or (B > 1 and allowed.stride(0) < allowed.shape[1]):
            allowed = allowed.contiguous()
        allowed_ld = max(allowed.stride(0), allowed.shape[1])
    _check_status(status)
    if out is None:
        out = torch.empty((B, V), dtype=logits.dtype, device=dev)
    elif (out.shape != (B, V) or out.dtype != logits.dtype or out.stride(1) != 1
          or (B > 1 and out.stride(0) < V)):
        raise ValueError("out must be [B, V] of the logits' dtype with unit column stride")
    if B == 0:
        return out
    ld, out_ld = max(logits.stride(0), V), max(out.stride(0), V)
    with _on(dev):
        check(
            lib().lk_process_logits(
                out.data_ptr(), out_ld, logits.data_ptr(), B, V, ld, _ptr(ids_args[0]), ids_args[1],
                _ptr(ids_args[2]), ids_args[3], _ptr(ids_args[4]), ids_args[5], _ptr(ids_args[6]),
                ids_args[7], _ptr(rows[0]), _ptr(rows[1]), _ptr(rows[2]), _ptr(bias_ids),
                _ptr(bias), nbias, _ptr(allowed), allowed_ld, code, _ptr(status), _stream(dev),
            )
        )
    return out


# ------------------------------------------------ norm + RoPE + KV store ---
def rope_store_kvcache(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    key_cache: Optional[torch.Tensor],
    value_cache: Optional[torch.Tensor],
    slot_mapping: Optional[torch.Tensor],
    positions: torch.Tensor,
    cos_cached: torch.Tensor,
    sin_cached: torch.Tensor,
    q_norm_weight: Optional[torch.Tensor] = None,
    k_norm_weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    status: Optional[torch.Tensor] = None,
    key_out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """In one launch: optional q/k RMSNorm, RoPE on q (in place) and k, and the
    store of k / v into the paged cache. Mirrors Qwen3Attention.forward
    (litevllm/models/qwen3.py:76-92) up to the attention call; returns query.
    key_out ([T, H_kv, D], may be key itself) receives the rotated k."""
    dev = _cuda(query, key, value, key_cache, value_cache, slot_mapping, positions, cos_cached,
                sin_cached, q_norm_weight, k_norm_weight, status, key_out)
    if key_out is not None and (key_out.shape != key.shape or key_out.dtype != key.dtype
                                or key_out.stride(2) != 1 or key_out.stride(1) != key.shape[2]):
        raise ValueError("key_out must match key's shape and dtype, unit d-stride, head stride D")
    T, H, D = query.shape
    H_kv = key.shape[1]
    for t in (query, key, value):
        if t.stride(2) != 1 or t.stride(1) != D:
            raise ValueError("q/k/v must have unit d-stride and head stride D")
    code = _dtype_code(query)
    if key.dtype != query.dtype or value.dtype != query.dtype:
        raise TypeError("q, k, v must share a dtype")
    if cos_cached.dtype != torch.float32 or sin_cached.dtype != torch.float32:
        raise TypeError("cos / sin tables must be fp32 (RotaryEmbedding buffers)")
    cos_cached, sin_cached = cos_cached.contiguous(), sin_cached.contiguous()
    positions = positions.to(torch.int64).contiguous()
    for w in (q_norm_weight, k_norm_weight):
        if w is not None and (w.dtype != query.dtype or w.numel() != D):
            raise TypeError("norm weights must be [D] in the activation dtype")
    num_slots = 0
    if slot_mapping is not None:
        if key_cache is None or value_cache is None or not key_cache.is_contiguous():
            raise ValueError("a slot mapping needs contiguous caches")
        slot_mapping = slot_mapping.to(torch.int64).contiguous()
        num_slots = key_cache.shape[0] * key_cache.shape[1]
    with _on(dev):
        check(
            lib().lk_rope_store_kv(
                query.data_ptr(), query.stride(0), key.data_ptr(), key.stride(0), value.data_ptr(),
                value.stride(0), _ptr(key_out), 0 if key_out is None else key_out.stride(0),
                _ptr(key_cache), _ptr(value_cache), num_slots, _ptr(slot_mapping),
                positions.data_ptr(), cos_cached.data_ptr(), sin_cached.data_ptr(),
                cos_cached.shape[0], _ptr(q_norm_weight), _ptr(k_norm_weight), float(eps), T, H,
                H_kv, D, code, _ptr(status), _stream(dev),
            )
        )
    return query


# ------------------------------------------------------------- block copies ---
def _device_address(t: torch.Tensor) -> int:
    if t.is_cuda:
        return t.data_ptr()
    if not t.is_pinned():
        raise RuntimeError("host caches must be pinned (page-locked) for device-side swaps")
    out = ctypes.c_uint64(0)
    check(lib().lk_host_device_pointer(t.data_ptr(), ctypes.byref(out)))
    return out.value


def copy_blocks_between(src_caches, dst_caches, mapping, device=None,
                        status: Optional[torch.Tensor] = None) -> None:
    """dst[layer][d] = src[layer][s] for every (s, d) in mapping and every layer,
    K and V, in one launch. src_caches / dst_caches: lists of (key_cache,
    value_cache) per layer ([num_blocks, bs, H_kv, D], contiguous); CUDA tensors
    or pinned host tensors. mapping: dict {src: dst}, list of pairs or int64
    [n, 2] tensor. Mirrors KVCache.swap_in / swap_out and blocks_to_copy
    (litevllm/cache/kv_cache.py:74-102, engine/scheduler.py:25-27)."""
    if len(src_caches) != len(dst_caches) or not src_caches:
        raise ValueError("need the same, non-zero number of layers on both sides")
    k0 = src_caches[0][0]
    for kc, vc in list(src_caches) + list(dst_caches):
        if kc.shape[1:] != k0.shape[1:] or vc.shape != kc.shape or kc.dtype != k0.dtype:
            raise ValueError("all caches must share block shape and dtype")
        if not (kc.is_contiguous() and vc.is_contiguous()):
            raise ValueError("caches must be contiguous")
    if device is None:
        devs = [t.device for pair in list(src_caches) + list(dst_caches) for t in pair if t.is_cuda]
        if not devs:
            raise RuntimeError("at least one side must be on a CUDA device")
        device = devs[0]
    device = torch.device(device)
    if isinstance(mapping, dict):
        pairs = list(mapping.items())
    elif isinstance(mapping, torch.Tensor):
        pairs = None
    else:
        pairs = list(mapping)
    if pairs is not None:
        if not pairs:
            return
        mapping = torch.tensor(pairs, dtype=torch.int64)
    mapping = mapping.to(device=device, dtype=torch.int64).contiguous().view(-1, 2)
    n = mapping.shape[0]
    if n == 0:
        return
    src_ptrs = torch.tensor([_device_address(t) for pair in src_caches for t in pair],
                            dtype=torch.uint64).to(device)
    dst_ptrs = torch.tensor([_device_address(t) for pair in dst_caches for t in pair],
                            dtype=torch.uint64).to(device)
    block_bytes = k0[0].numel() * k0.element_size()
    with _on(device):
        check(
            lib().lk_copy_blocks(
                src_ptrs.data_ptr(), dst_ptrs.data_ptr(), len(src_caches), mapping.data_ptr(), n,
                block_bytes, src_caches[0][0].shape[0], dst_caches[0][0].shape[0],
                _ptr(status), _stream(device),
            )
        )
    # src_ptrs / dst_ptrs / mapping are freed in stream order on the launching
    # stream, after the kernel that reads them.


def copy_blocks(caches, mapping) -> None:
    """Copy-on-write block copies inside one set of device caches."""
    copy_blocks_between(caches, caches, mapping)


def swap_in(gpu_caches, cpu_caches, mapping) -> None:
    """KVCache.swap_in: gpu[layer][dst] = cpu[layer][src] (pinned host caches)."""
    copy_blocks_between(cpu_caches, gpu_caches, mapping)


def swap_out(gpu_caches, cpu_caches, mapping) -> None:
    """KVCache.swap_out: cpu[layer][dst] = gpu[layer][src]; synchronises the
    stream so the host copy is complete on return."""
    copy_blocks_between(gpu_caches, cpu_caches, mapping)
    dev = next(t.device for pair in gpu_caches for t in pair)
    torch.cuda.current_stream(dev).synchronize()


def default_scale(head_dim: int) -> float:
    return 1.0 / math.sqrt(head_dim)

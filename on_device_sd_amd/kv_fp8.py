"""The paged KV cache in 8 bits: half the memory and half the traffic of a decode or verify step's attention.

A ``KVCacheFP8`` holds e4m3 numbers with a power-of-two scale for each block and KV head, one for K and one for V.
``store_kvcache_fp8`` is ``kv.store_kvcache`` for it, ``paged_attention_fp8`` is ``kv.paged_attention`` over it (the contexts are
the same).  The reference's cache is 16 bits wide (``demo/src/memory/paged_kv_cache.py:228-683``); there is no counterpart.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, Optional, Tuple

import torch

from . import _lib
from .ops import _NO_WORKSPACE, _ptr, _raw_device, _same_device, _stream, _wrote

_E4M3 = torch.float8_e4m3fn
_SHORT_LIST = 4096                                      # rows that the store takes without a workspace
_DTYPES = {torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_F16}


@dataclass
class KVCacheFP8:
    """One layer's cache; a value is its code times the scale of its block and head.  With a leading dimension of layers on all
    three it is a whole model's, and ``layer(i)`` is what store and attention take."""
    k: torch.Tensor        # float8_e4m3fn [num_blocks, num_kv_heads, block_size, head_dim]
    v: torch.Tensor        # float8_e4m3fn [num_blocks, num_kv_heads, head_dim, block_size]: transposed
    scales: torch.Tensor   # float32 [num_blocks, num_kv_heads, 2]: K's and V's, powers of two; 0: nothing is stored there

    @classmethod
    def zeros(cls, num_blocks: int, num_kv_heads: int, block_size: int, head_dim: int, device="cuda",
              layers: Optional[int] = None) -> "KVCacheFP8":
        """An empty cache.  block_size: a multiple of 16, 1024 at most; head_dim 64 or 128."""
        if block_size <= 0 or block_size % 16 or block_size > 1024 or head_dim not in (64, 128):
            raise ValueError(f"blocks of {block_size} tokens and heads of {head_dim}: a multiple of 16 up to 1024, and 64 or 128, are held")
        lead = () if layers is None else (layers,)
        make = lambda *shape: torch.zeros(lead + shape, dtype=torch.uint8, device=device).view(_E4M3)  # noqa: E731
        return cls(make(num_blocks, num_kv_heads, block_size, head_dim), make(num_blocks, num_kv_heads, head_dim, block_size),
                   torch.zeros(lead + (num_blocks, num_kv_heads, 2), dtype=torch.float32, device=device))

    def layer(self, i: int) -> "KVCacheFP8":
        return KVCacheFP8(self.k[i], self.v[i], self.scales[i])


def _cache_shape(cache: KVCacheFP8) -> Tuple[int, int, int, int]:
    """(blocks, KV heads, tokens of a block, head size) of one layer's cache."""
    k, v, scales = cache.k, cache.v, cache.scales
    shape = k.shape
    if len(shape) != 4:
        raise ValueError("the cache must be one layer's: k [num_blocks, num_kv_heads, block_size, head_dim]")
    blocks, heads, block_size, head_dim = shape
    if v.shape != (blocks, heads, head_dim, block_size) or scales.shape != (blocks, heads, 2):
        raise ValueError(f"k {tuple(shape)}, v {tuple(v.shape)} and scales {tuple(scales.shape)} are not one cache")
    if k.dtype != _E4M3 or v.dtype != _E4M3 or scales.dtype != torch.float32:
        raise TypeError("an 8-bit cache is float8_e4m3fn with float32 scales")
    if not (k.is_contiguous() and v.is_contiguous() and scales.is_contiguous()):
        raise ValueError("the cache must be contiguous")
    if blocks * max(block_size, heads) >> 31:              # (slots and block numbers are 31 bits in the library)
        raise _lib.OdsdError(f"8-bit cache: unsupported sizes: {blocks} blocks of {block_size} tokens, {heads} heads")
    return blocks, heads, block_size, head_dim


def store_kvcache_fp8(key: torch.Tensor, value: torch.Tensor, cache: KVCacheFP8, slot_mapping: torch.Tensor,
                      src_index: Optional[torch.Tensor] = None) -> None:
    """key, value [n, num_kv_heads, head_dim] (bfloat16 / float16; views of a fused projection as they are) to their slots of the
    cache: slot_mapping int32 [N], block * block_size + token of the block (-1 = no slot).  Without ``src_index`` N == n and row i
    is stored; with it (int32 [N]) row ``src_index[i]`` is.  Of two rows with one slot the later stays.

    A block's scale is the smallest power of two (2^-64 at least) by which all that is stored there is 448 at most.  It only rises: the
    codes of rows that stay are rounded again then, which costs bits only where they fall below 2^-6.  Token 0 of a block starts it
    anew: its scale is that of the call's rows, and what other tokens of the block held is given up (positions are written in order).
    Infinities become the largest number, 448 times the scale; NaN stays."""
    dev = key.get_device()
    _same_device(dev, value, cache.k, cache.v, cache.scales, slot_mapping, src_index)
    if dev != _raw_device():
        with torch.cuda.device(dev):
            return store_kvcache_fp8(key, value, cache, slot_mapping, src_index)
    code = _DTYPES.get(key.dtype)
    if code is None or value.dtype != key.dtype:
        raise TypeError(f"the 8-bit store takes bfloat16 or float16 keys and values alike, got {key.dtype} and {value.dtype}")
    blocks, heads, block_size, head_dim = _cache_shape(cache)
    shape = key.shape
    if len(shape) != 3 or value.shape != shape or shape[1:] != (heads, head_dim):
        raise ValueError(f"key {tuple(shape)} and value {tuple(value.shape)} must be [n, {heads}, {head_dim}]")
    n, N = shape[0], slot_mapping.numel()
    if slot_mapping.dtype != torch.int32:
        slot_mapping = slot_mapping.to(torch.int32)
    slot_mapping = slot_mapping.contiguous()
    if src_index is None:
        if N != n:
            raise ValueError("slot_mapping must name a slot (or -1) for every row that is stored")
    else:
        if src_index.numel() != N:
            raise ValueError("slot_mapping must name a slot (or -1) for every row that is stored")
        if src_index.dtype != torch.int32:
            src_index = src_index.to(torch.int32)
        src_index = src_index.contiguous()
    if (n | N) >> 31:
        raise _lib.OdsdError(f"8-bit store: unsupported sizes: {N} of {n} rows")
    ks, vs = key.stride(), value.stride()
    if ks[2] != 1:
        key = key.contiguous()
        ks = key.stride()
    if vs[2] != 1:
        value = value.contiguous()
        vs = value.stride()
    lib, ws, nbytes = _lib.load(), None, 0
    if N > _SHORT_LIST:
        nbytes = lib.odsd_kv_store_fp8_workspace_bytes(N)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=key.device)
    rc = lib.odsd_kv_store_fp8(key.data_ptr(), ks[0], ks[1], value.data_ptr(), vs[0], vs[1], cache.k.data_ptr(), cache.v.data_ptr(),
                               cache.scales.data_ptr(), slot_mapping.data_ptr(), _ptr(src_index), N, n, heads, head_dim, block_size, blocks,
                               code, _ptr(ws), nbytes, _stream())
    if rc:
        _lib.check(rc, "odsd_kv_store_fp8")
    _wrote(cache.k, cache.v, cache.scales)


def paged_attention_fp8(q: torch.Tensor, cache: KVCacheFP8, context: Dict[str, torch.Tensor], softmax_scale: Optional[float] = None,
                        max_q_len: Optional[int] = None) -> torch.Tensor:
    """``paged_attention`` over an 8-bit cache that holds this step's keys and values already: q [n_tokens, num_heads, head_dim]
    (bfloat16 / float16), ``context`` with ``block_tables`` int32 [n_seqs, max_blocks], ``context_lens`` int32 [n_seqs] and, for a verify
    step or a chunk of a prompt, ``verify_query_lens`` int32 [n_seqs].  Query j of a sequence attends positions 0 .. context_len -
    query_len + j; a sequence without keys gets zeros.  ``max_q_len`` bounds the query lengths (default: the context's
    ``max_query_len``, else n_tokens): rows of a sequence past it, and rows behind the last sequence's, hold nothing in particular."""
    dev = q.get_device()
    _same_device(dev, cache.k, cache.v, cache.scales)
    if dev != _raw_device():
        with torch.cuda.device(dev):
            return paged_attention_fp8(q, cache, context, softmax_scale, max_q_len)
    code = _DTYPES.get(q.dtype)
    if code is None:
        raise TypeError(f"attention over the 8-bit cache takes bfloat16 or float16 queries, got {q.dtype}")
    blocks, kv_heads, block_size, head_dim = _cache_shape(cache)
    if q.dim() != 3 or q.shape[2] != head_dim or q.shape[1] % max(kv_heads, 1):
        raise ValueError(f"q {tuple(q.shape)} does not fit {kv_heads} KV heads of {head_dim}")
    n_tokens, num_heads, _ = q.shape
    tables, lens, q_lens = context["block_tables"], context["context_lens"], context.get("verify_query_lens")
    n_seqs = lens.numel()
    if tables.dim() != 2 or tables.shape[0] != n_seqs:
        raise ValueError(f"block_tables {tuple(tables.shape)} for {n_seqs} sequences")
    most = 1
    if q_lens is None:
        if n_tokens != n_seqs:
            raise ValueError(f"{n_tokens} query tokens for {n_seqs} sequences without query lengths")
    else:
        if q_lens.numel() != n_seqs:
            raise ValueError(f"{q_lens.numel()} query lengths for {n_seqs} sequences")
        most = max_q_len or context.get("max_query_len") or n_tokens
        if not q_lens.is_cuda and n_seqs:                   # readable without a device synchronisation
            host = q_lens.tolist()
            if max(host) > most:
                raise ValueError(f"max_q_len={most} is below the longest query ({max(host)} tokens)")
            if min(host) < 0 or sum(host) > n_tokens:
                raise ValueError(f"query lengths {host} do not fit {n_tokens} tokens")
    q = q.contiguous()
    out = torch.empty_like(q)
    if n_seqs == 0 or n_tokens == 0:
        return out
    max_blocks = tables.shape[1]
    if max_blocks == 0:                                     # nobody has a key
        return out.zero_()
    tables, lens, q_lens = (t if t is None or (t.get_device() == dev and t.dtype == torch.int32 and t.is_contiguous())
                            else t.to(device=q.device, dtype=torch.int32).contiguous() for t in (tables, lens, q_lens))
    lib, nbytes = _lib.load(), 0
    if not (n_tokens | n_seqs | most | num_heads | max_blocks) >> 31:        # (sizes are 31 bits in the library)
        nbytes = lib.odsd_paged_attention_fp8_workspace_bytes(n_seqs, most, num_heads, kv_heads, head_dim, block_size, max_blocks)
    if nbytes == 0:
        raise _lib.OdsdError(f"attention over the 8-bit cache: unsupported shape: {n_seqs} sequences of up to {most} queries, {num_heads} / "
                             f"{kv_heads} heads of {head_dim}, {max_blocks} blocks of {block_size}")
    ws = None if nbytes == _NO_WORKSPACE else q.new_empty(nbytes // 2)       # (of two-byte numbers)
    scale = head_dim ** -0.5 if softmax_scale is None else softmax_scale
    rc = lib.odsd_paged_attention_fp8(q.data_ptr(), cache.k.data_ptr(), cache.v.data_ptr(), cache.scales.data_ptr(), tables.data_ptr(),
                                      lens.data_ptr(), _ptr(q_lens), n_tokens, n_seqs, most, num_heads, kv_heads, head_dim, block_size, max_blocks,
                                      blocks, scale, code, out.data_ptr(), _ptr(ws), nbytes, _stream())
    if rc:
        _lib.check(rc, "odsd_paged_attention_fp8")
    return out

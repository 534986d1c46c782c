"""Paged K/V caches in 8 bits (tensor functions over the C ABI).

Pools are ``[pages, Hkv, block_size, D]`` of ``torch.float8_e4m3fn`` (any strides with
contiguous rows), with a scale for each page and head of K and of V, ``[pages, Hkv]``
float32, finite and 0 (a page of zeros) at least: a row's value is its 8 bits times its page's
scale. Pages, slots and tables are those of ``dropkv_b200.paged``; ``block_tables`` hands them out.

* ``store_rows_fp8`` -- K/V rows to slots, quantised;
* ``load_rows_fp8``  -- rows at slots, read back;
* ``attention_fp8``  -- attention over such a cache: single tokens, drafted trees, prompt
  chunks, with a sliding window and first rows that stay visible.

Scales are powers of two, so that the 8 bits' rounding (2^-4 of a value) is the only one:
what is read back is exact in 16 bits, and a page whose scale grows keeps its rows but for
those bits that fall under the new scale's smallest steps. No call synchronises the host. The
reference's cache holds the model's own type only (dropkv_cache.py:581-617).
"""

from __future__ import annotations

import functools
from typing import Optional

import torch

from . import _lib
from .ops import _CHECK_STATUS, _DTYPE_CODE
from .paged import _ints, _new, _on_its_device, _on_one_device, _raw_stream, _rows_strides

__all__ = ["store_rows_fp8", "load_rows_fp8", "attention_fp8"]

_F8, _F32 = torch.float8_e4m3fn, torch.float32


@functools.lru_cache(maxsize=4096)
def _attention_workspace(index: int, B: int, Hq: int, Hkv: int, T: int, D: int, cap: int) -> int:
    """Bytes of an attention_fp8 workspace on the current device ``index``."""
    return int(_lib.load().dropkv_attention_fp8_workspace_size(B, Hq, Hkv, T, D, cap))


def _check_pool_fp8(K_pages, V_pages, K_scales, V_scales):
    """The pools' shape [pages, Hkv, block_size, D], and the pointers and strides of pages and scales."""
    shape = K_pages.shape
    if len(shape) != 4 or shape != V_pages.shape:
        raise ValueError(f"expected K and V pages [pages, Hkv, block_size, D] of one shape, got {tuple(shape)} and "
                         f"{tuple(V_pages.shape)}")
    if K_pages.dtype != _F8 or V_pages.dtype != _F8:
        raise TypeError(f"pages must be torch.float8_e4m3fn, got {K_pages.dtype} and {V_pages.dtype}")
    if K_scales.dtype != _F32 or V_scales.dtype != _F32:
        raise TypeError(f"scales must be float32, got {K_scales.dtype} and {V_scales.dtype}")
    of = shape[:2]
    if K_scales.shape != of or V_scales.shape != of:
        raise ValueError(f"scales must be {tuple(of)} (pages, heads), got {tuple(K_scales.shape)} and {tuple(V_scales.shape)}")
    return shape, (K_pages.data_ptr(), *_rows_strides(K_pages, "K_pages"), V_pages.data_ptr(),
                   *_rows_strides(V_pages, "V_pages"), K_scales.data_ptr(), *K_scales.stride(), V_scales.data_ptr(),
                   *V_scales.stride())


@_on_its_device
def store_rows_fp8(K: torch.Tensor, V: torch.Tensor, slots: torch.Tensor, K_pages: torch.Tensor, V_pages: torch.Tensor,
                   K_scales: torch.Tensor, V_scales: torch.Tensor) -> None:
    """Rows of K and V [B, Hkv, N, D] (fp32, fp16 or bf16; any strides, rows of D contiguous)
    to slots [B, N] (int64) of pools in 8 bits, in place; rows whose slot is outside the pool
    (-1) are left out.

    A page's scale becomes the smallest power of two that brings the call's largest value in it
    to at most 448, unless it is more already; rows that stand in the page follow a scale that
    grows. A call that writes a page's row 0 starts the page: what stood in it before means
    nothing, and its scale is the call's alone. Values are rounded to nearest, ties to even, NaN
    stays NaN and infinities (e4m3 has none) become NaN.

    The rows of one page belong to one sequence of the call and follow one another there, their slots ascending, as
    ``block_tables`` hands them out, with fewer than 256 rows without a slot between two of them;
    otherwise, and where rows share a slot, that page's contents are unspecified. K and V must not
    lie in the pages. block_size is at most 1024.
    """
    dev = _on_one_device(K, V, slots, K_pages, V_pages, K_scales, V_scales)
    ks, dtype = K.shape, K.dtype
    if len(ks) != 4 or ks != V.shape:
        raise ValueError("expected K, V [B, Hkv, N, D] of one shape")
    dt = _DTYPE_CODE.get(dtype)
    if dt is None or V.dtype != dtype:
        raise TypeError(f"K and V must share one of fp32/fp16/bf16; got {dtype}, {V.dtype}")
    B, Hkv, N, D = ks
    ps, pool = _check_pool_fp8(K_pages, V_pages, K_scales, V_scales)
    if ps[1] != Hkv or ps[3] != D:
        raise ValueError(f"rows of {Hkv} heads of {D} do not fit pages {tuple(ps)}")
    slots = _ints(slots, torch.int64, (B, N), "slots")
    pack, call = _lib.words("dropkv_store_rows_fp8")
    rc = call(pack(K.data_ptr(), *_rows_strides(K, "K"), V.data_ptr(), *_rows_strides(V, "V"), slots.data_ptr(), *pool,
                   ps[0], ps[2], dt, B, Hkv, N, D, _raw_stream(dev)))
    if rc:
        _lib.check(rc, "dropkv_store_rows_fp8")


@_on_its_device
def load_rows_fp8(K_pages: torch.Tensor, V_pages: torch.Tensor, K_scales: torch.Tensor, V_scales: torch.Tensor,
                  slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16):
    """(K, V) [B, Hkv, N, D] in ``dtype`` (fp32, fp16 or bf16): the rows at slots [B, N] (int64)
    of pools in 8 bits, zeros where a slot is outside the pool (-1). Exact in every dtype unless
    a value is outside its range."""
    dev = _on_one_device(K_pages, V_pages, K_scales, V_scales, slots)
    dt = _DTYPE_CODE.get(dtype)
    if dt is None:
        raise TypeError(f"dtype must be fp32/fp16/bf16; got {dtype}")
    ps, pool = _check_pool_fp8(K_pages, V_pages, K_scales, V_scales)
    if slots.dim() != 2:
        raise ValueError(f"slots must be [B, N], got {tuple(slots.shape)}")
    B, N = slots.shape
    slots = _ints(slots, torch.int64, (B, N), "slots")
    device = K_pages.device
    k_out = _new(dtype, device, B, ps[1], N, ps[3])
    v_out = torch.empty_like(k_out)
    pack, call = _lib.words("dropkv_load_rows_fp8")
    rc = call(pack(*pool, ps[0], ps[2], slots.data_ptr(), dt, B, ps[1], N, ps[3], k_out.data_ptr(), v_out.data_ptr(),
                   _raw_stream(dev)))
    if rc:
        _lib.check(rc, "dropkv_load_rows_fp8")
    return k_out, v_out


@_on_its_device
def attention_fp8(Q: torch.Tensor, K_pages: torch.Tensor, V_pages: torch.Tensor, K_scales: torch.Tensor,
                  V_scales: torch.Tensor, cache_lens: torch.Tensor, block_table: torch.Tensor,
                  tree_mask: Optional[torch.Tensor] = None, window: Optional[int] = None, sinks: int = 0,
                  scale: Optional[float] = None) -> torch.Tensor:
    """Attention of T tokens over a cache in 8 bits: Q [B, Hq, T, D] (any strides) -> [B, Hq, T, D].

    Row b's cache holds ``cache_lens[b]`` (int32, on the device) rows in the pages of
    ``block_table`` ([B, max_blocks] int32), and after them the T tokens' own K/V rows. Token i
    sees every row up to its own, ``cache_lens[b] + i``: T = 1 is a decode step, a longer chain
    drafted tokens or a prompt's chunk. With ``tree_mask`` (bool [T, T] or [B, T, T], T at most
    256) it sees the cached rows and the nodes j with ``tree_mask[i, j]``.

    ``window``: of those only the last ``window`` rows up to its own (for a tree's node: up to
    the row of its depth, the number of nodes it sees but itself, and of the cached rows only; the window
    holds the whole tree) and the cache's first ``sinks`` rows. Rows are counted as they
    are stored: after an eviction the window holds the last rows kept.

    Rows past the table and on missing pages (-1) are not seen; a token that sees nothing gives
    zeros; what is in rows, pages or scales that no token sees does not matter. bf16 or fp16, D 64
    or 128, at most 128 query heads a KV head, B * Hkv at most 65535, Hq * T at most 2^26,
    B * Hq * T under 2^31, tables of fewer than 2^31 - 65536 rows, block_size a power of two from 8
    to 1024, page rows on 16-byte boundaries that do not overlap.

    The 8 bits enter the products as they are, queries as sums of 8-bit parts that leave at most
    2^-21 (bf16) or 2^-24 (fp16) of a row's largest element; a weight times its page's scale of V
    has 16 bits, off by at most 2^-11 of itself or 2^-32 of the token's largest such product; sums
    and softmax statistics have 32. The call's workspace is 2 to 40 MB, and with more than 8 query
    rows a KV head (Hq / Hkv * T; 16 at D 64) three bytes an element of Q besides, which at the
    largest Hq * T are 25 GB a sequence.
    """
    dev = _on_one_device(Q, K_pages, V_pages, K_scales, V_scales, cache_lens, block_table,
                         *((tree_mask,) if tree_mask is not None else ()))
    qs, dtype = Q.shape, Q.dtype
    if len(qs) != 4:
        raise ValueError(f"expected Q [B, Hq, T, D], got {tuple(qs)}")
    if dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"attention_fp8 takes bf16 or fp16 queries, got {dtype}")
    B, Hq, T, D = qs
    ps, pool = _check_pool_fp8(K_pages, V_pages, K_scales, V_scales)
    n_pages, Hkv, block, Dk = ps
    if Dk != D or not Hkv or Hq % Hkv:
        raise ValueError(f"shape mismatch: Q {tuple(qs)}, pages {tuple(ps)}")
    cache_lens = _ints(cache_lens, torch.int32, (B,), "cache_lens")
    if block_table.dim() != 2:
        raise ValueError(f"block_table must be [B, max_blocks], got {tuple(block_table.shape)}")
    max_blocks = block_table.shape[1]
    block_table = _ints(block_table, torch.int32, (B, max_blocks), "block_table")
    mask = (0, 0, 0, 0)
    if tree_mask is not None:
        if tree_mask.dtype != torch.bool:
            raise TypeError(f"tree_mask must be bool, got {tree_mask.dtype}")
        ms, st = tree_mask.shape, tree_mask.stride()
        if ms not in ((T, T), (B, T, T)):
            raise ValueError(f"tree_mask must be [{T}, {T}] or [{B}, {T}, {T}], got {tuple(ms)}")
        mask = (tree_mask.data_ptr(), *(st if len(st) == 3 else (0, *st)))
    if window is not None and window < 1:
        raise ValueError(f"window must be at least 1 (None: every row is seen), got {window}")
    scale = float(D ** -0.5 if scale is None else scale)
    out = _new(dtype, Q.device, B, Hq, T, D)
    if B == 0 or T == 0 or Hq == 0:
        return out
    # a workspace of the call's own, from the caching allocator: calls on several streams share nothing
    need = max(_attention_workspace(dev, B, Hq, Hkv, T, D, max_blocks * block), 1)
    ws = _new(torch.uint8, Q.device, need)
    pack, call = _lib.words("dropkv_attention_fp8")
    rc = call(pack(
        Q.data_ptr(), *Q.stride(), *pool, n_pages, block, block_table.data_ptr(), max_blocks, cache_lens.data_ptr(), *mask,
        min(int(window or 0), 0x7fffffff), min(int(sinks), 0x7fffffff), _DTYPE_CODE[dtype], B, Hq, Hkv, T, D, scale,
        out.data_ptr(), ws.data_ptr(), need, _raw_stream(dev)))
    if rc:
        _lib.check(rc, "dropkv_attention_fp8")
    if _CHECK_STATUS and n_pages * max_blocks > 0 and not torch.cuda.is_current_stream_capturing():
        n = torch.cuda.get_device_properties(dev).multi_processor_count * 2  # a word for each CTA comes first
        st = int(ws[:4 * n].view(torch.int32).max().item())
        if st != 0:
            raise _lib.DropKVError(_lib.ERR_DEVICE, f"dropkv_attention_fp8: device status {st} "
                                                    "(a bounded wait timed out)")
    return out

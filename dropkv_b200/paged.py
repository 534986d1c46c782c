"""A speculative decode step over paged, compressed caches (tensor functions over the C ABI).

``compress_varlen`` leaves a ragged batch whose kept lengths exist on the device only,
and decoding over it needs nothing of the host if the pages are handed out there too:

* ``block_tables``   -- pages and slots from lengths on the device, in one launch;
* ``store_rows``     -- K/V rows to slots (the eviction's outputs, accepted drafts);
* ``qk_norm_rope``   -- head norms, position rotation and the cache write in one pass;
* ``tree_attention`` -- a tree of drafted tokens over a cache in pages or row buffers;
* ``token_logprobs`` -- log probabilities of given tokens, entropy, top alternatives.

K and V pools are ``[pages, Hkv, block_size, D]``, any strides with contiguous rows (a
pool stored ``[pages, block_size, Hkv, D]`` is passed transposed); slot ``s`` is row
``s % block_size`` of page ``s // block_size``. No call synchronises the host. Between two steps
``block_tables`` wants its free list without the pages already taken, whose number is on the
device: a loop reads it back, or shifts the list there (see ``block_tables``). Nothing here takes
pages back. The reference keeps one tensor per layer (dropkv_cache.py:581-617) and has no
counterparts.
"""

from __future__ import annotations

import functools
from typing import NamedTuple, Optional

import torch

from . import _lib
from .ops import _CHECK_STATUS, _DTYPE_CODE

__all__ = ["BlockTables", "TokenLogprobs", "block_tables", "store_rows", "qk_norm_rope", "tree_attention",
           "token_logprobs", "tree_mask_from_parents"]


class BlockTables(NamedTuple):
    table: torch.Tensor   # [B, max_blocks] int32, -1 past a request's pages
    held: torch.Tensor    # [B] int32
    slots: torch.Tensor   # [B, max_new] int64, -1 past a request's new tokens
    used: torch.Tensor    # [1] int64: free pages asked for


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor                 # fp32, the shape of tokens
    entropy: torch.Tensor                 # fp32, the shape of the rows
    top_logprobs: Optional[torch.Tensor]  # fp32 [..., top_k], None for top_k = 0
    top_tokens: Optional[torch.Tensor]    # int64 [..., top_k]


# The current stream's handle by device index: the raw query skips making a Stream object, 2 us of
# a call whose kernel takes 3.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _new(dtype: torch.dtype, device: torch.device, *shape: int) -> torch.Tensor:
    """An uninitialised contiguous tensor (of up to four dimensions). empty_strided takes 1.5 us
    where empty takes 2.3 to 3."""
    n = len(shape)
    if n == 2:
        stride = (shape[1], 1)
    elif n == 1:
        stride = (1,)
    elif n == 4:
        stride = (shape[1] * shape[2] * shape[3], shape[2] * shape[3], shape[3], 1)
    elif n == 3:
        stride = (shape[1] * shape[2], shape[2], 1)
    else:
        return torch.empty(shape, dtype=dtype, device=device)
    return torch.empty_strided(shape, stride, dtype=dtype, device=device)


def _on_one_device(*ts) -> int:
    """The index of the CUDA device that holds every tensor (-1 stands for the CPU)."""
    index = ts[0].get_device()
    for t in ts:
        if t.get_device() != index or index < 0:
            cpu = [x.device for x in ts if not x.is_cuda]
            if cpu:
                raise RuntimeError("dropkv_b200 runs on CUDA tensors only (no CPU path); got a "
                                   f"tensor on {cpu[0]}")
            raise RuntimeError(f"all tensors must be on one device; got {ts[0].device} and {t.device}")
    return index


def _device_of_call(args, kwargs) -> int:
    """The index of the device of a call's first tensor, however the arguments are given; -1 if
    that is the CPU, or there is none."""
    for x in args:
        if isinstance(x, torch.Tensor):
            return x.get_device()
    for x in kwargs.values():
        if isinstance(x, torch.Tensor):
            return x.get_device()
    return -1


def _on_its_device(fn):
    """The call under its tensors' device, entered only where another one is current. (That
    all of them are on one is the call's to check.)"""
    @functools.wraps(fn)
    def call(*args, **kwargs):
        index = _device_of_call(args, kwargs)
        if index < 0 or index == _current_device():
            return fn(*args, **kwargs)
        with torch.cuda.device(index):
            return fn(*args, **kwargs)
    return call


def _ints(t: torch.Tensor, dtype: torch.dtype, shape: tuple, what: str) -> torch.Tensor:
    if t.dtype != dtype:
        raise TypeError(f"{what} must be {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{what} must have shape {shape}, got {tuple(t.shape)}")
    return t.contiguous()


def _rows_strides(t: torch.Tensor, what: str):
    """Strides of the three outer dimensions of [A, B, C, D] rows (the library takes the
    packed one for a dimension of one)."""
    s = t.stride()
    if s[3] != 1 and t.shape[3] > 1:
        raise ValueError(f"{what} needs rows of D contiguous elements")
    return s[:3]


def _check_pool(K_pages, V_pages, Hkv, D, dtype):
    shape = K_pages.shape
    if len(shape) != 4 or shape != V_pages.shape or shape[1] != Hkv or shape[3] != D:
        raise ValueError(f"expected K and V pages [pages, {Hkv}, block_size, {D}], got {tuple(K_pages.shape)} and "
                         f"{tuple(V_pages.shape)}")
    if K_pages.dtype != dtype or V_pages.dtype != dtype:
        raise TypeError(f"pages must be {dtype}, got {K_pages.dtype} and {V_pages.dtype}")
    return shape


def _norm_weight(w: torch.Tensor, D: int, dtype: torch.dtype, what: str) -> torch.Tensor:
    if w.shape != (D,) or w.dtype != dtype:
        raise ValueError(f"{what} must be [{D}] {dtype}, got {tuple(w.shape)} {w.dtype}")
    return w.contiguous()


@functools.lru_cache(maxsize=4096)
def _tree_workspace(index: int, B: int, Hq: int, Hkv: int, T: int, D: int, cap: int) -> int:
    """Bytes of a tree_attention workspace on the current device ``index``."""
    return int(_lib.load().dropkv_tree_attention_workspace_size(B, Hq, Hkv, T, D, cap))


@_on_its_device
def block_tables(lens: torch.Tensor, block_size: int, free_blocks: torch.Tensor, max_blocks: int, max_new: int,
                 new_lens: Optional[torch.Tensor] = None, table: Optional[torch.Tensor] = None,
                 held: Optional[torch.Tensor] = None) -> BlockTables:
    """Block tables and slot maps from request lengths on the device.

    ``lens`` [B] int32: tokens that each request's cache holds once this step is done;
    the last ``new_lens`` [B] int32 of them (all, if None) are new and get slots.
    ``table`` [B, max_blocks] int32 with ``held`` [B] int32 are the pages that the
    requests hold already; the missing ones are taken from ``free_blocks`` [F] int32
    in order, request after request. Returns new tensors (``BlockTables``); the
    caller drops the first ``used`` entries of its free list: by reading ``used`` back, or,
    where a step is captured in a CUDA graph, by shifting the list on the device
    (``torch.where(i + taken < F, free[(i + taken).clamp(max=F - 1)], -1)`` for
    ``i = arange(F)``). A request takes at most ``max_blocks`` pages; its tokens past them
    get no slots. Where the list runs short, entries and slots are -1, ``held`` counts the
    pages really held and ``used`` is more than F. (A page of -1 in the list counts as held,
    and gives slots of -1.)
    """
    if (table is None) != (held is None):
        raise ValueError("table and held go together")
    if lens.dim() != 1:
        raise ValueError(f"lens must be [B], got {tuple(lens.shape)}")
    B, F = lens.shape[0], free_blocks.numel()
    max_blocks, max_new = int(max_blocks), int(max_new)
    device = lens.device
    dev = _on_one_device(lens, free_blocks)
    lens = _ints(lens, torch.int32, (B,), "lens")
    free_blocks = _ints(free_blocks, torch.int32, (F,), "free_blocks")
    new_ptr = table_ptr = held_ptr = None
    if new_lens is not None:
        _on_one_device(lens, new_lens)
        new_lens = _ints(new_lens, torch.int32, (B,), "new_lens")
        new_ptr = new_lens.data_ptr()
    if table is not None:
        _on_one_device(lens, table, held)
        table = _ints(table, torch.int32, (B, max_blocks), "table")
        held = _ints(held, torch.int32, (B,), "held")
        table_ptr, held_ptr = table.data_ptr(), held.data_ptr()
    out = BlockTables(_new(torch.int32, device, B, max_blocks), _new(torch.int32, device, B),
                      _new(torch.int64, device, B, max_new), _new(torch.int64, device, 1))
    if B == 0:
        out.used.zero_()
        return out
    rc = _lib.load().dropkv_block_tables(
        lens.data_ptr(), new_ptr, table_ptr, max_blocks, held_ptr, B, int(block_size), free_blocks.data_ptr(), F,
        max_blocks, max_new, out.table.data_ptr(), out.held.data_ptr(), out.slots.data_ptr(), out.used.data_ptr(),
        _raw_stream(dev))
    if rc:
        _lib.check(rc, "dropkv_block_tables")
    return out


@_on_its_device
def store_rows(K: torch.Tensor, V: torch.Tensor, slots: torch.Tensor, K_pages: torch.Tensor,
               V_pages: torch.Tensor) -> None:
    """Rows of K and V [B, Hkv, N, D] (any strides, rows of D contiguous) to slots [B, N]
    (int64) of the pools, in place; rows whose slot is outside the pool (-1) are left
    out. Rows go in no order: those that share a slot leave a mixture of them there, and
    K and V must not lie where rows are written, such as in the same pages (move rows
    within a pool by way of a copy). fp32, fp16 or bf16."""
    dev = _on_one_device(K, V, slots, K_pages, V_pages)
    ks, dtype = K.shape, K.dtype
    if len(ks) != 4 or ks != V.shape:
        raise ValueError("expected K, V [B, Hkv, N, D] of one shape")
    if dtype not in _DTYPE_CODE or V.dtype != dtype:
        raise TypeError(f"K and V must share one of fp32/fp16/bf16; got {dtype}, {V.dtype}")
    B, Hkv, N, D = ks
    ps = _check_pool(K_pages, V_pages, Hkv, D, dtype)
    slots = _ints(slots, torch.int64, (B, N), "slots")
    rc = _lib.load().dropkv_store_rows(
        K.data_ptr(), *_rows_strides(K, "K"), V.data_ptr(), *_rows_strides(V, "V"), slots.data_ptr(),
        K_pages.data_ptr(), *_rows_strides(K_pages, "K_pages"), V_pages.data_ptr(),
        *_rows_strides(V_pages, "V_pages"), ps[0], ps[2], K.element_size(), B, Hkv, N, D,
        _raw_stream(dev))
    if rc:
        _lib.check(rc, "dropkv_store_rows")


@_on_its_device
def qk_norm_rope(Q: torch.Tensor, K: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor,
                 q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                 interleaved: bool = False, V: Optional[torch.Tensor] = None, slots: Optional[torch.Tensor] = None,
                 K_pages: Optional[torch.Tensor] = None, V_pages: Optional[torch.Tensor] = None):
    """(Q_out, K_out): the heads of Q [B, Hq, L, D] and K [B, Hkv, L, D] (any strides,
    rows of D contiguous) normed and rotated, contiguous and in the input dtype.

    ``q_weight`` / ``k_weight`` [D]: RMS norm over each head with ``eps`` and that weight
    (None: no norm). ``cos`` / ``sin`` [P, R / 2] fp32: the first R elements of a head
    turn by row ``positions`` ([B, L] or [L], int64) of them, in pairs (i, i + R / 2), or
    (2i, 2i + 1) if ``interleaved``; a position outside [0, P) gives NaN. After an
    eviction positions go on from the tokens seen, not from the rows stored, and a drafted
    node's position is its depth's. With ``V``, ``slots`` [B, L], ``K_pages`` and
    ``V_pages`` the finished K rows and V's also go to the pool, as ``store_rows`` puts
    them. fp32, fp16 or bf16; sums in fp32, rounded once.
    """
    given = (V is not None) + (slots is not None) + (K_pages is not None) + (V_pages is not None)
    if given not in (0, 4):
        raise ValueError("V, slots, K_pages and V_pages go together")
    cache = (V, slots, K_pages, V_pages) if given else ()
    dev = _on_one_device(Q, K, cos, sin, positions, *cache)
    for w in (q_weight, k_weight):
        if w is not None:
            _on_one_device(Q, w)
    qs, ks, cs = Q.shape, K.shape, cos.shape  # (once each: a shape takes 0.3 us to make)
    if len(qs) != 4 or len(ks) != 4 or qs[0] != ks[0] or qs[2] != ks[2] or qs[3] != ks[3]:
        raise ValueError(f"expected Q [B,Hq,L,D] and K [B,Hkv,L,D], got {tuple(qs)} and {tuple(ks)}")
    dtype = Q.dtype
    dt = _DTYPE_CODE.get(dtype)
    if dt is None or K.dtype != dtype:
        raise TypeError(f"Q and K must share one of fp32/fp16/bf16; got {dtype}, {K.dtype}")
    B, Hq, L, D = qs
    Hkv = ks[1]
    if len(cs) != 2 or cs != sin.shape:
        raise ValueError(f"cos and sin must be [P, R / 2] of one shape, got {tuple(cs)} and {tuple(sin.shape)}")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise TypeError("cos and sin must be float32")
    cos, sin = cos.contiguous(), sin.contiguous()
    if positions.dim() == 1:
        positions, pos_sb = _ints(positions, torch.int64, (L,), "positions"), 0
    else:
        positions, pos_sb = _ints(positions, torch.int64, (B, L), "positions"), L
    qw_ptr = kw_ptr = None
    if q_weight is not None:
        q_weight = _norm_weight(q_weight, D, dtype, "q_weight")
        qw_ptr = q_weight.data_ptr()
    if k_weight is not None:
        k_weight = _norm_weight(k_weight, D, dtype, "k_weight")
        kw_ptr = k_weight.data_ptr()
    if cache:
        if V.shape != ks or V.dtype != dtype:
            raise ValueError(f"V must be {tuple(ks)} {dtype}, got {tuple(V.shape)} {V.dtype}")
        ps = _check_pool(K_pages, V_pages, Hkv, D, dtype)
        slots = _ints(slots, torch.int64, (B, L), "slots")
        tail = (V.data_ptr(), *_rows_strides(V, "V"), slots.data_ptr(), K_pages.data_ptr(),
                *_rows_strides(K_pages, "K_pages"), V_pages.data_ptr(), *_rows_strides(V_pages, "V_pages"),
                ps[0], ps[2])
    else:
        tail = (None, 0, 0, 0, None, None, 0, 0, 0, None, 0, 0, 0, 0, 1)
    device = Q.device
    q_out = _new(dtype, device, B, Hq, L, D)
    k_out = _new(dtype, device, B, Hkv, L, D)
    rc = _lib.load().dropkv_qk_norm_rope(
        Q.data_ptr(), *_rows_strides(Q, "Q"), K.data_ptr(), *_rows_strides(K, "K"),
        qw_ptr, kw_ptr, float(eps), cos.data_ptr(), sin.data_ptr(), cs[0], 2 * cs[1], int(bool(interleaved)),
        positions.data_ptr(), pos_sb, dt, B, Hq, Hkv, L, D, q_out.data_ptr(), k_out.data_ptr(), *tail, _raw_stream(dev))
    if rc:
        _lib.check(rc, "dropkv_qk_norm_rope")
    return q_out, k_out


def tree_mask_from_parents(parents: torch.Tensor):
    """(mask, depth) of draft trees given by parents [..., T] (the index of a node's
    parent, below its own; -1 for a child of the last cached token): mask
    [..., T, T] bool shows each node its ancestors and itself, depth [..., T] int64
    counts its ancestors (its position after the last cached token's). On the
    parents' device, without synchronising."""
    T = parents.shape[-1]
    node = torch.arange(T, device=parents.device)
    mask = (parents.unsqueeze(-1) == node) | torch.eye(T, dtype=torch.bool, device=parents.device)
    n = 1
    while n < T:  # nodes within n steps up, doubled (counts stay exact: at most T)
        mask = (mask.float() @ mask.float()) > 0
        n *= 2
    return mask, mask.sum(-1) - 1


@_on_its_device
def tree_attention(Q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, cache_lens: torch.Tensor,
                   tree_mask: Optional[torch.Tensor] = None, block_table: Optional[torch.Tensor] = None,
                   scale: Optional[float] = None) -> torch.Tensor:
    """Attention of a tree of T drafted tokens over a cache: Q [B, Hq, T, D] (any
    strides) -> [B, Hq, T, D].

    Row b's cache holds ``cache_lens[b]`` (int32, on the device) rows, and after them the
    tree's own K/V rows in node order. Node i sees every cached row and the nodes j with
    ``tree_mask[i, j]`` (bool [T, T] or [B, T, T]; None: j <= i, a chain). K and V are
    row buffers [B, Hkv, cap, D] or, with ``block_table`` ([B, max_blocks] int32), pools
    [pages, Hkv, block_size, D]; any strides with contiguous rows on 16-byte boundaries that
    do not overlap (no broadcast heads or sequences).
    Rows past the capacity are not seen, nor are those on missing pages (-1); a node that
    sees nothing gives zeros; what is in rows that no node sees does not matter. bf16 or
    fp16, D 64 or 128, T <= 256, block_size a power of two from 8 to 1024. Products of 16
    bits, sums and softmax statistics in fp32.
    """
    dev = _on_one_device(Q, K, V, cache_lens, *[t for t in (tree_mask, block_table) if t is not None])
    qs, ks, dtype = Q.shape, K.shape, Q.dtype
    if len(qs) != 4 or len(ks) != 4 or ks != V.shape:
        raise ValueError("expected Q [B,Hq,T,D] and K, V [B,Hkv,cap,D] or [pages,Hkv,block_size,D] of one shape")
    if not (dtype == K.dtype == V.dtype) or dtype not in (torch.bfloat16, torch.float16):
        raise TypeError("tree attention takes bf16 or fp16 Q, K and V of one dtype")
    B, Hq, T, D = qs
    n0, Hkv, rows, Dk = ks
    if Dk != D or not Hkv or Hq % Hkv or (block_table is None and n0 != B):
        raise ValueError(f"shape mismatch: Q {tuple(qs)}, K {tuple(ks)}")
    cache_lens = _ints(cache_lens, torch.int32, (B,), "cache_lens")
    if block_table is not None:
        if block_table.dim() != 2:
            raise ValueError(f"block_table must be [B, max_blocks], got {tuple(block_table.shape)}")
        max_blocks = block_table.shape[1]
        block_table = _ints(block_table, torch.int32, (B, max_blocks), "block_table")
        paging = (block_table.data_ptr(), max_blocks, rows, n0)
        cap = max_blocks * rows
    else:
        paging = (None, 0, 0, 0)
        cap = rows
    mask = (None, 0, 0, 0)
    if tree_mask is not None:
        if tree_mask.dtype != torch.bool:
            raise TypeError(f"tree_mask must be bool, got {tree_mask.dtype}")
        ms, st = tree_mask.shape, tree_mask.stride()
        if ms not in ((T, T), (B, T, T)):
            raise ValueError(f"tree_mask must be [{T}, {T}] or [{B}, {T}, {T}], got {tuple(ms)}")
        mask = (tree_mask.data_ptr(), *(st if len(st) == 3 else (0, *st)))
    scale = float(D ** -0.5 if scale is None else scale)
    lib = _lib.load()
    device = Q.device
    out = _new(dtype, device, B, Hq, T, D)
    if B == 0 or T == 0:
        return out
    # a workspace of the call's own, from the caching allocator: calls on several streams share nothing
    need = max(_tree_workspace(dev, B, Hq, Hkv, T, D, cap), 1)
    ws = _new(torch.uint8, device, need)
    rc = lib.dropkv_tree_attention(
        Q.data_ptr(), *Q.stride(), K.data_ptr(), *_rows_strides(K, "K"), V.data_ptr(), *_rows_strides(V, "V"),
        *paging, cache_lens.data_ptr(), *mask, _DTYPE_CODE[dtype], B, Hq, Hkv, T, D, cap, scale,
        out.data_ptr(), ws.data_ptr(), need, _raw_stream(dev))
    if rc:
        _lib.check(rc, "dropkv_tree_attention")
    if _CHECK_STATUS and cap * n0 > 0 and not torch.cuda.is_current_stream_capturing():
        n = torch.cuda.get_device_properties(dev).multi_processor_count  # a word for each CTA comes first
        st = int(ws[:4 * n].view(torch.int32).max().item()) if need >= 4 * n else 0
        if st != 0:
            raise _lib.DropKVError(_lib.ERR_DEVICE, f"dropkv_tree_attention: device status {st} "
                                                    "(a bounded wait timed out)")
    return out


@_on_its_device
def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top_k: int = 0,
                   temperature: float = 1.0) -> TokenLogprobs:
    """Under softmax(logits / temperature) for rows of logits [..., V] (fp32, fp16 or
    bf16): log probabilities of ``tokens`` (int64, [...] or [..., C]; -inf for one outside
    [0, V), such as a draft tree's padding), the entropy of each row, and its ``top_k``
    (at most 64) likeliest tokens, best first, ties to the lower index. fp32 sums and
    results. A row that holds NaN or +inf, or nothing but -inf, gives NaN. Rows of
    contiguous logits at one stride are read where they are; where the leading dimensions
    do not merge into one (``logits[:, :-1]`` of a batch of several) the logits are copied
    first, which costs more than the call: pass a sequence at a time, or all positions."""
    dev = _on_one_device(logits, tokens)
    dt = _DTYPE_CODE.get(logits.dtype)
    if dt is None:
        raise TypeError(f"logits must be fp32/fp16/bf16; got {logits.dtype}")
    if tokens.dtype != torch.int64:
        raise TypeError(f"tokens must be int64, got {tokens.dtype}")
    ls, ts = tuple(logits.shape), tuple(tokens.shape)
    lead = ls[:-1]
    if not ls or len(ts) - len(ls) not in (-1, 0) or ts[:len(lead)] != lead:
        raise ValueError(f"expected logits [..., V] and tokens [...] or [..., C], got {ls} and {ts}")
    V, device = ls[-1], logits.device
    rows = logits if len(ls) == 2 else logits.reshape(-1, V)
    if V > 1 and rows.stride(1) != 1:
        rows = rows.contiguous()
    N, top_k = rows.shape[0], int(top_k)
    C = ts[-1] if len(ts) == len(ls) else 1
    tokens = tokens.contiguous()
    logprob = _new(torch.float32, device, *ts)
    entropy = _new(torch.float32, device, *lead)
    top_lp = top_id = None
    if top_k > 0:
        top_lp = _new(torch.float32, device, *lead, top_k)
        top_id = _new(torch.int64, device, *lead, top_k)
    lib = _lib.load()
    rc = lib.dropkv_token_logprobs(rows.data_ptr(), rows.stride(0), dt, N, V, tokens.data_ptr(), C, top_k,
                                   float(temperature), logprob.data_ptr(), entropy.data_ptr(),
                                   top_lp.data_ptr() if top_k > 0 else None, top_id.data_ptr() if top_k > 0 else None,
                                   None, 0, _raw_stream(dev))  # (no workspace is needed)
    if rc:
        _lib.check(rc, "dropkv_token_logprobs")
    return TokenLogprobs(logprob, entropy, top_lp, top_id)

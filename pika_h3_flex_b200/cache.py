"""Paged K/V cache and the attention that reads it: ``cache_write``, ``cache_read`` and ``cache_attn`` over the C ABI.

For callers whose K and V of some tokens stay the same between calls: a model that looks at fixed states by cross attention
at every evaluation of a sampler, a clip that grows by a few frames at a time whose past does not change, a prompt model.
(The reference runs one joint sequence through the model at every evaluation, ``src/pika_h3/core/sampling.py:87-109,160-169``;
text is part of it, so its K and V change from block to block and evaluation to evaluation and are nothing to keep.)

    cache = KVCache.empty(n_pages, page_size, kv_heads, quantised=True)
    batch = CacheBatch(pages, lengths, starts)      # lengths include the new tokens
    cache_write(cache, batch, k, v)                 # k after qk_prep: normalised and rotated
    out = cache_attn(q, cache, batch)               # causal: token p sees the keys 0 .. p

Packed tensors have logical shape ``[rows, heads, 128]`` like everywhere in the package; rows ``starts[b]`` to
``starts[b + 1] - 1`` are the LAST tokens of sequence b, which holds ``lengths[b]`` tokens.
"""
from __future__ import annotations

import ctypes as C
from functools import lru_cache
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import check
from .ops import HEAD_DIM, _require_cuda

PAGE_MULTIPLE = 16


def _stride(t: torch.Tensor, dim: int) -> int:
    """Stride of a dimension in elements; a dimension of one entry is never stepped over and may say anything."""
    return t.stride(dim) if t.shape[dim] > 1 else HEAD_DIM


class KVCache:
    """Pages of cached rows of one attention layer.  ``k``, ``v``: logical ``[n_pages, page_size, heads, 128]`` with any
    page / token / head strides, bf16, or for a quantised cache e4m3 (``torch.float8_e4m3fn`` or ``uint8`` bytes) with
    ``k_exp``, ``v_exp`` ``[n_pages, page_size, heads]`` uint8: a code stands for ``code * 2 ** (exp - 127)``.  Expanded
    exponents (stride 0) can be read, not written."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_exp: Optional[torch.Tensor] = None, v_exp: Optional[torch.Tensor] = None):
        _require_cuda(k, v, k_exp, v_exp)
        self.quantised = k_exp is not None
        dtypes = (torch.float8_e4m3fn, torch.uint8) if self.quantised else (torch.bfloat16,)
        if (k_exp is None) != (v_exp is None):
            raise ValueError("k_exp and v_exp go together")
        for name, t in (("k", k), ("v", v)):
            if t.dim() != 4 or t.shape[3] != HEAD_DIM or t.stride(3) != 1 or t.shape != k.shape or 0 in t.shape:
                raise ValueError(f"{name}: expected logical [n_pages, page_size, heads, 128] with a contiguous last dim, got {tuple(t.shape)} / {t.stride()}")
            if t.dtype not in dtypes:
                raise TypeError(f"{name}: dtype {t.dtype} not in {dtypes}")
        for name, t in (("k_exp", k_exp), ("v_exp", v_exp)):
            if t is not None and (t.dtype != torch.uint8 or t.shape != k.shape[:3]):
                raise ValueError(f"{name} must be uint8 [n_pages, page_size, heads]")
        if any(t is not None and t.device != k.device for t in (v, k_exp, v_exp)):
            raise ValueError("the cache's tensors are on different devices")
        if k.shape[1] % PAGE_MULTIPLE:
            raise ValueError(f"the page size must be a multiple of {PAGE_MULTIPLE}")
        self.k, self.v, self.k_exp, self.v_exp = k, v, k_exp, v_exp
        self.n_pages, self.page_size, self.heads = (int(x) for x in k.shape[:3])
        self.device = k.device
        c = self._c = _lib.Cache()
        self._ref = C.byref(c)
        c.n_pages, c.page_size, c.heads, c.d, c.quantised = self.n_pages, self.page_size, self.heads, HEAD_DIM, int(self.quantised)
        for name, t in (("k", k), ("v", v), ("k_exp", k_exp), ("v_exp", v_exp)):
            if t is not None:
                setattr(c, name, t.data_ptr())
                for dim, what in enumerate(("page", "token", "head")):
                    setattr(c, f"{name}_stride_{what}", _stride(t, dim))

    @staticmethod
    def empty(n_pages: int, page_size: int, heads: int, quantised: bool = False, device=None) -> "KVCache":
        """A cache with its own memory, a head's rows of a page next to each other.  The rows hold nothing yet."""
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else device
        dtype = torch.float8_e4m3fn if quantised else torch.bfloat16
        pools = [torch.empty(n_pages, heads, page_size, HEAD_DIM, dtype=dtype, device=device).transpose(1, 2) for _ in range(2)]
        exps = [torch.empty(n_pages, heads, page_size, dtype=torch.uint8, device=device).transpose(1, 2) if quantised else None for _ in range(2)]
        return KVCache(*pools, *exps)


class CacheBatch:
    """Which tokens a call is about: ``pages [B, max_pages]``, ``lengths [B]`` and ``starts [B + 1]``, int32 on the device.
    They are read when a kernel runs, so they may be updated in place between the replays of a captured graph."""

    def __init__(self, pages: torch.Tensor, lengths: torch.Tensor, starts: torch.Tensor):
        _require_cuda(pages, lengths, starts)
        if any(t.dtype != torch.int32 for t in (pages, lengths, starts)):
            raise TypeError("pages, lengths and starts must be int32")
        n = lengths.shape[0] if lengths.dim() == 1 else -1
        if n < 1 or pages.dim() != 2 or pages.shape[0] != n or pages.shape[1] < 1 or tuple(starts.shape) != (n + 1,):
            raise ValueError("expected pages [B, max_pages], lengths [B] and starts [B + 1]")
        if (pages.shape[1] > 1 and pages.stride(1) != 1) or starts.stride(0) != 1 or (n > 1 and lengths.stride(0) != 1):
            raise ValueError("pages must have contiguous rows, lengths and starts must be contiguous")
        if pages.device != lengths.device or pages.device != starts.device:
            raise ValueError("pages, lengths and starts are on different devices")
        self.pages, self.lengths, self.starts = pages, lengths, starts
        self.device = pages.device
        c = self._c = _lib.CacheBatch()
        c.pages, c.lengths, c.starts = pages.data_ptr(), lengths.data_ptr(), starts.data_ptr()
        c.pages_stride = pages.stride(0) if n > 1 else pages.shape[1]
        c.n_seqs, c.max_pages = n, pages.shape[1]
        self._by_rows = {}

    def _for(self, rows: int):
        """The C description of this batch for packed tensors of so many rows."""
        ref = self._by_rows.get(rows)
        if ref is None:
            c = _lib.CacheBatch.from_buffer_copy(self._c)
            c.rows = rows
            if len(self._by_rows) >= 64:
                self._by_rows.clear()
            ref = self._by_rows[rows] = C.byref(c)  # holds on to c
        return ref


def _call(name: str, device: torch.device, *args) -> None:
    """A C call on the tensors' device and its current stream, whichever device is current."""
    fn = getattr(_lib.load(), name)
    if torch.cuda.current_device() == device.index:
        check(fn(*args, _stream(device)), name)
    else:
        with torch.cuda.device(device):
            check(fn(*args, _stream(device)), name)


def _stream(device: torch.device) -> int:
    """The current stream of a device as CUDA knows it.  (``torch.cuda.current_stream`` builds a Python object around it
    first: 2.2 us of a call that takes 8.)"""
    return torch._C._cuda_getCurrentRawStream(device.index)


def _rows(t: torch.Tensor, name: str, heads: int, device: torch.device) -> Tuple[int, int, int]:
    """Rows and the two strides of a packed [rows, heads, 128] bf16 tensor (these calls are made for single tokens too,
    so the checks are few and cheap)."""
    if t.device != device:
        _require_cuda(t)
        raise ValueError(f"expected everything on {device}, got {name} on {t.device}")
    shape, stride = t.shape, t.stride()
    if len(shape) != 3 or shape[2] != HEAD_DIM or stride[2] != 1:
        raise ValueError(f"{name}: expected logical [rows, heads, 128] with a contiguous last dim, got {tuple(shape)} / {stride}")
    if t.dtype != torch.bfloat16:
        raise TypeError(f"{name}: dtype {t.dtype} is not bfloat16")
    if shape[1] != heads:
        raise ValueError(f"{name} has {shape[1]} heads, expected {heads}")
    return shape[0], stride[0] if shape[0] > 1 else HEAD_DIM, stride[1] if heads > 1 else HEAD_DIM


def _status_ptr(status_word: Optional[torch.Tensor], device: torch.device) -> Optional[int]:
    if status_word is None:
        return None
    if status_word.dtype != torch.int32 or status_word.device != device:
        raise ValueError(f"status_word must be an int32 tensor on {device}")
    return status_word.data_ptr()


def _check_workspace(workspace: torch.Tensor, device: torch.device) -> None:
    if workspace.device != device:
        raise ValueError(f"expected everything on {device}, got the workspace on {workspace.device}")
    if not workspace.is_contiguous():  # its bytes are counted, and an expanded tensor has fewer than that
        raise ValueError("the workspace must be contiguous")


def _move(name: str, cache: KVCache, batch: CacheBatch, k: torch.Tensor, v: torch.Tensor, status_word: Optional[torch.Tensor]) -> None:
    device = cache.device
    L, ksl, ksh = _rows(k, "k", cache.heads, device)
    Lv, vsl, vsh = _rows(v, "v", cache.heads, device)
    if L != Lv:
        raise ValueError("k and v disagree on the number of rows")
    if batch.device != device:
        raise ValueError(f"expected everything on {device}, got the batch on {batch.device}")
    status = _status_ptr(status_word, device)
    if L == 0:
        return
    _call(name, device, cache._ref, batch._for(L), k.data_ptr(), ksl, ksh, v.data_ptr(), vsl, vsh, status)


def cache_write(cache: KVCache, batch: CacheBatch, k: torch.Tensor, v: torch.Tensor, status_word: Optional[torch.Tensor] = None) -> None:
    """Put the batch's rows ``k``, ``v`` ``[rows, heads, 128]`` bf16 into the cache, quantised if it is (per row: the
    smallest power of two that brings the largest magnitude to at most 448, then e4m3).  A page that is written to must
    belong to one sequence only; pages that are only read may be shared."""
    _move("h3a_cache_write", cache, batch, k, v, status_word)


def cache_read(cache: KVCache, batch: CacheBatch, rows: Optional[int] = None, out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
               status_word: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The batch's rows as bf16 ``(k, v)`` ``[rows, heads, 128]``: of each sequence its last ``starts[b + 1] - starts[b]``
    tokens (all of them where that is ``lengths[b]``).  ``rows``: how many rows the packed tensors have (``starts[B]`` on
    the host); or ``out``, two tensors to fill, whose rows outside every sequence stay as they are."""
    if (rows is None) == (out is None):
        raise ValueError("pass either rows or out")
    if out is None:
        if rows < 0:
            raise ValueError("rows must not be negative")
        out = torch.empty(2, rows, cache.heads, HEAD_DIM, dtype=torch.bfloat16, device=cache.device).unbind()
    k, v = out
    _move("h3a_cache_read", cache, batch, k, v, status_word)
    return k, v


@lru_cache(maxsize=256)
def _workspace_bytes(device_index: int, rows: int, n_seqs: int, heads: int, kv_heads: int, quantised: bool, max_new: int) -> int:
    p = _lib.CacheAttnParams()
    p.cache.heads, p.cache.quantised, p.batch.rows, p.batch.n_seqs, p.heads, p.max_new = kv_heads, int(quantised), rows, n_seqs, heads, max_new
    need = C.c_size_t(0)
    with torch.cuda.device(device_index):
        check(_lib.load().h3a_cache_attn_workspace_bytes(C.byref(p), C.byref(need)), "h3a_cache_attn_workspace_bytes")
    return int(need.value)


def cache_attn_workspace_bytes(cache: KVCache, batch: CacheBatch, rows: int, heads: int, max_new: Optional[int] = None) -> int:
    """Bytes of device scratch a ``cache_attn`` call of this shape needs; callers in a loop can allocate it once (32-byte
    aligned; one per stream: calls that may run at the same time must not share it)."""
    return _workspace_bytes(cache.device.index, int(rows), batch._c.n_seqs, int(heads), cache.heads, cache.quantised, int(max_new or 0))


def cache_attn(q: torch.Tensor, cache: KVCache, batch: CacheBatch, causal: bool = True, softmax_scale: float = 0.0,
               out: Optional[torch.Tensor] = None, return_lse: bool = False, status_word: Optional[torch.Tensor] = None,
               workspace: Optional[torch.Tensor] = None, wait_limit_ns: int = 0, max_new: Optional[int] = None):
    """Attention of the batch's rows ``q [rows, heads, 128]`` bf16 over their sequences' cached keys; ``heads`` is a
    multiple of the cache's (query head h reads K/V head ``h // (heads // cache.heads)``).  ``causal``: row i of a sequence
    is the token at position ``lengths[b] - n_b + i`` and sees the keys up to itself (write its K and V first); otherwise
    every row sees all ``lengths[b]`` keys.  A row without a key is zeros (lse -inf).  Returns ``out [rows, heads, 128]``
    bf16 (and ``lse [heads, rows]``); rows outside every sequence are not written; ``out`` must not overlap ``q``.  ``softmax_scale`` 0: ``1/sqrt(128)``.
    ``max_new``, the most rows any one sequence has, only chooses the kernel, which otherwise goes by the average: worth
    saying for a batch that mixes single tokens with long chunks."""
    _require_cuda(q)
    device = cache.device
    H = q.shape[1] if q.dim() == 3 else 0
    L, qsl, qsh = _rows(q, "q", H, device)
    if H == 0 or H % cache.heads:
        raise ValueError(f"q has {H} heads: not a multiple of the cache's {cache.heads}")
    if batch.device != device:
        raise ValueError(f"expected everything on {device}, got the batch on {batch.device}")
    if out is None:
        out = torch.empty(L, H, HEAD_DIM, dtype=torch.bfloat16, device=device)
        osl, osh = H * HEAD_DIM, HEAD_DIM
    else:
        Lo, osl, osh = _rows(out, "out", H, device)
        if Lo != L:
            raise ValueError("out must have q's shape")
    status = _status_ptr(status_word, device)
    lse = torch.empty(H, L, dtype=torch.float32, device=device) if return_lse else None
    if L == 0:
        return (out, lse) if return_lse else out
    if workspace is None:
        workspace = torch.empty(_workspace_bytes(device.index, L, batch._c.n_seqs, H, cache.heads, cache.quantised, max_new or 0), dtype=torch.uint8, device=device)
    else:
        _check_workspace(workspace, device)
    p = _lib.CacheAttnParams(cache._c, batch._c, q.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else None, qsl, qsh, osl, osh,
                             H, 1 if causal else 0, softmax_scale, max_new or 0, workspace.data_ptr(), workspace.nbytes, status, wait_limit_ns)
    p.batch.rows = L
    _call("h3a_cache_attn", device, C.byref(p))
    return (out, lse) if return_lse else out

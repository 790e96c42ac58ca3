"""A paged cache of keys and values in 8 bits, and attention over it: pages of T tokens, e4m3 with one exponent for the block
of each page and head (``dsb_kv_cache`` in include/dsb.h says what a block stands for).  Sequences are rows of a page table;
who owns which page is the caller's business."""
import ctypes
import math

import torch

from . import _lib, ops
from ._lib import check
from .ops import _ptr, _require_cuda, _stream, status_word

HEAD_DIM = 128
PAGE_TOKENS = (16, 32, 64, 128)


class PagedKVCache:
    """``k``, ``v``: float8_e4m3fn ``[pages, heads, T, 128]``; ``k_exp``, ``v_exp``: int8 ``[pages, heads]``, the power of two
    that a block's values are multiplied by.  A page needs no preparation: the append that writes its first token sets its
    exponent."""

    def __init__(self, k, v, k_exp, v_exp):
        for t in (k, v):
            if t.dtype != torch.float8_e4m3fn or t.dim() != 4 or t.shape != k.shape or t.shape[3] != HEAD_DIM or not t.is_contiguous():
                raise _lib.DsbError("PagedKVCache k and v are contiguous float8_e4m3fn [pages, heads, T, 128] tensors of one shape")
        if k.shape[2] not in PAGE_TOKENS:
            raise _lib.DsbError(f"PagedKVCache pages hold {PAGE_TOKENS} tokens, got {k.shape[2]}")
        for t in (k_exp, v_exp):
            if t.dtype != torch.int8 or t.shape != k.shape[:2] or not t.is_contiguous():
                raise _lib.DsbError("PagedKVCache k_exp and v_exp are contiguous int8 [pages, heads] tensors")
        if k.numel() == 0 or k.numel() // HEAD_DIM > 0x7fffffff:
            raise _lib.DsbError("PagedKVCache: pages x heads x T must be between 1 and 2^31 - 1")
        if len({t.device for t in (k, v, k_exp, v_exp)}) != 1:
            raise _lib.DsbError("PagedKVCache: all four tensors live on one device")
        if k.is_cuda and any(t.data_ptr() % 128 for t in (k, v)):
            raise _lib.DsbError("PagedKVCache k and v are 128-byte aligned")
        self._t = (k, v, k_exp, v_exp)
        self._args = _lib.KVCacheArgs(k.data_ptr(), v.data_ptr(), k_exp.data_ptr(), v_exp.data_ptr(), *k.shape[:3])
        self._ref = ctypes.byref(self._args)

    @classmethod
    def empty(cls, pages: int, heads: int, page_tokens: int = 64, device="cuda") -> "PagedKVCache":
        k, v = (torch.empty((pages, heads, page_tokens, HEAD_DIM), dtype=torch.float8_e4m3fn, device=device) for _ in range(2))
        return cls(k, v, *(torch.zeros((pages, heads), dtype=torch.int8, device=device) for _ in range(2)))

    # the kernels hold these tensors' addresses, so they cannot be replaced
    k = property(lambda self: self._t[0])
    v = property(lambda self: self._t[1])
    k_exp = property(lambda self: self._t[2])
    v_exp = property(lambda self: self._t[3])
    pages = property(lambda self: self._args.n_pages)
    heads = property(lambda self: self._args.heads)
    page_tokens = property(lambda self: self._args.page_tokens)

    def pages_for(self, tokens: int) -> int:
        """Table entries that a sequence of ``tokens`` needs."""
        return -(-tokens // self.page_tokens)


def _table(table, B):
    if table.dtype != torch.int32 or table.dim() != 2 or table.shape[0] != B or table.shape[1] == 0 or table.stride(1) != 1 \
            or (B > 1 and table.stride(0) < table.shape[1]):
        raise _lib.DsbError(f"the page table is an int32 [{B}, pages] tensor with contiguous rows")
    return max(table.stride(0), table.shape[1]), table.shape[1]


def _per_sequence(t, B, what):
    if t.dtype != torch.int32 or tuple(t.shape) != (B,) or not t.is_contiguous():
        raise _lib.DsbError(f"{what} is an int or a contiguous int32 [{B}] tensor")


def _rows4(t, what):
    if t.dim() != 4 or t.shape[3] != HEAD_DIM or t.dtype != torch.bfloat16 or t.stride(3) != 1 or t.data_ptr() % 16 \
            or any(s % 8 or s < 0 for s in t.stride()[:3]):
        raise _lib.DsbError(f"{what} is a bf16 [B, tokens, heads, 128] tensor with a contiguous head dimension, 16-byte aligned, "
                            "with strides that are multiples of 8")


def append(cache: PagedKVCache, k, v, table, start, counts=None, rope=None, rope_row0: int = 0):
    """Appends ``k`` and ``v`` (bf16 ``[B, n, heads, 128]``, any strides that are multiples of 8) to the sequences of ``table``
    (int32 ``[B, pages]``), from position ``start`` (int, or int32 ``[B]``) on; ``counts`` (int32 ``[B]``): how many of the n rows
    belong to each sequence.  ``rope`` (fp32 ``[rows, 64, 2]`` = cos, sin): ``k`` is rotated by row ``rope_row0 + position``.
    A position or page outside its table leaves that part unwritten and raises at the next ``ops.check_status``."""
    B, n = k.shape[0], k.shape[1]
    dev_start = start if isinstance(start, torch.Tensor) else None
    _require_cuda(cache.k, k, v, table, dev_start, counts, rope)
    _rows4(k, "k")
    _rows4(v, "v")
    if v.shape != k.shape or k.shape[2] != cache.heads:
        raise _lib.DsbError(f"k and v are [B, n, {cache.heads}, 128] rows of one shape")
    ld, width = _table(table, B)
    if dev_start is not None:
        _per_sequence(dev_start, B, "start")
    elif not 0 <= start <= width * cache.page_tokens - (n if counts is None else 0):
        raise _lib.DsbError(f"{n} rows from position {start} on do not fit a table of {width} pages")
    if counts is not None:
        _per_sequence(counts, B, "counts")
    if rope is not None:
        if rope.dtype != torch.float32 or rope.dim() != 3 or tuple(rope.shape[1:]) != (64, 2) or not rope.is_contiguous():
            raise _lib.DsbError("rope is a contiguous float32 [rows, 64, 2] table")
        if rope.data_ptr() % 16 or not -(1 << 31) <= rope_row0 < 1 << 31:
            raise _lib.DsbError("rope is 16-byte aligned and rope_row0 a 32-bit number")
    rc = _lib.lib().dsb_kv_append(
        cache._ref, _ptr(k), k.stride(0), k.stride(1), k.stride(2), _ptr(v), v.stride(0), v.stride(1), v.stride(2), B, n,
        _ptr(table), ld, width, _ptr(dev_start), 0 if dev_start is not None else start, _ptr(counts), _ptr(rope),
        0 if rope is None else rope.shape[0], rope_row0, _ptr(status_word(k.device)), _stream())
    check(rc, "dsb_kv_append")


def read(cache: PagedKVCache, table, n: int, first: int = 0):
    """Tokens ``first .. first + n - 1`` of each sequence as bf16 ``(k, v)``, each ``[B, n, heads, 128]`` (exact)."""
    _require_cuda(cache.k, table)
    B = table.shape[0]
    ld, width = _table(table, B)
    if n < 0 or first < 0 or first + n > width * cache.page_tokens:
        raise _lib.DsbError(f"tokens {first}..{first + n - 1} are not in a table of {width} pages")
    k, v = (torch.empty((B, n, cache.heads, HEAD_DIM), dtype=torch.bfloat16, device=table.device) for _ in range(2))
    rc = _lib.lib().dsb_kv_read(cache._ref, _ptr(table), ld, width, B, first, n, _ptr(k), k.stride(0), k.stride(1), k.stride(2),
                                _ptr(v), v.stride(0), v.stride(1), v.stride(2), _ptr(status_word(table.device)), _stream())
    check(rc, "dsb_kv_read")
    return k, v


_workspace = {}


def workspace_bytes(device) -> int:
    """Bytes of scratch that a call of :func:`attend` on ``device`` takes (``dsb_kv_attn_workspace_bytes``)."""
    n = _workspace.get(device.index)
    if n is None:
        with torch.cuda.device(device):
            n = _workspace[device.index] = int(_lib.lib().dsb_kv_attn_workspace_bytes())
        if n <= 0:
            _workspace.pop(device.index)
            raise _lib.DsbError("dsb_kv_attn_workspace_bytes failed")
    return n


def attend(q, cache: PagedKVCache, table, lens, causal: bool = False, sm_scale=None, out=None):
    """Attention of ``q`` (bf16 ``[B, Sq, H, 128]``) over the first ``lens`` tokens (int, or int32 ``[B]``) of each sequence; H is a
    multiple of the cache's heads, query head h reads cache head ``h // (H // heads)``.  ``causal``: query i sees the keys up to
    position ``lens - Sq + i`` (the queries are the sequence's last tokens, already appended).  A query that sees no key gives
    zeros."""
    dev_lens = lens if isinstance(lens, torch.Tensor) else None
    _require_cuda(q, cache.k, table, dev_lens, out)
    _rows4(q, "q")
    B, Sq, H, _ = q.shape
    if H == 0 or H % cache.heads:
        raise _lib.DsbError(f"{H} query heads do not share {cache.heads} cache heads evenly")
    ld, width = _table(table, B)
    if dev_lens is not None:
        _per_sequence(dev_lens, B, "lens")
    elif not 0 <= lens <= width * cache.page_tokens:
        raise _lib.DsbError(f"{lens} tokens do not fit a table of {width} pages")
    if out is None:
        out = torch.empty((B, Sq, H, HEAD_DIM), dtype=torch.bfloat16, device=q.device)
    else:
        _rows4(out, "out")
        if out.shape != q.shape or any(st == 0 and n > 1 for st, n in zip(out.stride(), out.shape)):
            raise _lib.DsbError("out has the shape of q and a place for each of its values")
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(HEAD_DIM)
    ws = torch.empty(workspace_bytes(q.device), dtype=torch.uint8, device=q.device)
    rc = _lib.lib().dsb_kv_attn(
        cache._ref, _ptr(q), q.stride(0), q.stride(1), q.stride(2), _ptr(out), out.stride(0), out.stride(1), out.stride(2), B, Sq, H,
        _ptr(table), ld, width, _ptr(dev_lens), 0 if dev_lens is not None else lens, 1 if causal else 0, float(sm_scale),
        _ptr(ws), ws.numel(), _ptr(status_word(q.device)), _stream())
    check(rc, "dsb_kv_attn")
    return out

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
_SM_SCALE = 1.0 / math.sqrt(HEAD_DIM)
UNCUT_TOKENS = 256     # sequences up to this length are never cut (DSB_KV_UNCUT_TOKENS): no workspace
DENSE_QUERIES = 256    # fewer queries of a sequence always read the pages
PAGE_TOKENS = (16, 32, 64, 128)


class PagedKVCache:
    """``k``, ``v``: float8_e4m3fn ``[pages, heads, T, 128]``; ``k_exp``, ``v_exp``: int8 ``[pages, heads]``, the power of two
    that a block's values are multiplied by, -64 to 64 (others count as the nearer of the two).  A page needs no preparation: the append that writes its first token sets its
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
        self._device = k.get_device()
        self.pages, self.heads, self.page_tokens = k.shape[:3]

    @classmethod
    def empty(cls, pages: int, heads: int, page_tokens: int = 64, device="cuda") -> "PagedKVCache":
        k, v = (torch.empty((pages, heads, page_tokens, HEAD_DIM), dtype=torch.float8_e4m3fn, device=device) for _ in range(2))
        return cls(k, v, *(torch.zeros((pages, heads), dtype=torch.int8, device=device) for _ in range(2)))

    # the kernels hold these tensors' addresses, so they cannot be replaced
    k = property(lambda self: self._t[0])
    v = property(lambda self: self._t[1])
    k_exp = property(lambda self: self._t[2])
    v_exp = property(lambda self: self._t[3])

    def pages_for(self, tokens: int) -> int:
        """Table entries that a sequence of ``tokens`` needs."""
        return -(-tokens // self.page_tokens)


def _here(cache, *ts):
    """The current device, on which the cache and every tensor of a call must live."""
    dev = cache._device
    if dev < 0 or dev != torch._C._cuda_getDevice():
        _require_cuda(cache.k)
    for t in ts:
        if t is not None and t.get_device() != dev:
            _require_cuda(t)
    return dev


def _table(table, B):
    shape, st = table.shape, table.stride()
    if table.dtype is not torch.int32 or len(shape) != 2:
        raise _lib.DsbError(f"the page table is an int32 [{B}, pages] tensor with contiguous rows")
    (rows, width), (ld, inner) = shape, st
    if rows != B or width == 0 or (inner != 1 and width > 1) or (ld < width and B > 1):
        raise _lib.DsbError(f"the page table is an int32 [{B}, pages] tensor with contiguous rows")
    return (ld if ld > width else width), width


def _per_sequence(t, B, what):
    if t.dtype is not torch.int32 or t.shape != (B,) or not t.is_contiguous():
        raise _lib.DsbError(f"{what} is an int or a contiguous int32 [{B}] tensor")


def _rows4(t, what):
    """(shape, strides, address) of rows that the kernels take."""
    shape, st, ptr = t.shape, t.stride(), t.data_ptr()
    if len(shape) != 4 or shape[3] != HEAD_DIM or t.dtype is not torch.bfloat16 or st[3] != 1 or ptr % 16 \
            or (st[0] | st[1] | st[2]) & 7 or st[0] < 0 or st[1] < 0 or st[2] < 0:
        raise _lib.DsbError(f"{what} is a bf16 [B, tokens, heads, 128] tensor with a contiguous head dimension, 16-byte aligned, "
                            "with strides that are multiples of 8")
    return shape, st, ptr


def append(cache: PagedKVCache, k, v, table, start, counts=None, rope=None, rope_row0: int = 0):
    """Appends ``k`` and ``v`` (bf16 ``[B, n, heads, 128]``, any strides that are multiples of 8) to the sequences of ``table``
    (int32 ``[B, pages]``), from position ``start`` (int, or int32 ``[B]``) on; ``counts`` (int32 ``[B]``): how many of the n rows
    belong to each sequence.  ``rope`` (fp32 ``[rows, 64, 2]`` = cos, sin): ``k`` is rotated by row ``rope_row0 + position``.
    A position or page outside its table leaves that part unwritten and raises at the next ``ops.check_status``."""
    dev_start = start if isinstance(start, torch.Tensor) else None
    dev = _here(cache, k, v, table, dev_start, counts, rope)
    shape, ks, k_ptr = _rows4(k, "k")
    v_shape, vs, v_ptr = _rows4(v, "v")
    B, n, heads, _ = shape
    if v_shape != shape or heads != cache.heads:
        raise _lib.DsbError(f"k and v are [B, n, {cache.heads}, 128] rows of one shape")
    ld, width = _table(table, B)
    if dev_start is not None:
        _per_sequence(dev_start, B, "start")
        start = 0
    elif not 0 <= start <= width * cache.page_tokens - (n if counts is None else 0):
        raise _lib.DsbError(f"{n} rows from position {start} on do not fit a table of {width} pages")
    if counts is not None:
        _per_sequence(counts, B, "counts")
    rope_rows = 0
    if rope is not None:
        if rope.dtype != torch.float32 or rope.dim() != 3 or rope.shape[1:] != (64, 2) or not rope.is_contiguous():
            raise _lib.DsbError("rope is a contiguous float32 [rows, 64, 2] table")
        if rope.data_ptr() % 16 or not -(1 << 31) <= rope_row0 < 1 << 31:
            raise _lib.DsbError("rope is 16-byte aligned and rope_row0 a 32-bit number")
        rope_rows = rope.shape[0]
    rc = _lib.lib().dsb_kv_append(cache._ref, k_ptr, ks[0], ks[1], ks[2], v_ptr, vs[0], vs[1], vs[2], B, n, table.data_ptr(), ld, width,
                                  _ptr(dev_start), start, _ptr(counts), _ptr(rope), rope_rows, rope_row0, _status_ptr(dev), _stream())
    check(rc, "dsb_kv_append")


def _status_ptr(dev: int):
    word = ops._status.get(dev)
    return (word if word is not None else status_word(torch.device("cuda", dev))).data_ptr()


def read(cache: PagedKVCache, table, n: int, first: int = 0):
    """Tokens ``first .. first + n - 1`` of each sequence as bf16 ``(k, v)``, each ``[B, n, heads, 128]`` (exact)."""
    dev = _here(cache, table)
    B = table.shape[0]
    ld, width = _table(table, B)
    if n < 0 or first < 0 or first + n > width * cache.page_tokens:
        raise _lib.DsbError(f"tokens {first}..{first + n - 1} are not in a table of {width} pages")
    k, v = torch.empty((2, B, n, cache.heads, HEAD_DIM), dtype=torch.bfloat16, device=table.device).unbind(0)
    sb, sn, sh, _ = k.stride()
    rc = _lib.lib().dsb_kv_read(cache._ref, table.data_ptr(), ld, width, B, first, n, k.data_ptr(), sb, sn, sh, v.data_ptr(), sb, sn, sh,
                                _status_ptr(dev), _stream())
    check(rc, "dsb_kv_read")
    return k, v


_workspace = {}


def workspace_bytes(device: int) -> int:
    """Bytes of scratch that a call of :func:`attend` on a device takes (``dsb_kv_attn_workspace_bytes``)."""
    n = _workspace.get(device)
    if n is None:
        with torch.cuda.device(device):
            n = int(_lib.lib().dsb_kv_attn_workspace_bytes())
        if n <= 0:
            raise _lib.DsbError("dsb_kv_attn_workspace_bytes failed")
        _workspace[device] = n
    return n


def dense_pays(batch: int, queries: int, heads: int, cache_heads: int, tokens: int) -> bool:
    """Whether ``attend`` gathers the sequences as bf16 rows for the dense attention kernel, instead of reading the pages: an estimate
    of both in microseconds, from times on one B200 (148 SMs).  Pages: 9, 9 more where sequences may be cut, and 210 Mflop a microsecond.  Dense: 8 for the gather (4
    on the device, but two calls' arguments) and its bytes, then for each query head of a group one launch of items of 256 rows, 74 at
    a time, each 2.4 and 0.62 a tile of 128 keys; one cache head's query heads are rows of one launch.  Measured on the device (pages,
    dense; heads / cache heads, queries x tokens): 24/24 256 x 77: 9, 13; 256 x 512: 24, 16; 4096 x 4096: 925, 190; 32/8 512 x 512:
    38, 45; 4096 x 77: 50, 51; 4096 x 4096: 1228, 251; 4/1 1200 x 77: 10, 12; 1200 x 4096: 61, 37; 24440 x 512: 149, 39."""
    if queries < DENSE_QUERIES or tokens <= 0 or batch <= 0:
        return False
    share = heads // cache_heads
    pages = (9 if tokens <= UNCUT_TOKENS else 18) + 4 * HEAD_DIM * batch * queries * heads * (tokens + 64) / 210e6
    waves = max(1.0, batch * cache_heads * -(-queries // 256) / 74)
    dense = 8 + batch * tokens * cache_heads * 768 / 4e6 + share * (5 + waves * (2.4 + 0.62 * -(-tokens // 128)))
    return dense < pages


def attend(q, cache: PagedKVCache, table, lens, causal: bool = False, sm_scale=None, out=None, pages_only: bool = False):
    """Attention of ``q`` (bf16 ``[B, Sq, H, 128]``) over the first ``lens`` tokens (int, or int32 ``[B]``) of each sequence; H is a
    multiple of the cache's heads, query head h reads cache head ``h // (H // heads)``.  ``causal``: query i sees the keys up to
    position ``lens - Sq + i`` (the queries are the sequence's last tokens, already appended).  A query that sees no key gives
    zeros.  Table entries that are no pages raise at the next ``ops.check_status``; until then their keys count as masked.

    Many queries over a length that is an int, without ``causal``, are faster with the dense attention kernel over the sequences' rows in
    bf16, and take it where ``dense_pays`` says so.  That differs in three things: the rows take 512 bytes a token and cache head for
    the time of the call; probabilities are rounded to bf16, 8 bits where the pages keep 11 (an error of 0.0024 instead of 0.0017 of the
    result, most of it the result's own rounding); and keys of table entries that are no pages count as zeros.  ``pages_only``: never."""
    dev_lens = lens if isinstance(lens, torch.Tensor) else None
    dev = _here(cache, q, table, dev_lens, out)
    shape, qs, q_ptr = _rows4(q, "q")
    B, Sq, H, _ = shape
    heads = cache.heads
    if H == 0 or H % heads:
        raise _lib.DsbError(f"{H} query heads do not share {heads} cache heads evenly")
    ld, width = _table(table, B)
    most = width * cache.page_tokens
    if dev_lens is not None:
        _per_sequence(dev_lens, B, "lens")
        lens = 0
    elif not 0 <= lens <= most:
        raise _lib.DsbError(f"{lens} tokens do not fit a table of {width} pages")
    else:
        most = lens
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        out_ptr, os = out.data_ptr(), (Sq * H * HEAD_DIM, H * HEAD_DIM, HEAD_DIM)
    else:
        out_shape, os, out_ptr = _rows4(out, "out")
        if out_shape != shape or any(st == 0 and n > 1 for st, n in zip(os, shape)):
            raise _lib.DsbError("out has the shape of q and a place for each of its values")
    if sm_scale is None:
        sm_scale = _SM_SCALE
    # (the dense kernel's tensor maps have no stride of 0)
    if dev_lens is None and not causal and not pages_only and qs[0] and qs[1] and qs[2] and os[0] and os[1] and os[2]:
        share, rows, q_row, o_row = H // heads, Sq, qs[1], os[1]
        if heads == 1 and q_row == share * qs[2] and o_row == share * os[2]:
            share, rows, q_row, o_row = 1, Sq * share, qs[2], os[2]       # one cache head: its query heads are rows like any others
        if dense_pays(B, rows, heads * share, heads, lens):
            k, v = read(cache, table, lens)
            sb, sn, sh, _ = k.stride()
            for g in range(share):      # a cache head's queries, one of its query heads at a time
                rc = _lib.lib().dsb_flash_attn(
                    q_ptr + 2 * g * qs[2], k.data_ptr(), v.data_ptr(), out_ptr + 2 * g * os[2], B, heads, rows, lens, HEAD_DIM,
                    qs[0], q_row, share * qs[2], sb, sn, sh, sb, sn, sh, os[0], o_row, share * os[2], sm_scale, _status_ptr(dev), _stream())
                check(rc, "dsb_flash_attn")
            return out
    ws_ptr = ws_bytes = 0
    if most > UNCUT_TOKENS:         # a sequence may be cut along its keys
        ws_bytes = workspace_bytes(dev)
        ws = q.new_empty(ws_bytes, dtype=torch.uint8)
        ws_ptr = ws.data_ptr()
    rc = _lib.lib().dsb_kv_attn(
        cache._ref, q_ptr, qs[0], qs[1], qs[2], out_ptr, os[0], os[1], os[2], B, Sq, H, table.data_ptr(), ld, width, _ptr(dev_lens), lens,
        1 if causal else 0, sm_scale, ws_ptr, ws_bytes, _status_ptr(dev), _stream())
    check(rc, "dsb_kv_attn")
    return out

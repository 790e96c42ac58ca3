"""Linears whose weights stay in 4 bits, with one fp16 scale (and, optionally, minimum) per row and group of columns: code
``c`` (0..15) stands for ``s * (c - 8)``, or ``s * c + m``.  GGUF Q4_0, Q4_1 and Q4_K weights are taken over with their own
codes; any other weight is quantised here.  A few activation rows are multiplied as they are (``dsb_gemv_int4``); for more rows
the weight is expanded to bf16 (``dequant``) and goes through the GEMM."""
import ctypes
from dataclasses import dataclass
from typing import List, Optional

import torch

from . import _lib, ops
from ._lib import ACT_NONE, check
from .ops import _ptr, _require_cuda, _rows, _stream

GROUPS = (32, 64, 128)
MAX_ROWS = 32     # DSB_INT4_MAX_ROWS: activation rows of one product
GGUF_TYPES = ("Q4_0", "Q4_1", "Q4_K")


@dataclass
class Int4Linear:
    """A 4-bit weight and its fp32 bias (``packed.PackedLinear`` of the other formats)."""
    w: "Int4Weight"
    bias: Optional[torch.Tensor]

    @property
    def out_features(self):
        return self.w.N

    @property
    def in_features(self):
        return self.w.K


class Int4Weight:
    """A 4-bit ``[N, K]`` weight laid out for the kernels (``dsb_int4_pack``): ``payload`` uint8 ``[ceil(N/16), ceil(K/64), 512]``,
    ``scales`` and ``mins`` (or None) fp16 ``[ceil(N/16), tiles, 8, groups per tile, 2]``.  The tensors cannot be replaced: the
    kernels take their addresses, which are checked here."""

    __slots__ = ("_t", "N", "K", "group", "_device", "_args", "_ref")

    def __init__(self, payload, scales, mins, N: int, K: int, group: int):
        if N <= 0 or K <= 0 or K % 2 or group not in GROUPS:
            raise _lib.DsbError(f"Int4Weight: [{N}, {K}] in groups of {group} is no 4-bit weight")
        rb, tiles = -(-N // 16), -(-K // (128 if group == 128 else 64))
        need = rb * tiles * 16 * (2 if group == 32 else 1)
        if payload.dtype != torch.uint8 or not payload.is_contiguous() or payload.numel() != rb * -(-K // 64) * 512:
            raise _lib.DsbError("Int4Weight: the payload is not a contiguous uint8 tensor of its size")
        for t in (scales, mins):
            if t is not None and (t.dtype != torch.float16 or not t.is_contiguous() or t.numel() != need or t.device != payload.device):
                raise _lib.DsbError("Int4Weight: scales and mins are contiguous float16 tensors of their size, where the payload is")
        self._t, self.N, self.K, self.group, self._device = (payload, scales, mins), N, K, group, payload.get_device()
        self._args = _lib.Int4Args(payload.data_ptr(), scales.data_ptr(), _ptr(mins), N, K, group)
        self._ref = ctypes.byref(self._args)

    payload = property(lambda self: self._t[0])
    scales = property(lambda self: self._t[1])
    mins = property(lambda self: self._t[2])
    out_features = property(lambda self: self.N)
    in_features = property(lambda self: self.K)
    device = property(lambda self: self._t[0].device)

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self._t if t is not None)


def _empty(N, K, group, has_min, device) -> Int4Weight:
    rb = -(-N // 16)
    shape = (rb, -(-K // 128), 8, 1, 2) if group == 128 else (rb, -(-K // 64), 8, 64 // group, 2)
    scales = torch.empty(shape, dtype=torch.float16, device=device)
    return Int4Weight(torch.empty((rb, -(-K // 64), 512), dtype=torch.uint8, device=device), scales,
                      torch.empty_like(scales) if has_min else None, N, K, group)


def _check_weight(w):
    if type(w) is not Int4Weight:
        raise _lib.DsbError("expected an Int4Weight (int4.from_codes, int4.quantize, int4.from_gguf)")
    if w._device != torch._C._cuda_getDevice():
        _require_cuda(w.payload)


def _rows_apart(t):
    """``t`` as rows that the kernels can step through: a copy where they overlap (a broadcast tensor)."""
    return t.contiguous() if t.shape[0] > 1 and t.stride(0) < t.shape[1] else t


def from_codes(codes, scales, mins=None, group=32) -> Int4Weight:
    """Lays out a weight that is quantised already: ``codes`` uint8 ``[N, K/2]`` (even column in the low nibble), ``scales`` and
    ``mins`` fp16 ``[N, ceil(K / group)]``."""
    _require_cuda(codes, scales, mins)
    if group not in GROUPS:
        raise _lib.DsbError(f"int4 groups are {GROUPS} columns, got {group}")
    _rows(codes)
    codes = _rows_apart(codes)
    N, half, ld = _rows(codes)
    K = 2 * half
    if codes.dtype != torch.uint8 or N == 0 or K == 0:
        raise _lib.DsbError("int4.from_codes takes uint8 codes [N, K/2], two per byte")
    for name, t in (("scales", scales), ("mins", mins)):
        if t is None:
            continue
        if t.dtype != torch.float16 or t.dim() != 2 or tuple(t.shape) != (N, -(-K // group)):
            raise _lib.DsbError(f"int4.from_codes {name} must be float16 [{N}, {-(-K // group)}], got {t.dtype} {tuple(t.shape)}")
    if scales.stride(1) != 1 or _rows_apart(scales) is not scales or (mins is not None and mins.stride() != scales.stride()):
        scales, mins = scales.contiguous(), None if mins is None else mins.contiguous()
    w = _empty(N, K, group, mins is not None, codes.device)
    rc = _lib.lib().dsb_int4_pack(_ptr(codes), max(ld, half), _ptr(scales), _ptr(mins), max(scales.stride(0), scales.shape[1]), N, K, group,
                                  _ptr(w.payload), _ptr(w.scales), _ptr(w.mins), _stream())
    check(rc, "dsb_int4_pack")
    return w


def quantize_codes(W, group=32, asymmetric=False):
    """(codes, scales, mins or None) of a float weight ``[N, K]``: per group s = amax / 7, or with ``asymmetric``
    s = (max - min) / 15 and m = min, rounded to fp16 before the codes are."""
    _require_cuda(W)
    if group not in GROUPS:
        raise _lib.DsbError(f"int4 groups are {GROUPS} columns, got {group}")
    _rows(W)
    W = _rows_apart(W)
    N, K, ld = _rows(W)
    if W.dtype not in (torch.float32, torch.bfloat16) or N == 0 or K == 0 or K % 2:
        raise _lib.DsbError("int4.quantize takes fp32 or bf16 weights [N, K] with an even K")
    codes = torch.empty((N, K // 2), dtype=torch.uint8, device=W.device)
    scales = torch.empty((N, -(-K // group)), dtype=torch.float16, device=W.device)
    mins = torch.empty_like(scales) if asymmetric else None
    rc = _lib.lib().dsb_int4_quantize(_ptr(W), max(ld, K), W.dtype == torch.bfloat16, N, K, group, _ptr(codes), codes.stride(0),
                                      _ptr(scales), _ptr(mins), _stream())
    check(rc, "dsb_int4_quantize")
    return codes, scales, mins


def quantize(W, group=32, asymmetric=False) -> Int4Weight:
    """Quantises a float weight ``[N, K]`` and lays it out."""
    return from_codes(*quantize_codes(W, group, asymmetric), group=group)


def gguf_codes(raw, qtype: str):
    """(codes, scales, mins or None) of GGUF bytes ``[N, K / block * bytes]`` (uint8), group 32.  The codes, and the scales and
    minima of Q4_0 and Q4_1, are the file's own; Q4_K's products of a scale and a 6-bit factor are rounded to fp16."""
    _require_cuda(raw)
    if qtype not in GGUF_TYPES:
        raise _lib.DsbError(f"int4.from_gguf takes {GGUF_TYPES} blocks, got {qtype}")
    code, tsz, bsz = ops.GGUF_TYPES[qtype]
    if raw.dtype != torch.uint8 or raw.dim() != 2 or raw.stride(1) != 1 or raw.shape[0] == 0 or raw.shape[1] == 0 or raw.shape[1] % tsz:
        raise _lib.DsbError(f"int4.from_gguf({qtype}) takes uint8 rows of {tsz}-byte blocks")
    raw = _rows_apart(raw)
    N, K = raw.shape[0], raw.shape[1] // tsz * bsz
    codes = torch.empty((N, K // 2), dtype=torch.uint8, device=raw.device)
    scales = torch.empty((N, K // 32), dtype=torch.float16, device=raw.device)
    mins = None if qtype == "Q4_0" else torch.empty_like(scales)
    rc = _lib.lib().dsb_int4_from_gguf(code, _ptr(raw), max(raw.stride(0), raw.shape[1]), N, K, _ptr(codes), codes.stride(0),
                                       _ptr(scales), _ptr(mins), _stream())
    check(rc, "dsb_int4_from_gguf")
    return codes, scales, mins


def from_gguf(raw, qtype: str) -> Int4Weight:
    """A GGUF Q4_0, Q4_1 or Q4_K weight that stays in 4 bits."""
    return from_codes(*gguf_codes(raw, qtype), group=32)


def stack(parts: List[Int4Weight]) -> Int4Weight:
    """The weights below one another, as one: Linears that share their input run in one launch.  Every part but the last has a
    multiple of 16 rows."""
    first = parts[0]
    for p in parts:
        _check_weight(p)
        if (p.K, p.group, p.mins is None, p.device) != (first.K, first.group, first.mins is None, first.device):
            raise _lib.DsbError("int4.stack takes weights of one width, group size, kind and device")
    if any(p.N % 16 for p in parts[:-1]):
        raise _lib.DsbError("int4.stack: every part but the last has a multiple of 16 rows")
    return Int4Weight(torch.cat([p.payload for p in parts]), torch.cat([p.scales for p in parts]),
                      None if first.mins is None else torch.cat([p.mins for p in parts]), sum(p.N for p in parts), first.K, first.group)


def pack_linear(weight, bias, device, group=32, asymmetric=True) -> Int4Linear:
    """Quantises one ``[N, K]`` weight on the device."""
    w = weight.reshape(weight.shape[0], -1).to(device=device)
    if w.dtype not in (torch.float32, torch.bfloat16):
        w = w.float()
    b = None if bias is None else bias.to(device=device, dtype=torch.float32).contiguous()
    return Int4Linear(quantize(w.contiguous(), group, asymmetric), b)


def stack_for_gemv(parts: List[Int4Linear]) -> Int4Linear:
    """Linears that share their input, as one (``packed.stack_for_gemv`` of the other formats)."""
    return Int4Linear(stack([p.w for p in parts]), torch.cat([p.bias for p in parts]).contiguous())


def dequant(w: Int4Weight, out=None):
    """The weight as bf16 ``[N, K]``."""
    _check_weight(w)
    _require_cuda(out)
    if out is None:
        out = torch.empty((w.N, w.K), dtype=torch.bfloat16, device=w.device)
    if out.dtype != torch.bfloat16 or tuple(out.shape) != (w.N, w.K) or out.stride(1) != 1 or (w.N > 1 and out.stride(0) < w.K):
        raise _lib.DsbError(f"int4.dequant output must be bfloat16 [{w.N}, {w.K}] rows")
    rc = _lib.lib().dsb_int4_dequant(w._ref, _ptr(out), max(out.stride(0), w.K), _stream())
    check(rc, "dsb_int4_dequant")
    return out


def gemv(w: Int4Weight, x, bias=None, act_in=ACT_NONE, act_out=ACT_NONE, out=None, accumulate=False):
    """``act_out(act_in(x) @ w.T + bias)`` for one row ``x[K]`` or up to ``MAX_ROWS`` rows ``x[M, K]`` (float32 or bfloat16),
    fp32 arithmetic; ``out`` (default: the dtype of ``x``) is float32 or bfloat16 and, with ``accumulate``, added to."""
    _check_weight(w)
    dev, N, K = w._device, w.N, w.K
    if x.get_device() != dev or (bias is not None and bias.get_device() != dev) or (out is not None and out.get_device() != dev):
        _require_cuda(w.payload, x, bias, out)
    shape, st = x.shape, x.stride()
    if len(shape) == 2:
        M, ld_x = shape[0], st[0]
    elif len(shape) == 1:
        M, ld_x = 1, K
    else:
        raise _lib.DsbError(f"int4.gemv takes x as [{K}] or [M, {K}], got {tuple(shape)}")
    if shape[-1] != K or st[-1] != 1 or (M > 1 and ld_x < K):
        raise _lib.DsbError(f"int4.gemv takes x as [{K}] or [M, {K}] with contiguous rows that do not overlap, got {tuple(shape)}")
    if M > MAX_ROWS:
        raise _lib.DsbError(f"int4.gemv takes up to {MAX_ROWS} rows, got {M}: expand the weight (int4.dequant) for more")
    dtype = x.dtype
    x_bf16 = dtype is torch.bfloat16
    if not x_bf16 and dtype is not torch.float32:
        raise _lib.DsbError(f"int4.gemv takes float32 or bfloat16 rows, got {dtype}")
    if out is None:
        if accumulate:
            raise _lib.DsbError("int4.gemv: accumulate needs an out to add to")
        out, ld_y, y_bf16 = x.new_empty((M, N) if len(shape) == 2 else (N,)), N, x_bf16
    else:
        want = (M, N) if len(shape) == 2 else (N,)
        ld_y, y_bf16 = out.stride(0) if len(want) == 2 else N, out.dtype is torch.bfloat16
        if out.shape != want or (out.stride(-1) != 1 and N > 1) or (M > 1 and ld_y < N):
            raise _lib.DsbError(f"int4.gemv output must be {want} with contiguous rows, got {tuple(out.shape)}")
        if not y_bf16 and out.dtype is not torch.float32:
            raise _lib.DsbError(f"int4.gemv writes float32 or bfloat16 rows, got {out.dtype}")
    bias_ptr = None
    if bias is not None:
        if bias.dtype is not torch.float32 or bias.numel() != N or not bias.is_contiguous():
            raise _lib.DsbError(f"int4.gemv bias must be contiguous float32 with {N} elements")
        bias_ptr = bias.data_ptr()
    rc = _lib.lib().dsb_gemv_int4(w._ref, x.data_ptr(), ld_x, x_bf16, bias_ptr, out.data_ptr(), ld_y, y_bf16, M, act_in, act_out,
                                  accumulate, _stream())
    check(rc, "dsb_gemv_int4")
    return out

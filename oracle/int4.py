"""4-bit weights with group scales, restated on the CPU: codes 0..15 that stand for ``s * (c - 8)`` or ``s * c + m``."""
import torch


def unpack(codes):
    """uint8 [N, K/2] -> int64 [N, K]; the even column is in the low nibble."""
    return torch.stack([codes & 15, codes >> 4], dim=-1).reshape(codes.shape[0], -1).long()


def pack(q):
    """int [N, K] (0..15) -> uint8 [N, K/2]."""
    q = q.to(torch.uint8)
    return q[:, 0::2] | (q[:, 1::2] << 4)


def values(codes, scales, mins, group, dtype=torch.float64):
    """The weight that the codes stand for, in ``dtype`` (fp32: product and sum rounded one after the other)."""
    q = unpack(codes).to(dtype)
    at = torch.arange(q.shape[1]) // group
    s = scales.to(dtype)[:, at]
    return s * (q - 8) if mins is None else s * q + mins.to(dtype)[:, at]


def quantize(W, group, asymmetric):
    """(codes, scales, mins) in fp32 arithmetic: s = amax / 7, or s = (max - min) / 15 and m = min, rounded to fp16."""
    N, K = W.shape
    groups = -(-K // group)
    w = W.float()
    pad = torch.nn.functional.pad(w, (0, groups * group - K), value=float("nan")).view(N, groups, group)
    hi = pad.nan_to_num(nan=-float("inf")).amax(-1)
    lo = pad.nan_to_num(nan=float("inf")).amin(-1)
    s = ((hi - lo) / 15 if asymmetric else torch.maximum(hi.abs(), lo.abs()) / 7).clamp(max=65504).half()
    m = lo.clamp(-65504, 65504).half() if asymmetric else None
    at = torch.arange(K) // group
    sf = s.float()[:, at]
    u = torch.where(sf > 0, torch.round((w - m.float()[:, at] if asymmetric else w) / sf), torch.zeros_like(w))
    q = u.clamp(0, 15) if asymmetric else u.clamp(-8, 7) + 8
    return pack(q), s, m


def gguf_fields(raw, qtype):
    """(codes [N, K], scales, mins) of Q4_0, Q4_1 or Q4_K rows, element by element; group 32."""
    size, block = {"Q4_0": (18, 32), "Q4_1": (20, 32), "Q4_K": (144, 256)}[qtype]
    N = raw.shape[0]
    blk = raw.reshape(-1, size)
    f16 = lambda off: blk[:, off:off + 2].contiguous().view(torch.float16)  # noqa: E731
    if qtype != "Q4_K":
        qs = blk[:, size - 16:]
        q = torch.cat([qs & 15, qs >> 4], dim=1)
        s, m = f16(0), None if qtype == "Q4_0" else f16(2)
        return q.reshape(N, -1), s.reshape(N, -1), None if m is None else m.reshape(N, -1)
    from .gguf import _k_scales
    sc, mn = _k_scales(blk[:, 4:16])
    s = (f16(0).float() * sc.float()).half()
    m = (-(f16(2).float() * mn.float())).half()
    qs = blk[:, 16:144].reshape(-1, 4, 1, 32)
    q = ((qs >> torch.tensor([0, 4], dtype=torch.uint8).view(1, 1, 2, 1)) & 15).reshape(-1, 256)
    return q.reshape(N, -1), s.reshape(N, -1), m.reshape(N, -1)


def linear(x, w, bias=None, act_in=None, act_out=None):
    """act_out(act_in(x) @ w.T + bias) in 64 bits."""
    x = x.double()
    y = (act_in(x) if act_in else x) @ w.double().t()
    if bias is not None:
        y = y + bias.double()
    return act_out(y) if act_out else y

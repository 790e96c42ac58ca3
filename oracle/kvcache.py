"""The paged 8-bit key/value cache restated on the CPU, one sequence, page and head at a time, in 64 bits."""
import math

import torch

D = 128


def exponent(amax: float) -> int:
    """The least e in -64..64 with amax <= 448 * 2^e."""
    e = -64
    while e < 64 and amax > 448.0 * 2.0 ** e:
        e += 1
    return e


def round_e4m3(x):
    """The nearest e4m3 value (ties to the even one, largest 448) of 64-bit numbers; NaN stays."""
    ex = torch.frexp(x)[1] - 1
    step = torch.ldexp(torch.ones_like(x), ex.clamp(min=-6) - 3)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def rotate(k, table, first):
    """Rows k [n, H, 128] (fp32) rotated by rows first.. of a (cos, sin) table, each operation rounded to fp32."""
    cs = table[first:first + k.shape[0]]
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    a, b = k[..., 0::2], k[..., 1::2]
    out = torch.empty_like(k)
    out[..., 0::2], out[..., 1::2] = a * c - b * s, a * s + b * c
    return out


def append(pages, exps, table, start, counts, rows):
    """In place on one pool: ``pages`` float64 [P, H, T, 128] (the e4m3 values), ``exps`` int [P, H]; rows fp32 [B, n, H, 128]."""
    T, H = pages.shape[2], pages.shape[1]
    for b in range(rows.shape[0]):
        t, end = int(start[b]), int(start[b]) + int(counts[b])
        while t < end:
            upto = min(end, (t // T + 1) * T)
            p, slot = int(table[b, t // T]), t % T
            new = rows[b, t - int(start[b]):upto - int(start[b])].double()
            for h in range(H):
                r = new[:, h]
                fin = r[r.isfinite()].abs()
                e = exponent(float(fin.max()) if fin.numel() else 0.0)
                if slot > 0:
                    was = int(exps[p, h])
                    e = max(e, was)
                    if e > was:
                        pages[p, h, :slot] = round_e4m3(pages[p, h, :slot] * 2.0 ** (was - e))
                exps[p, h] = e
                pages[p, h, slot:slot + upto - t] = round_e4m3((r * 2.0 ** -e).clamp(-448, 448))
            t = upto


def held(pages, exps, table_row, n):
    """Values of the first n tokens of a sequence, float64 [n, H, 128]."""
    T = pages.shape[2]
    idx = table_row[: -(-n // T)].long()
    x = pages[idx].double() * (2.0 ** exps[idx].double())[..., None, None]
    return x.permute(0, 2, 1, 3).reshape(-1, pages.shape[1], D)[:n]


def attend(q, pages, exps, table, lens, causal=False, sm_scale=None, ok=None):
    """Attention in 64 bits; ``pages`` and ``exps`` are (k, v) pairs.  ``ok`` (bool [B, tokens]): keys that count."""
    B, Sq, H, _ = q.shape
    Hk = pages[0].shape[1]
    scale = 1 / math.sqrt(D) if sm_scale is None else sm_scale
    out = torch.zeros(B, Sq, H, D, dtype=torch.float64)
    for b in range(B):
        n = int(lens[b])
        if n == 0:
            continue
        k, v = (held(pages[i], exps[i], table[b], n) for i in (0, 1))
        for h in range(H):
            s = q[b, :, h].double() @ k[:, h // (H // Hk)].t() * scale
            for i in range(Sq):
                m = min(n, n - Sq + i + 1) if causal else n
                keep = torch.arange(n) < m
                if ok is not None:
                    keep &= ok[b, :n]
                if keep.any():
                    out[b, i, h] = torch.softmax(s[i, keep], -1) @ v[keep, h // (H // Hk)]
    return out

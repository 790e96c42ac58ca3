"""The operators on what a model keeps in few bits, as cases that can be timed and compared: products of a few activation
rows with 4-bit weights, keys and values appended to a paged 8-bit cache, and attention over that cache.

4-bit weights: code ``c`` (0..15) of row n and column k stands for ``s * (c - 8)``, or ``s * c + m`` where the group has a
minimum, with one fp16 ``s`` (and ``m``) for each row and group of consecutive columns.

Cache: pages of T tokens, ``[page, head, token, 128]`` in e4m3; the block of one page and head stands for its e4m3 values times
2^e, with one whole exponent e for the block.  A block that begins with an append takes the least e that its new rows' largest
magnitude fits under (448 * 2^e); one that has rows already keeps the larger of its own and that, and its rows are rounded
again if it grew."""
import math

import torch

own = False

DEV = "cuda"
D = 128


def listed():
    return [
        # second Linear of a small timestep embedder: one fp32 row, a call that is all latency
        {"name": "rows4-one-small", "op": "rows4", "rows": 1, "n": 768, "k": 256, "group": 32, "mins": False, "bf16": False,
         "bias": True, "silu": False},
        # time embedding of the 5120-wide video model, 32-column blocks with minima: one conditioning vector
        {"name": "rows4-embedder", "op": "rows4", "rows": 1, "n": 5120, "k": 5120, "group": 32, "mins": True, "bf16": False,
         "bias": True, "silu": True},
        # a feed-forward's first Linear on five bf16 rows; odd row count, a last group that is not full
        {"name": "rows4-few-odd", "op": "rows4", "rows": 5, "n": 13827, "k": 5104, "group": 64, "mins": True, "bf16": True,
         "bias": True, "silu": False},
        # modulation Linears of many blocks stacked: one vector against 2.5 G weights, bound by their bytes
        {"name": "rows4-modulation", "op": "rows4", "rows": 1, "n": 491520, "k": 5120, "group": 32, "mins": False,
         "bf16": False, "bias": True, "silu": True},
        # one token of each of sixteen sequences, in the middle of a page or at the start of one
        {"name": "append-token", "op": "append", "batch": 16, "n": 1, "heads": 8, "page": 64, "past": 4096, "rope": True},
        # the 512 text tokens of a prompt, all heads of the 5120-wide model, no rotation
        {"name": "append-prompt", "op": "append", "batch": 1, "n": 512, "heads": 40, "page": 64, "past": 0, "rope": False},
        # four latent frames of 1560 tokens behind what two sequences hold, ragged
        {"name": "append-frames", "op": "append", "batch": 2, "n": 6240, "heads": 40, "page": 64, "past": 9000, "rope": True},
        # the shortest call: one query of one sequence over 77 text tokens
        {"name": "attend-token-short", "op": "attend", "batch": 1, "sq": 1, "heads": 24, "kv_heads": 24, "page": 16, "len": 77,
         "ragged": True, "causal": False},
        # one token of each of sixteen sequences of very different lengths, five query heads to a key head
        {"name": "attend-token-batch", "op": "attend", "batch": 16, "sq": 1, "heads": 40, "kv_heads": 8, "page": 64,
         "len": 16384, "ragged": True, "causal": False},
        # four new tokens over two long sequences, one length odd: split over the keys
        {"name": "attend-long", "op": "attend", "batch": 2, "sq": 4, "heads": 32, "kv_heads": 4, "page": 128, "len": 131071,
         "ragged": True, "causal": True},
        # a chunk of new tokens over ragged sequences, each token up to itself
        {"name": "attend-chunk", "op": "attend", "batch": 3, "sq": 260, "heads": 40, "kv_heads": 8, "page": 32, "len": 8100,
         "ragged": True, "causal": True},
        # cross-attention of an 81-frame 480p video's tokens with a prompt's 512
        {"name": "attend-prompt", "op": "attend", "batch": 1, "sq": 32760, "heads": 40, "kv_heads": 40, "page": 64, "len": 512,
         "ragged": False, "causal": False},
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(("rows4", "append", "attend", "attend"))
    if op == "rows4":
        k = _spread(rng, 40, 13824)
        n = min(_spread(rng, 16, 491520), 491520 * 5120 // k)
        rows = 1 if n * k > 1 << 28 else rng.choice((1, 1, 2, 3, 4, 7, 8, 16))
        return {"op": op, "rows": rows, "n": n, "k": k // 2 * 2, "group": rng.choice((32, 32, 64, 128)),
                "mins": rng.random() < 0.5, "bf16": rng.random() < 0.5, "bias": rng.random() < 0.7, "silu": rng.random() < 0.3}
    if op == "append":
        heads, batch = rng.choice((1, 4, 8, 24, 40)), _spread(rng, 1, 16)
        n = min(_spread(rng, 1, 6240), 2 * 6240 * 40 // (heads * batch))
        return {"op": op, "batch": batch, "n": n, "heads": heads, "page": rng.choice((16, 32, 64, 128)),
                "past": rng.choice((0, _spread(rng, 1, 9000))), "rope": rng.random() < 0.7}
    kv_heads = rng.choice((1, 2, 4, 8, 24, 40))
    page = rng.choice((16, 32, 64, 128))
    if rng.random() < 0.25:      # many queries over a length that the caller knows
        heads = kv_heads if kv_heads >= 24 else 4 * kv_heads
        return {"op": op, "batch": 1, "sq": _spread(rng, 200, 32760), "heads": heads, "kv_heads": kv_heads, "page": page,
                "len": _spread(rng, 1, 512), "ragged": False, "causal": False}
    share = rng.choice((1, 2, 5, 8)) if kv_heads <= 8 else 1
    batch, causal = _spread(rng, 1, 16), rng.random() < 0.5
    length = min(_spread(rng, 1, 131071), max(1, (1 << 20) // (batch * kv_heads)))
    sq = min(rng.choice((1, 1, 2, _spread(rng, 1, 400))), max(1, (1 << 28) // (batch * kv_heads * share * length)))
    return {"op": op, "batch": batch, "sq": sq, "heads": kv_heads * share, "kv_heads": kv_heads, "page": page, "len": length,
            "ragged": True, "causal": causal}


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed * 7919 + 1)


def _pool(g, pages, heads, page):
    """A pool's keys or values and their exponents: blocks of about unit variance, as earlier appends left them."""
    x = torch.randn(pages, heads, page, D, generator=g, device=DEV).mul_(90).clamp_(-448, 448).to(torch.float8_e4m3fn)
    return x, torch.randint(-9, -4, (pages, heads), generator=g, device=DEV, dtype=torch.int8)


def _table(g, batch, width):
    """Pages of each sequence, scattered over the pool as they were handed out, and two spare ones."""
    return torch.randperm(batch * width + 2, generator=g, device=DEV)[: batch * width].view(batch, width).int()


def _angles(rows):
    """(cos, sin) of a position for 64 pairs, fp32, from angles in 64 bits."""
    f = 10000.0 ** (-torch.arange(64, device=DEV, dtype=torch.float64) / 64)
    a = torch.outer(torch.arange(rows, device=DEV, dtype=torch.float64), f)
    return torch.stack([a.cos(), a.sin()], dim=-1).float().contiguous()


def _rand_int(g, lo, hi, n):
    return torch.randint(lo, hi + 1, (n,), generator=g, device=DEV, dtype=torch.int32)


def prepare(case, seed):
    g, c = _gen(seed), case
    if c["op"] == "rows4":
        n, k, groups = c["n"], c["k"], -(-c["k"] // c["group"])
        s = {"codes": torch.randint(0, 256, (n, k // 2), generator=g, device=DEV, dtype=torch.uint8),
             "scales": (torch.rand(n, groups, generator=g, device=DEV) * 0.004 + 0.002).half(), "mins": None, "bias": None}
        if c["mins"]:
            s["mins"] = (torch.randn(n, groups, generator=g, device=DEV) * 0.004 - 0.03).half()
        x = torch.randn(c["rows"], k, generator=g, device=DEV)
        s["x"] = x.bfloat16() if c["bf16"] else x
        if c["bias"]:
            s["bias"] = torch.randn(n, generator=g, device=DEV)
        if own:      # laid out once, as a model keeps its weights
            from diffsynth_engine_b200 import int4
            s["weight"] = int4.from_codes(s["codes"], s["scales"], s["mins"], group=c["group"])
            del s["codes"], s["scales"], s["mins"]
        return {**s, "case": c}
    batch, page = c["batch"], c["page"]
    if c["op"] == "append":
        n, heads = c["n"], c["heads"]
        width = -(-(c["past"] + n) // page)
        s = {"table": _table(g, batch, width), "start": _rand_int(g, c["past"] // 2, c["past"], batch),
             "counts": _rand_int(g, max(1, n // 2), n, batch) if batch > 1 else None,
             "rope": _angles(c["past"] + n) if c["rope"] else None}
        s["k_new"], s["v_new"] = (torch.randn(batch, n, heads, D, generator=g, device=DEV).bfloat16() for _ in range(2))
    else:
        heads, width = c["kv_heads"], -(-c["len"] // page)
        s = {"table": _table(g, batch, width), "lens": c["len"]}
        if c["ragged"]:
            s["lens"] = _rand_int(g, min(c["len"], c["sq"]) if c["len"] < 1000 else c["len"] // 8, c["len"], batch)
            s["lens"][0] = c["len"]
        s["q"] = torch.randn(batch, c["sq"], c["heads"], D, generator=g, device=DEV).bfloat16()
    (s["k"], s["k_exp"]), (s["v"], s["v_exp"]) = (_pool(g, batch * width + 2, heads, page) for _ in range(2))
    if own:
        from diffsynth_engine_b200 import kvcache
        s["cache"] = kvcache.PagedKVCache(s["k"], s["v"], s["k_exp"], s["v_exp"])
    return {**s, "case": c}


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return {"rows4": _rows4, "append": _append, "attend": _attend}[state["case"]["op"]](state)


def _rows4(s):
    c = s["case"]
    if own:
        from diffsynth_engine_b200 import int4, ops
        return int4.gemv(s["weight"], s["x"], s["bias"], act_in=ops.ACT_SILU if c["silu"] else ops.ACT_NONE)
    q = torch.stack([s["codes"] & 15, s["codes"] >> 4], dim=-1).view(c["n"], c["k"]).float()
    at = torch.arange(c["k"], device=DEV) // c["group"]
    scale = s["scales"].float()[:, at]
    w = (q - 8).mul_(scale) if s["mins"] is None else q.mul_(scale).add_(s["mins"].float()[:, at])
    x = s["x"].float()
    if c["silu"]:
        x = x / (1 + torch.exp(-x))
    y = x @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(s["x"].dtype)


def _exponent(amax):
    """The least e in -64..64 with amax <= 448 * 2^e (448 = 0.875 * 2^9)."""
    m, e = torch.frexp(amax)
    e = torch.where(amax > 0, e - 9 + (m > 0.875).int(), torch.full_like(e, -64))
    return e.clamp(-64, 64)


def _e4m3(x, e):
    return torch.ldexp(x, -e).clamp(-448, 448).to(torch.float8_e4m3fn)


def _put(pages, exps, table, start, counts, x):
    """Appends rows x [B, n, H, 128] (fp32) to the blocks of one pool."""
    B, n, H, _ = x.shape
    T = pages.shape[2]
    J = min(table.shape[1], (n + T - 2) // T + 1)                # pages that n rows can touch
    first = start // T
    ids = table.gather(1, (first[:, None] + torch.arange(J, device=DEV)).clamp(max=table.shape[1] - 1).long()).long()
    slot = torch.arange(J * T, device=DEV) - (start % T)[:, None]     # row of x that belongs at each slot of those pages
    new = (slot >= 0) & (slot < counts[:, None])
    rows = x.gather(1, slot.clamp(0, n - 1).long()[:, :, None, None].expand(B, J * T, H, D))
    rows = rows.view(B, J, T, H, D).transpose(2, 3)
    new = new.view(B, J, 1, T, 1)
    touched = new.any(dim=3).view(B, J)
    size = torch.where(new & rows.isfinite(), rows.abs(), 0).amax(dim=(3, 4))
    begun = (torch.arange(J, device=DEV) == 0) & (start % T > 0)[:, None]            # pages that hold earlier rows
    was = exps[ids].int()
    e = torch.where(begun[:, :, None], torch.maximum(was, _exponent(size)), _exponent(size))
    held = pages.view(torch.uint8)[ids]
    old = (slot < 0).view(B, J, 1, T, 1)
    grown = _e4m3(held.view(torch.float8_e4m3fn).float(), (e - was)[..., None, None])
    put = torch.where(new, _e4m3(rows, e[..., None, None]).view(torch.uint8), torch.where(old, grown.view(torch.uint8), held))
    pages.view(torch.uint8)[ids[touched]] = put[touched]
    exps[ids[touched]] = e[touched].to(torch.int8)


def _append(s):
    if own:
        from diffsynth_engine_b200 import kvcache
        kvcache.append(s["cache"], s["k_new"], s["v_new"], s["table"], s["start"], s["counts"], rope=s["rope"])
    else:
        B, n, H, _ = s["k_new"].shape
        counts = torch.full((B,), n, dtype=torch.int32, device=DEV) if s["counts"] is None else s["counts"]
        k = s["k_new"].float()
        if s["rope"] is not None:
            at = (s["start"][:, None] + torch.arange(n, device=DEV)).clamp(max=s["rope"].shape[0] - 1).long()
            cos, sin = s["rope"][at][:, :, None].unbind(-1)
            a, b = k.view(B, n, H, 64, 2).unbind(-1)
            k = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).view(B, n, H, D)
        _put(s["k"], s["k_exp"], s["table"], s["start"], counts, k)
        _put(s["v"], s["v_exp"], s["table"], s["start"], counts, s["v_new"].float())
    # the cache itself: its e4m3 values, and the whole exponent of each block of them
    return {"k": s["k"], "v": s["v"], "k_exp": s["k_exp"], "v_exp": s["v_exp"]}


def _held(pages, exps, table, dtype):
    """The values of each sequence's pages in a row: [B, H, tokens, 128]."""
    at = table.long()
    x = pages.view(torch.uint8)[at].view(torch.float8_e4m3fn).to(dtype)
    x = x * torch.exp2(exps[at].to(dtype))[..., None, None]
    return x.transpose(1, 2).flatten(2, 3)


def _attend(s):
    c = s["case"]
    if own:
        from diffsynth_engine_b200 import kvcache
        return kvcache.attend(s["q"], s["cache"], s["table"], s["lens"], causal=c["causal"])
    B, sq, G = c["batch"], c["sq"], c["heads"] // c["kv_heads"]
    k, v = _held(s["k"], s["k_exp"], s["table"], torch.float32), _held(s["v"], s["v_exp"], s["table"], torch.float32)
    q = s["q"].float().view(B, sq, c["kv_heads"], G, D).permute(0, 2, 1, 3, 4).reshape(B, c["kv_heads"], sq * G, D)
    lens = torch.full((B,), s["lens"], device=DEV) if not c["ragged"] else s["lens"]
    at = torch.arange(k.shape[2], device=DEV)
    see = lens[:, None] - sq + 1 + torch.arange(sq, device=DEV) if c["causal"] else lens[:, None].expand(B, sq)
    hidden = (at >= see[:, :, None]).repeat_interleave(G, dim=1)[:, None]
    x = (q @ k.transpose(2, 3)).mul_(D ** -0.5).masked_fill_(hidden, -math.inf)
    x = x.sub_(x.amax(dim=-1, keepdim=True).clamp(min=-1e30)).exp_()
    y = (x @ v) / x.sum(dim=-1, keepdim=True).clamp(min=1e-30)
    return y.view(B, c["kv_heads"], sq, G, D).permute(0, 2, 1, 3, 4).reshape(B, sq, c["heads"], D).bfloat16()


# ------------------------------------------------------------------------------------------------ work and 64 bits
def work(case):
    c = case
    if c["op"] == "rows4":
        groups = -(-c["k"] // c["group"])
        size = c["rows"] * (c["n"] + c["k"]) * (2 if c["bf16"] else 4)
        return {"bytes": c["n"] * c["k"] / 2 + c["n"] * groups * (4 if c["mins"] else 2) + size + 4 * c["n"] * c["bias"],
                "flops": 2 * c["rows"] * c["n"] * c["k"]}
    if c["op"] == "append":
        rows = c["batch"] * c["n"] * (0.75 if c["batch"] > 1 else 1)           # ragged counts: between half and all
        return {"bytes": rows * (c["heads"] * 2 * D * 3 + (512 if c["rope"] else 0)), "flops": rows * c["heads"] * D * 6}
    low = (min(c["len"], c["sq"]) if c["len"] < 1000 else c["len"] // 8) if c["ragged"] else c["len"]
    keys = c["len"] + (c["batch"] - 1) * (low + c["len"]) / 2
    pairs = max(0.0, keys - c["batch"] * (c["sq"] - 1) / 2) if c["causal"] else keys
    return {"bytes": keys * c["kv_heads"] * 2 * D + c["batch"] * c["sq"] * c["heads"] * 4 * D,
            "flops": 4 * D * c["sq"] * c["heads"] * pairs}


def _round_e4m3(x):
    """The nearest e4m3 value of each x (64 bits), ties to the even one: steps of 2^(e - 3) from 2^e on, 2^-9 below 2^-6."""
    step = torch.ldexp(torch.ones_like(x), (torch.frexp(x)[1] - 1).clamp(min=-6) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _exact_blocks(pages, exps, table, start, counts, x, page):
    """One pool's values and exponents after an append, block by block."""
    pages, exps = pages.double(), exps.long()
    for b, (t0, n) in enumerate(zip(start, counts)):
        for j in range(t0 // page, (t0 + n - 1) // page + 1):
            lo, hi = max(t0, j * page), min(t0 + n, (j + 1) * page)
            p, rows = int(table[b][j]), x[b, lo - t0:hi - t0].transpose(0, 1)
            e = torch.ceil(torch.log2(rows.abs().amax(dim=(1, 2)) / 448)).long().clamp(-64, 64)
            if lo > j * page:
                e = torch.maximum(e, exps[p])
                fall = torch.exp2((exps[p] - e).double())[:, None, None]
                pages[p, :, :lo - j * page] = _round_e4m3(pages[p, :, :lo - j * page] * fall)
            exps[p] = e
            pages[p, :, lo - j * page:hi - j * page] = _round_e4m3(rows * torch.exp2(-e.double())[:, None, None])
    return pages, exps


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s, c = prepare(case, seed), case
    finally:
        own = was
    if c["op"] == "rows4":
        x, outs = s["x"].double(), []
        if c["silu"]:
            x = x * torch.sigmoid(x)
        cut = max(1, (1 << 28) // c["k"])
        for lo in range(0, c["n"], cut):
            part = s["codes"][lo:lo + cut]
            w = torch.empty(part.shape[0], c["k"], dtype=torch.float64, device=DEV)
            w[:, 0::2], w[:, 1::2] = part % 16, part // 16
            sc = s["scales"][lo:lo + cut].double().repeat_interleave(c["group"], dim=1)[:, :c["k"]]
            if c["mins"]:
                w = w * sc + s["mins"][lo:lo + cut].double().repeat_interleave(c["group"], dim=1)[:, :c["k"]]
            else:
                w = (w - 8) * sc
            y = torch.einsum("mk,nk->mn", x, w)
            outs.append(y if s["bias"] is None else y + s["bias"][lo:lo + cut].double())
        return torch.cat(outs, dim=1)
    if c["op"] == "append":
        start, counts = s["start"].tolist(), [c["n"]] * c["batch"] if s["counts"] is None else s["counts"].tolist()
        table, k = s["table"].tolist(), s["k_new"].double()
        if c["rope"]:
            z = torch.view_as_complex(k.view(*k.shape[:3], 64, 2))
            turn = torch.view_as_complex(s["rope"].double())
            at = [turn[t0:t0 + c["n"]] for t0 in start]
            k = torch.stack([torch.view_as_real(z[b] * at[b][:, None]).flatten(2) for b in range(c["batch"])])
        kp, ke = _exact_blocks(s["k"], s["k_exp"], table, start, counts, k, c["page"])
        vp, ve = _exact_blocks(s["v"], s["v_exp"], table, start, counts, s["v_new"].double(), c["page"])
        return {"k": kp, "v": vp, "k_exp": ke, "v_exp": ve}
    G, sq = c["heads"] // c["kv_heads"], c["sq"]
    out = torch.zeros(c["batch"], sq, c["heads"], D, dtype=torch.float64, device=DEV)
    lens = s["lens"].tolist() if c["ragged"] else [c["len"]] * c["batch"]
    for b, n in enumerate(lens):
        kv = [_held(p, e, s["table"][b:b + 1], torch.float64)[0, :, :n] for p, e in ((s["k"], s["k_exp"]), (s["v"], s["v_exp"]))]
        for h in range(c["heads"]):
            x = s["q"][b, :, h].double() @ kv[0][h // G].t() / math.sqrt(D)
            if c["causal"]:
                x = x + torch.full_like(x, -math.inf).triu(n - sq + 1)
            out[b, :, h] = torch.nan_to_num(torch.softmax(x, dim=-1), nan=0.0) @ kv[1][h // G]
    return out

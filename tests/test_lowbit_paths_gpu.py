"""What the library's own paths do with 4-bit weights and the 8-bit cache - the patched F.linear, the Flux modulation stack, the
Wan prompt cache - and the operators run together: projections in 4 bits, rotated appends and attention, token by token, eagerly
and as a replayed graph.

Tolerances: products as in test_int4_gpu (2e-6 in fp32); where two bf16 roundings of nearly the same value are compared, a bf16
step (2^-7) per value at most and half a step (2^-8) of the norm."""
import pytest
import torch

from oracle import gguf as G
from oracle import int4 as O4
from oracle import kvcache as OK
from oracle import ops as O

pytestmark = pytest.mark.gpu
synth = __import__("importlib").import_module("diffsynth_engine_b200.synth")


class _GGUF(torch.nn.Parameter):
    """A GGUF weight as the engine's own class presents it: raw bytes and a format tag."""

    def __new__(cls, raw, qtype):
        self = torch.Tensor._make_subclass(cls, raw, False)
        self.quant_dtype = qtype
        return self


@pytest.mark.parametrize("M", [1, 3, 32, 33, 130])
@pytest.mark.parametrize("source", ["Q4_0", "Q4_K", "Q6_K", "float"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float16])
def test_patched_linear(dsb, cuda_dev, M, source, dtype):
    from diffsynth_engine_b200 import int4, quant
    N, K = 72, 256
    layer = torch.nn.Linear(K, N).to(cuda_dev, torch.bfloat16)
    if source == "float":
        w = layer.weight.data.cpu()
    else:
        raw = G.random_blocks(source, N, K, seed=M)
        layer.weight = _GGUF(raw.to(cuda_dev), source)
    quant.enable_b200_linear(layer, "int4_group")
    assert isinstance(layer.weight, quant.Int4LinearWeight)
    if source in ("Q4_0", "Q4_K"):
        q, s, m = O4.gguf_fields(raw, source)
        W = O4.values(O4.pack(q), s, m, 32)
    else:
        if source == "Q6_K":
            w = dsb.ops.dequant_gguf(raw.to(cuda_dev), "Q6_K").cpu()
        W = O4.values(*O4.quantize(w, 32, True), 32)
    x = torch.randn(2 * M, 2 * K, device=cuda_dev).to(dtype)
    for rows in (x[:M, :K], x[::2, K:], x[:M, 1:K + 1], x[:M, :K].reshape(1, M, K)):
        with quant.b200_inference():
            got = layer(rows)
        assert got.shape == (*rows.shape[:-1], N) and got.dtype == dtype
        xr = rows.reshape(-1, K)
        if M > 32:      # through the bf16 expansion and the GEMM: operands and result rounded to bf16
            xr, W_ = xr.to(torch.bfloat16), W.to(torch.bfloat16)
        else:
            W_ = W
        ref = O4.linear(xr.cpu(), W_, layer.bias.detach().float().cpu())
        half = {torch.bfloat16: 2.0 ** -8, torch.float32: 2e-6 if M <= 32 else 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
        if M > 32 and dtype == torch.float16:
            half = 2.0 ** -8
        assert O.rel_l2(got.detach().reshape(-1, N).cpu(), ref) < half * 1.05      # (one rounding, and the fp32 sum under it)
    assert layer.weight.weight4.nbytes() <= 80 * K * 0.625        # 72 rows in five blocks of 16; 4 bits and 2 x 16 for 32 columns


def test_lora_keeps_4_bit_linears_unfused(dsb, cuda_dev):
    from diffsynth_engine_b200 import lora, quant

    class Lora(torch.nn.Linear):
        def __init__(self, *a):
            super().__init__(*a)
            self._lora_dict = {}

    layer = Lora(64, 32).to(cuda_dev)
    quant.enable_b200_linear(layer, "int4_group")
    assert lora.fuse_lora(layer) == 0


@pytest.mark.parametrize("graph", [False, True])
def test_flux_modulation_in_4_bits(dsb, cuda_dev, graph):
    """The modulation vector of the step is the 64-bit product of the quantised weights; the rest of the step is what the same
    vector gives."""
    from diffsynth_engine_b200.flux import FluxDiTEngine
    d, H = 256, 2
    shapes = synth.flux_dit_shapes(d=d, H=H, n_double=1, n_single=1, txt_dim=512, pooled_dim=96)
    w = {k: v.bfloat16().float() for k, v in synth.make_state_dict(shapes, seed=3).items()}
    lat, pe = synth.randn((1, 16, 16, 16), 1).bfloat16().to(cuda_dev), synth.randn((1, 32, 512), 2).bfloat16().to(cuda_dev)
    pooled, t, g = synth.randn((1, 96), 3).to(cuda_dev), torch.tensor([500.0], device=cuda_dev), torch.tensor([3.5], device=cuda_dev)
    eng = FluxDiTEngine(dict(w), fmt="bf16", device=cuda_dev, n_double=1, n_single=1, num_heads=H, mod_fmt="int4_group")
    eng.prepare(32, 16, 16, 512, 96)
    eng.set_inputs(lat, t, pe, pooled, g)
    if graph:
        eng.capture()
    out = eng.step().clone()
    names = ["blocks.0.norm1_a.linear", "blocks.0.norm1_b.linear", "single_blocks.0.norm.linear", "final_norm_out.linear"]
    W = torch.cat([O4.values(*O4.quantize(w[n + ".weight"], 32, True), 32) for n in names])
    bias = torch.cat([w[n + ".bias"] for n in names])
    ref = O4.linear(eng._bufs["cond"].cpu()[None], W, bias, act_in=torch.nn.functional.silu)[0]
    assert O.rel_l2(eng._bufs["modv"].cpu(), ref) < 2e-6
    # an engine whose modulation weights are the 4-bit ones, expanded: they are rounded to bf16 there (2^-9 rms each, independent)
    w2 = dict(w)
    for n in names:
        w2[n + ".weight"] = O4.values(*O4.quantize(w[n + ".weight"], 32, True), 32).float()
    eng2 = FluxDiTEngine(w2, fmt="bf16", device=cuda_dev, n_double=1, n_single=1, num_heads=H)
    out2 = eng2(lat, t, pe, pooled, g)
    assert O.rel_l2(out.float(), out2.float()) < 2.0 ** -7
    dsb.ops.check_status(0)
    with pytest.raises(ValueError):
        FluxDiTEngine(dict(w), fmt="bf16", device=cuda_dev, n_double=1, n_single=1, num_heads=H, mod_fmt="fp8_tensor")


@pytest.mark.parametrize("grid,image", [((3, 8, 10), False), ((3, 8, 10), True), ((3, 20, 24), True)])
def test_wan_prompt_cache_in_8_bits(dsb, cuda_dev, monkeypatch, grid, image):
    """The engine with its prompt's keys and values in the 8-bit cache is the engine whose bf16 ones have been rounded like that:
    60 queries (attention over the pages) and 360 (dense attention over rows read back, bit for bit the same)."""
    from diffsynth_engine_b200 import kvcache
    from diffsynth_engine_b200.wan import WanDiTEngine
    monkeypatch.setattr(kvcache, "dense_pays", lambda batch, queries, *sizes: queries >= kvcache.DENSE_QUERIES)
    L, H, d = 2, 2, 256
    more = dict(in_dim=36, has_image_input=True) if image else {}
    w = {k: v.bfloat16().float() for k, v in synth.make_state_dict(
        synth.wan_dit_shapes(d=d, ffn=512, num_layers=L, text_dim=64, **more), seed=5).items()}
    x = synth.randn((1, 16, *grid), 1).bfloat16().to(cuda_dev)
    ctx, t = synth.randn((1, 70, 64), 2).bfloat16().to(cuda_dev), torch.tensor([417.0], device=cuda_dev)
    extra = (synth.randn((1, 257, 1280), 3).bfloat16().to(cuda_dev), synth.randn((1, 20, *grid), 4).bfloat16().to(cuda_dev)) if image else ()
    outs = []
    for fmt in ("bf16", "e4m3"):
        eng = WanDiTEngine(dict(w), fmt="bf16", device=cuda_dev, num_layers=L, num_heads=H, ckv_fmt=fmt)
        out = eng(x, ctx, t, *extra)
        if fmt == "bf16":
            plain = out
            ckv, n_img = eng._bufs["ckv"], eng._bufs["n_img"]
            for li in range(L):
                for lo, hi in ((0, n_img), (n_img, n_img + 70)):
                    if hi == lo:
                        continue
                    c = kvcache.PagedKVCache.empty(8, H, 64, cuda_dev)
                    pages = torch.arange(8, dtype=torch.int32, device=cuda_dev)[None]
                    kvcache.append(c, ckv[li, 0, lo:hi].view(1, -1, H, 128), ckv[li, 1, lo:hi].view(1, -1, H, 128), pages, 0)
                    for i, r in enumerate(kvcache.read(c, pages, hi - lo)):
                        ckv[li, i, lo:hi] = r.view(hi - lo, d)
        else:
            assert eng._bufs["ckv8"].k.numel() < 2 * ckv[:, 0].numel()          # (whole pages)
        outs.append(eng(x, ctx, t, *extra))                                    # the same prompt: its keys and values are kept
    dsb.ops.check_status(0)
    a, b = (o.float() for o in outs)
    assert not torch.equal(a, plain.float()) and O.rel_l2(b, plain.float()) < 2.0 ** -4   # e4m3 half a step, diluted
    if grid[1] * grid[2] * grid[0] // 4 >= kvcache.DENSE_QUERIES:
        assert torch.equal(a, b)
    else:
        assert O.rel_l2(b, a) < 2.0 ** -7
    with pytest.raises(ValueError):
        WanDiTEngine(dict(w), fmt="bf16", device=cuda_dev, num_layers=L, num_heads=H, ckv_fmt="int8")


@pytest.mark.parametrize("captured", [False, True])
def test_tokens_one_by_one(dsb, cuda_dev, captured):
    """Three sequences of different lengths grow by 20 tokens: 4-bit q, k and v projections of the new token, rotated append, causal
    attention over the cache, 4-bit output projection.  Each step against the 64-bit restatement of the same cache."""
    from diffsynth_engine_b200 import int4, kvcache
    B, H, Hk, T, d, steps = 3, 4, 2, 16, 512, 20
    g = torch.Generator().manual_seed(1)
    W = {n: torch.randn(rows, cols, generator=g) * cols ** -0.5 for n, rows, cols in
         (("q", H * 128, d), ("k", Hk * 128, d), ("v", Hk * 128, d), ("o", d, H * 128))}
    host = {n: O4.quantize(w, 64, True) for n, w in W.items()}
    dev = {n: int4.from_codes(*(t.to(cuda_dev) for t in h), group=64) for n, h in host.items()}
    Wv = {n: O4.values(*h, 64) for n, h in host.items()}
    f = 10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)
    ang = torch.outer(torch.arange(64, dtype=torch.float64), f)
    rope = torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()
    table = torch.randperm(3 * B + 2, generator=g)[:3 * B].view(B, 3).int()
    start0 = torch.tensor([0, 9, 27], dtype=torch.int32)
    past = [torch.randn(B, 27, Hk, 128, generator=g).bfloat16() for _ in range(2)]
    cache = kvcache.PagedKVCache.empty(3 * B + 2, Hk, T, cuda_dev)
    pages = [torch.zeros(3 * B + 2, Hk, T, 128, dtype=torch.float64) for _ in range(2)]
    exps = [torch.zeros(3 * B + 2, Hk, dtype=torch.int8) for _ in range(2)]
    rope_d, table_d = rope.to(cuda_dev), table.to(cuda_dev)
    kvcache.append(cache, past[0].to(cuda_dev), past[1].to(cuda_dev), table_d, 0, start0.to(cuda_dev), rope=rope_d)
    for i in (0, 1):
        rows = past[i].float()
        rows = torch.stack([OK.rotate(r, rope, 0) for r in rows]) if i == 0 else rows
        OK.append(pages[i], exps[i], table, [0] * B, start0, rows)
    x_d, start, lens = torch.zeros(B, d, dtype=torch.bfloat16, device=cuda_dev), start0.to(cuda_dev), (start0 + 1).to(cuda_dev)
    buf = {n: torch.zeros(B, W[n].shape[0], dtype=torch.bfloat16, device=cuda_dev) for n in "qkvo"}
    att = torch.zeros(B, 1, H, 128, dtype=torch.bfloat16, device=cuda_dev)

    def step():
        for n in "qkv":
            int4.gemv(dev[n], x_d, out=buf[n])
        kvcache.append(cache, buf["k"].view(B, 1, Hk, 128), buf["v"].view(B, 1, Hk, 128), table_d, start, rope=rope_d)
        kvcache.attend(buf["q"].view(B, 1, H, 128), cache, table_d, lens, causal=True, out=att)
        int4.gemv(dev["o"], att.view(B, H * 128), out=buf["o"])
        start.add_(1)
        lens.add_(1)

    run = step
    if captured:
        side = torch.cuda.Stream(cuda_dev)
        with torch.cuda.stream(side):
            step()                      # (warms up; the first graph step writes the same token again)
            start.copy_(start0)
            lens.copy_(start0 + 1)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
        run = graph.replay
    for s in range(steps):
        x = torch.randn(B, d, generator=g).bfloat16()
        x_d.copy_(x)
        run()
        torch.cuda.synchronize()
        for n in "qkv":
            assert O.rel_l2(buf[n].cpu(), O4.linear(x, Wv[n])) < 2.0 ** -8
        at = (start0 + s).tolist()
        for i, n in enumerate("kv"):
            rows = buf[n].cpu().float().view(B, 1, Hk, 128)
            if i == 0:
                rows = torch.stack([OK.rotate(rows[b], rope, at[b]) for b in range(B)])
            OK.append(pages[i], exps[i], table, at, [1] * B, rows)
        ref = OK.attend(buf["q"].cpu().view(B, 1, H, 128), pages, exps, table, [a + 1 for a in at], True)
        assert O.rel_l2(att.cpu(), ref) < 2.0 ** -8 + 2.0 ** -11
        assert O.rel_l2(buf["o"].cpu(), O4.linear(att.cpu().view(B, H * 128), Wv["o"])) < 2.0 ** -8
    for got, want, e, ew in zip((cache.k, cache.v), pages, (cache.k_exp, cache.v_exp), exps):
        for b in range(B):
            n = int(start0[b]) + steps
            idx = table[b, : -(-n // T)].long()
            assert torch.equal(e.cpu()[idx], ew[idx])
            have = got.cpu()[idx].double().transpose(1, 2).reshape(-1, Hk, 128)[:n]
            assert torch.equal(have, want[idx].transpose(1, 2).reshape(-1, Hk, 128)[:n])
    dsb.ops.check_status(0)


def test_streams_and_two_graphs(dsb, cuda_dev):
    """Calls on two streams at once, and two captured graphs replayed together, each with its own workspace: the results of calls
    that run alone."""
    from diffsynth_engine_b200 import int4, kvcache
    g = torch.Generator(device=cuda_dev).manual_seed(0)
    caches, tables, qs, ws, xs = [], [], [], [], []
    for i in range(2):
        c = kvcache.PagedKVCache.empty(200, 2, 64, cuda_dev)
        rows = [torch.randn(1, 12000, 2, 128, generator=g, device=cuda_dev).bfloat16() for _ in range(2)]
        tables.append(torch.randperm(200, generator=g, device=cuda_dev)[None, :188].int().contiguous())
        kvcache.append(c, *rows, tables[-1], 0)
        caches.append(c)
        qs.append(torch.randn(1, 3, 8, 128, generator=g, device=cuda_dev).bfloat16())
        ws.append(int4.quantize(torch.randn(4096, 1024, generator=g, device=cuda_dev)))
        xs.append(torch.randn(4, 1024, generator=g, device=cuda_dev))
    lens = torch.tensor([11999], dtype=torch.int32, device=cuda_dev)

    def work(i):
        return kvcache.attend(qs[i], caches[i], tables[i], lens, causal=True), int4.gemv(ws[i], xs[i])

    want = [work(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(cuda_dev) for _ in range(2)]
    for _ in range(5):
        got = []
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got.append([work(i) for _ in range(10)])
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(a, b) for r in got[i] for a, b in zip(r, want[i]))
    graphs, outs = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=streams[i]):
            outs.append(work(i))
        graphs.append(graph)
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(outs[i], want[i]))
    dsb.ops.check_status(0)

"""4-bit weights with group scales: quantisation, layout, products and the entry points that use them.

Tolerances.  Products and sums are fp32: a sum of n rounded terms is off by at most about n * 2^-24 of the sum of magnitudes in
the worst case and sqrt(n) * 2^-24 (n = 4304: 4e-6) of it when the roundings are independent; relative to the result's own norm
(a random sum's norm is the magnitudes' over sqrt(n), so the two cancel) that is a few times 2^-24 per term: 2e-6 is asked.
A bf16 output adds half a step, at most 2^-8 of a value: 2^-8 of the norm is asked.
SiLU's exponential and division are good to about 2^-21: 2e-6 covers them too; GELU (erf) likewise."""
import pytest
import torch

from oracle import gguf as G
from oracle import int4 as O4
from oracle import ops as O

pytestmark = pytest.mark.gpu


def _weight(N, K, group, mins, seed):
    g = torch.Generator().manual_seed(seed)
    groups = -(-K // group)
    codes = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8)
    scales = (torch.rand(N, groups, generator=g) * 0.01 + 0.001).half()
    m = (torch.randn(N, groups, generator=g) * 0.02 - 0.03).half() if mins else None
    return codes, scales, m


def _on(dev, *ts):
    return [None if t is None else t.to(dev) for t in ts]


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("mins", [False, True])
@pytest.mark.parametrize("N,K", [(1, 2), (16, 64), (17, 66), (40, 160), (130, 322)])
def test_layout_is_exact(dsb, cuda_dev, N, K, group, mins):
    """What the laid-out weight stands for is the fp32 value of its codes, rounded once to bf16."""
    from diffsynth_engine_b200 import int4
    c, s, m = _weight(N, K, group, mins, N + K)
    w = int4.from_codes(*_on(cuda_dev, c, s, m), group=group)
    want = O4.values(c, s, m, group, torch.float32).bfloat16()
    assert torch.equal(int4.dequant(w).cpu(), want)
    wide = torch.full((N, K + 8), 7.0, dtype=torch.bfloat16, device=cuda_dev)
    int4.dequant(w, out=wide[:, :K])
    assert torch.equal(wide[:, :K].cpu(), want) and bool((wide[:, K:] == 7).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("group,asym", [(32, False), (64, True), (128, False), (128, True)])
def test_quantize_is_exact(dsb, cuda_dev, dtype, group, asym):
    from diffsynth_engine_b200 import int4
    W = (torch.randn(70, 338, generator=torch.Generator().manual_seed(1)) * 0.05).to(dtype)
    W[3] = 0
    W[4, :200] = 0.25       # constant groups
    W[5] *= 1e9             # scales that leave fp16 saturate
    c, s, m = O4.quantize(W, group, asym)
    gc, gs, gm = int4.quantize_codes(W.to(cuda_dev), group, asym)
    assert torch.equal(gs.cpu(), s) and torch.equal(gc.cpu(), c)
    assert (m is None) == (gm is None) and (m is None or torch.equal(gm.cpu(), m))


@pytest.mark.parametrize("qtype", ["Q4_0", "Q4_1", "Q4_K"])
def test_gguf_blocks_are_taken_over(dsb, cuda_dev, qtype):
    from diffsynth_engine_b200 import int4
    N, K = 21, 512
    raw = G.random_blocks(qtype, N, K, seed=5)
    q, s, m = O4.gguf_fields(raw, qtype)
    c, gs, gm = int4.gguf_codes(raw.to(cuda_dev), qtype)
    assert torch.equal(O4.unpack(c.cpu()), q.long())
    assert torch.equal(gs.cpu().view(torch.int16), s.contiguous().view(torch.int16))
    assert (m is None) == (gm is None) and (m is None or torch.equal(gm.cpu(), m))
    w = int4.from_gguf(raw.to(cuda_dev), qtype)
    want = O4.values(O4.pack(q), s, m, 32, torch.float32).bfloat16()
    assert torch.equal(int4.dequant(w).cpu(), want)
    # next to the 16-bit expansion of the same blocks, which rounds scales and products to bf16: 2^-8 each of up to three
    ref = dsb.ops.dequant_gguf(raw.to(cuda_dev), qtype).float().cpu()
    assert float((want.float() - ref).abs().max()) <= 3 * 2.0 ** -8 * float(ref.abs().max())


SHAPES = [(1, 2), (7, 34), (16, 64), (48, 256), (33, 130), (129, 1026), (768, 256), (1000, 4304), (5120, 512), (20001, 192)]


@pytest.mark.parametrize("N,K", SHAPES)
@pytest.mark.parametrize("M", [1, 2, 5, 8, 9, 17, 32])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_product(dsb, cuda_dev, N, K, M, dtype):
    from diffsynth_engine_b200 import int4
    group = (32, 64, 128)[(N + M) % 3]
    c, s, m = _weight(N, K, group, (N + K + M) % 2 == 1, N + M)
    w = int4.from_codes(*_on(cuda_dev, c, s, m), group=group)
    g = torch.Generator().manual_seed(M)
    x, b = torch.randn(M, K, generator=g).to(dtype), torch.randn(N, generator=g)
    y = int4.gemv(w, x.to(cuda_dev), b.to(cuda_dev))
    ref = O4.linear(x, O4.values(c, s, m, group), b)
    assert y.dtype == dtype and O.rel_l2(y.cpu(), ref) < (2e-6 if dtype == torch.float32 else 2.0 ** -8)
    f = int4.gemv(w, x.to(cuda_dev), b.to(cuda_dev), out=torch.empty(M, N, device=cuda_dev))
    assert O.rel_l2(f.cpu(), ref) < 2e-6
    assert torch.equal(f.to(dtype), y)                                           # one rounding, of the same value
    assert torch.equal(int4.gemv(w, x.to(cuda_dev), b.to(cuda_dev)), y)            # and the same every time


def test_product_strides_activations_and_accumulation(dsb, cuda_dev):
    from diffsynth_engine_b200 import int4
    ops = dsb.ops
    c, s, m = _weight(200, 194, 64, True, 3)
    w = int4.from_codes(*_on(cuda_dev, c, s, m), group=64)
    W = O4.values(c, s, m, 64)
    g = torch.Generator().manual_seed(0)
    big, b = torch.randn(9, 401, generator=g), torch.randn(200, generator=g)
    acts = {ops.ACT_NONE: None, ops.ACT_SILU: torch.nn.functional.silu, ops.ACT_GELU: torch.nn.functional.gelu,
            ops.ACT_GELU_TANH: lambda t: torch.nn.functional.gelu(t, approximate="tanh")}
    for dtype in (torch.float32, torch.bfloat16):
        d = big.to(dtype).to(cuda_dev)
        for x in (d[:3, 1:195], d[::2, 207:], d[4, 3:197]):
            for a_in in (ops.ACT_NONE, ops.ACT_SILU):
                for a_out in acts:
                    out = torch.full((*x.shape[:-1], 203), 3.0, device=cuda_dev)
                    y = out[..., :200]
                    int4.gemv(w, x, b.to(cuda_dev), act_in=a_in, act_out=a_out, out=y)
                    ref = O4.linear(x.cpu(), W, b, acts[a_in], acts[a_out])
                    assert O.rel_l2(y.cpu(), ref) < 2e-6
                    assert bool((out[..., 200:] == 3).all())
                    int4.gemv(w, x, b.to(cuda_dev), act_in=a_in, act_out=a_out, out=y, accumulate=True)
                    assert O.rel_l2(y.cpu(), 2 * ref) < 2e-6
    # large, tiny and zero rows keep their own scale; a row that is not finite touches no other
    x = torch.randn(6, 194, generator=g)
    x[0] *= 1e30
    x[1] *= 1e-30
    x[2] = 0
    x[3, 7] = float("nan")
    x[4, 9] = float("inf")
    y = int4.gemv(w, x.to(cuda_dev)).cpu()
    ref = O4.linear(x, W)
    for r in (0, 1, 5):
        assert O.rel_l2(y[r], ref[r]) < 2e-6
    assert bool((y[2] == 0).all()) and bool(y[3].isnan().all())
    assert not bool(y[4][W[:, 9] != 0].isfinite().any())


@pytest.mark.parametrize("M,K,dtype", [(1, 70002, torch.float32), (16, 70002, torch.bfloat16), (8, 120000, torch.float32)])
def test_long_rows(dsb, cuda_dev, M, K, dtype):
    """Rows that do not fit the shared memory of a CTA, or of a cluster, all at once."""
    from diffsynth_engine_b200 import int4
    c, s, m = _weight(33, K, 128, True, K)
    w = int4.from_codes(*_on(cuda_dev, c, s, m), group=128)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).to(dtype)
    y = int4.gemv(w, x.to(cuda_dev), out=torch.empty(M, 33, device=cuda_dev))
    assert O.rel_l2(y.cpu(), O4.linear(x, O4.values(c, s, m, 128))) < 4e-6        # (sixteen times the terms of the other shapes)


def test_offsets_pass_32_bits(dsb, cuda_dev):
    """2.5 GB of codes: rows at the end, and a dequantised row there."""
    from diffsynth_engine_b200 import int4
    N, K = 1200016, 4096
    g = torch.Generator(device=cuda_dev).manual_seed(0)
    codes = torch.randint(0, 256, (N, K // 2), generator=g, device=cuda_dev, dtype=torch.uint8)
    scales = torch.rand(N, K // 64, generator=g, device=cuda_dev).half()
    w = int4.from_codes(codes, scales, group=64)
    x = torch.randn(1, K, generator=g, device=cuda_dev)
    y = int4.gemv(w, x)[0]
    for lo in (0, N // 2, N - 40):
        ref = O4.linear(x.cpu(), O4.values(codes[lo:lo + 40].cpu(), scales[lo:lo + 40].cpu(), None, 64))[0]
        assert O.rel_l2(y[lo:lo + 40].cpu(), ref) < 2e-6
    del y
    full = int4.dequant(w)
    assert torch.equal(full[-3:].cpu(), O4.values(codes[-3:].cpu(), scales[-3:].cpu(), None, 64, torch.float32).bfloat16())


def test_refusals(dsb, cuda_dev):
    from diffsynth_engine_b200 import int4
    c, s, m = _on(cuda_dev, *_weight(32, 64, 32, True, 0))
    w = int4.from_codes(c, s, m)
    x = torch.zeros(2, 64, device=cuda_dev)
    for bad in (lambda: int4.from_codes(c, s, m, group=16), lambda: int4.from_codes(c, s[:, :1], m), lambda: int4.from_codes(c.int(), s),
                lambda: int4.from_codes(c, s.float()), lambda: int4.from_codes(c.cpu(), s.cpu()), lambda: int4.quantize(x[:, :63]),
                lambda: int4.quantize(x.half()), lambda: int4.from_gguf(c, "Q6_K"), lambda: int4.from_gguf(c[:, :17], "Q4_0"),
                lambda: int4.gemv(w, x[:, :62]), lambda: int4.gemv(w, x.half()), lambda: int4.gemv(w, x.cpu()),
                lambda: int4.gemv(w, torch.zeros(33, 64, device=cuda_dev)), lambda: int4.gemv(w, x, torch.zeros(31, device=cuda_dev)),
                lambda: int4.gemv(w, x, act_in=dsb.ops.ACT_GELU), lambda: int4.gemv(w, x, act_out=9), lambda: int4.gemv(w, x, accumulate=True),
                lambda: int4.gemv(w, x, out=torch.zeros(2, 31, device=cuda_dev)), lambda: int4.gemv(w, x.expand(2, 64)[:1].expand(2, 64)),
                lambda: int4.gemv(w, x, out=torch.zeros(1, 32, device=cuda_dev).expand(2, 32)),
                lambda: int4.gemv(c, x), lambda: int4.stack([w, int4.from_codes(c, s)]), lambda: int4.dequant(w, out=x)):
        with pytest.raises(dsb.DsbError):
            bad()
    assert int4.gemv(w, x[:0]).shape == (0, 32)

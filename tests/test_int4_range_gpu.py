"""4-bit weights at the borders of their calls: rows shared in memory, activations that lie far apart or are not finite, Linears
of odd widths.

Tolerances as in test_int4_gpu: 2e-6 of the norm for fp32 results; half a bf16 step, 2^-8, where operands or results are rounded to
bf16."""
import pytest
import torch

from oracle import int4 as O4
from oracle import ops as O

pytestmark = pytest.mark.gpu


def _weight(N, K, group, mins, seed):
    g = torch.Generator().manual_seed(seed)
    groups = -(-K // group)
    codes = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8)
    scales = (torch.rand(N, groups, generator=g) * 0.01 + 0.001).half()
    return codes, scales, (torch.randn(N, groups, generator=g) * 0.02 - 0.03).half() if mins else None


def _on(dev, *ts):
    return [None if t is None else t.to(dev) for t in ts]


@pytest.mark.parametrize("group,mins", [(32, True), (128, False)])
def test_rows_shared_by_broadcasting(dsb, cuda_dev, group, mins):
    """Codes, scales and minima, or a weight, whose rows are one row of memory: the same as with rows of their own."""
    from diffsynth_engine_b200 import int4
    N, K = 50, 258
    c, s, m = _on(cuda_dev, *_weight(1, K, group, mins, 5))
    wide = [None if t is None else t.expand(N, -1) for t in (c, s, m)]
    got = int4.dequant(int4.from_codes(*wide, group=group))
    want = int4.dequant(int4.from_codes(*(None if t is None else t.contiguous() for t in wide), group=group))
    assert torch.equal(got, want) and torch.equal(got.cpu(), O4.values(*(None if t is None else t.cpu() for t in wide), group, torch.float32).bfloat16())
    W = torch.randn(1, K, generator=torch.Generator().manual_seed(3)).to(cuda_dev).expand(N, K)
    for a, b in zip(int4.quantize_codes(W, group, mins), int4.quantize_codes(W.contiguous(), group, mins)):
        assert (a is None) == (b is None) and (a is None or torch.equal(a, b))


@pytest.mark.parametrize("outlier", [2.0 ** 20, 2.0 ** 27])
@pytest.mark.parametrize("N,K,M", [(64, 256, 1), (200, 1026, 3), (3000, 320, 9)])
@pytest.mark.parametrize("silu", [False, True])
def test_small_activations_beside_an_outlier(dsb, cuda_dev, outlier, N, K, M, silu):
    """Outputs whose weight is zero at a row's outlier are made of its small activations alone, and as good as they would be without it."""
    from diffsynth_engine_b200 import int4, ops
    c, s, _ = _weight(N, K, 32, False, K)
    at = K // 2 & ~1
    c[:, at // 2] = c[:, at // 2] & 0xf0 | 8
    w = int4.from_codes(*_on(cuda_dev, c, s), group=32)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(M))
    x[:, at] = outlier
    y = int4.gemv(w, x.to(cuda_dev), act_in=ops.ACT_SILU if silu else ops.ACT_NONE).cpu()
    x[:, at] = 0
    ref = O4.linear(x, O4.values(c, s, None, 32), act_in=torch.nn.functional.silu if silu else None)
    for got, want in zip(y, ref):
        assert O.rel_l2(got, want) < 2e-6


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("mins", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,K", [(70, 192), (200, 1026), (5000, 320)])
def test_infinite_activations(dsb, cuda_dev, group, mins, dtype, N, K):
    """A row with infinities gives what the products of its weights give: infinities of the weights' signs, NaN where the weight is
    zero or the signs disagree; the other rows are as ever."""
    from diffsynth_engine_b200 import int4, ops
    c, s, m = _weight(N, K, group, mins, N + K)
    if mins:
        s[3], m[3] = 0.0078125, -0.015625           # code 2 is a zero
    w = int4.from_codes(*_on(cuda_dev, c, s, m), group=group)
    W = O4.values(c, s, m, group)
    x = torch.randn(12, K, generator=torch.Generator().manual_seed(1))
    inf = float("inf")
    x[0, 5], x[2, K - 1], x[3, 40], x[3, 41] = inf, -inf, inf, inf
    x[4, 7], x[4, K - 2], x[5, 0], x[5, 33], x[5, K // 2] = inf, -inf, -inf, -inf, -inf
    x[7, 9], x[7, 10] = inf, float("nan")
    x[9, ::3] = inf
    x = x.to(dtype)
    for act, f in ((ops.ACT_NONE, None), (ops.ACT_SILU, lambda t: torch.where(t == -inf, 0.0, t * torch.sigmoid(t)))):
        y = int4.gemv(w, x.to(cuda_dev), act_in=act, out=torch.empty(12, N, device=cuda_dev)).cpu()
        if f is not None:       # (the activation of -infinity is NaN or 0, as 0 * -inf is taken)
            keep = ~(x == -inf).any(1)
        else:
            keep = torch.ones(12, dtype=torch.bool)
        ref = O4.linear(x, W, act_in=f)
        y, ref = y[keep], ref[keep]
        assert torch.equal(y.isnan(), ref.isnan())
        assert torch.equal(y.isposinf(), ref.isposinf()) and torch.equal(y.isneginf(), ref.isneginf())
        rows = ref.isfinite().all(1)
        assert rows.sum() >= 5 and O.rel_l2(y[rows], ref[rows]) < 2e-6


@pytest.mark.parametrize("N,K", [(72, 256), (70, 256), (72, 258), (70, 258), (1, 2), (9, 34)])
@pytest.mark.parametrize("M", [32, 33, 140])
@pytest.mark.parametrize("bias", [False, True])
def test_linears_of_odd_widths(dsb, cuda_dev, N, K, M, bias):
    """A Linear that 32 rows can go through takes any number."""
    from diffsynth_engine_b200 import quant
    layer = torch.nn.Linear(K, N, bias=bias).to(cuda_dev)
    W = O4.values(*O4.quantize(layer.weight.data.cpu(), 32, True), 32)
    quant.enable_b200_linear(layer, "int4_group")
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.randn(2 * M, K + 1, device=cuda_dev).to(dtype)
        for rows in (x[:M, :K], x[::2, 1:], x[:M, :K].reshape(1, M, K), x[:1, :K].expand(M, K)):
            with quant.b200_inference():
                got = layer(rows)
            assert got.shape == (*rows.shape[:-1], N) and got.dtype == dtype and got.is_contiguous()
            xr, W_ = rows.reshape(-1, K).cpu(), W
            if M > 32:
                xr, W_ = xr.bfloat16(), W.bfloat16()
            ref = O4.linear(xr, W_, layer.bias.detach().cpu() if bias else None)
            tol = 2e-6 if M <= 32 and dtype == torch.float32 else 2.0 ** -8 * 1.05
            assert O.rel_l2(got.detach().reshape(-1, N).cpu(), ref) < tol

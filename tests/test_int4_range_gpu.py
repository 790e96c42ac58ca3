"""4-bit weights at the borders of their calls: rows shared in memory, activations that lie far apart.

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

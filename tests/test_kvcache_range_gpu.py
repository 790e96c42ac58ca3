"""Attention over the paged cache where its numbers lie far apart: value blocks of one sequence with very different exponents, one
key far above a flat tail, and exponents that no append has written.

Tolerance: the output is rounded to bf16 (2^-8 of a value at most, 2^-8 / sqrt 3 rms), and each probability to 11 bits (2^-11), as in
test_kvcache_gpu: 2^-8 + 2^-11 of each row's own norm, and per value 2^-8 of it plus 2^-10 of the largest value that the row
averages with any weight to speak of."""
import pytest
import torch

from oracle import kvcache as OK
from oracle import ops as O

pytestmark = pytest.mark.gpu


def _filled(dev, B, Hk, T, lens, k, v, table):
    from diffsynth_engine_b200 import kvcache
    cache = kvcache.PagedKVCache.empty(int(table.max()) + 1, Hk, T, dev)
    kvcache.append(cache, k.to(dev), v.to(dev), table.to(dev), 0, torch.tensor(lens, dtype=torch.int32, device=dev))
    return cache


def _held(cache):
    return [cache.k.cpu().double(), cache.v.cpu().double()], [cache.k_exp.cpu(), cache.v_exp.cpu()]


def _rows_near(out, ref, top):
    out = out.double().cpu()
    assert bool(out.isfinite().all())
    for got, want in zip(out.reshape(-1, 128), ref.reshape(-1, 128)):
        assert O.rel_l2(got, want) < 2.0 ** -8 + 2.0 ** -11
        assert float(((got - want).abs() - want.abs() * 2.0 ** -8).max()) <= 2.0 ** -10 * top


@pytest.mark.parametrize("T", [16, 64])
@pytest.mark.parametrize("B,Sq,H,Hk,lens,causal", [(1, 1, 1, 1, [200], False), (2, 3, 8, 2, [256, 130], True), (1, 40, 4, 2, [230], False),
                                                   (1, 2, 4, 2, [3000], False), (3, 1, 4, 4, [900, 1500, 33], True), (1, 70, 2, 1, [1200], True)])
@pytest.mark.parametrize("big", [1e4, 1e6, 1e8, 1e18])
def test_a_large_value_that_nobody_looks_at(dsb, cuda_dev, T, B, Sq, H, Hk, lens, causal, big):
    """One token of a sequence has a large value and no weight: every row is an average of the values around 0.02."""
    from diffsynth_engine_b200 import kvcache
    W = -(-max(lens) // T)
    table = torch.randperm(B * W, generator=torch.Generator().manual_seed(3)).view(B, W).int()
    g = torch.Generator().manual_seed(T + Sq)
    n = max(lens)
    q, k = torch.randn(B, Sq, H, 128, generator=g), torch.randn(B, n, Hk, 128, generator=g)
    v = (torch.randn(B, n, Hk, 128, generator=g) * 0.005 + 0.02)
    q[..., 0] = 30.0
    k[..., 0] = 0.0
    k[:, 21, :, 0] = -300.0              # a score of about -800: its weight is 0 in any arithmetic
    v[:, 21] *= big
    q, k, v = q.bfloat16(), k.bfloat16(), v.bfloat16()
    cache = _filled(cuda_dev, B, Hk, T, lens, k, v, table)
    kv, ex = _held(cache)
    ref = OK.attend(q, kv, ex, table, lens, causal)
    lt = torch.tensor(lens, dtype=torch.int32, device=cuda_dev)
    top = 0.05                           # (the largest of the values that have a weight)
    out = kvcache.attend(q.to(cuda_dev), cache, table.to(cuda_dev), lt, causal=causal)
    _rows_near(out, ref, top)
    assert torch.equal(out, kvcache.attend(q.to(cuda_dev), cache, table.to(cuda_dev), lt, causal=causal))


@pytest.mark.parametrize("exps", [[-64, 64, -64, 64, -64, 64, -64, 64], [64, -64, -64, -64, -64, -64, -64, -64], [-64] * 7 + [64], [0, -30, 20, -64, 64, 3, -3, 12]])
@pytest.mark.parametrize("T,copies", [(16, 1), (32, 1), (64, 1), (16, 20), (64, 12)])
def test_weight_on_blocks_of_any_exponent(dsb, cuda_dev, exps, T, copies):
    """Query i looks at the keys of every eighth page from i on, evenly: it gets their values with their own precision, whatever the others hold."""
    from diffsynth_engine_b200 import kvcache
    P = 8
    g = torch.Generator().manual_seed(T)
    v = (torch.rand(P, 2, T, 128, generator=g) * 200 + 200).to(torch.float8_e4m3fn)
    k = torch.zeros(P, 2, T, 128)
    for j in range(P):
        k[j, :, :, j] = 16.0
    q = torch.zeros(1, P, 4, 128)
    for i in range(P):
        q[0, i, :, i] = 60.0            # a score of 960 against 0: the other pages have no weight
    k, q = k.to(torch.float8_e4m3fn), q.bfloat16()
    ex = [torch.zeros(P, 2, dtype=torch.int8), torch.tensor(exps, dtype=torch.int8)[:, None].repeat(1, 2).contiguous()]
    cache = kvcache.PagedKVCache(k.to(cuda_dev), v.to(cuda_dev), *(e.to(cuda_dev) for e in ex))
    table = torch.arange(P, dtype=torch.int32).repeat(copies)[None].contiguous()
    n = P * T * copies
    ref = OK.attend(q, [k.double(), v.double()], ex, table, [n], sm_scale=1.0)
    out = kvcache.attend(q.to(cuda_dev), cache, table.to(cuda_dev), torch.tensor([n], dtype=torch.int32, device=cuda_dev), sm_scale=1.0)
    for i in range(P):
        _rows_near(out[0, i], ref[0, i], 448.0 * 2.0 ** exps[i])


@pytest.mark.parametrize("above", [20.6, 21.5, 23.4, 28.0, 40.0])
@pytest.mark.parametrize("B,Sq,H,Hk,T,n", [(64, 1, 24, 24, 64, 4096), (64, 1, 8, 8, 16, 4095), (1, 20, 2, 2, 32, 250), (2, 1, 2, 1, 64, 9000)])
def test_a_flat_tail_behind_one_key(dsb, cuda_dev, above, B, Sq, H, Hk, T, n):
    """One key's score is `above` powers of two over all the others', which are equal, and its value is zero: what comes out is the
    tail's values times 2^-above of their number, each probability with its 11 bits.

    But for the keys that share a tile of 32 with that one key: their probabilities are rounded on the scale of its own, to a multiple
    of 2^-24 where it is 2^12, so each is off by 2^-37 of it at most, and never by more than itself.  31 of n tail keys, of 2^-above
    each: min(1, 2^(above - 37)) * 31 / (n - 1) of the result (values between 200 and 300 times their mean's 250: 1.2 of that)."""
    from diffsynth_engine_b200 import kvcache
    W = -(-n // T)
    g = torch.Generator().manual_seed(n)
    v = (torch.rand(W, Hk, T, 128, generator=g) * 100 + 200).to(torch.float8_e4m3fn)
    k = torch.zeros(W, Hk, T, 128)
    k[0, :, 3], v[0, :, 3] = 2.0, 0
    k = k.to(torch.float8_e4m3fn)
    q = torch.full((1, Sq, H, 128), 0.5).bfloat16()
    scale = above * 0.6931471805599453 / 128                # the score is 128, and 2^above its power
    ex = [torch.zeros(W, Hk, dtype=torch.int8), torch.full((W, Hk), -8, dtype=torch.int8)]
    table = torch.arange(W, dtype=torch.int32)[None]
    cache = kvcache.PagedKVCache(k.to(cuda_dev), v.to(cuda_dev), *(e.to(cuda_dev) for e in ex))
    rows = OK.held(v.double(), ex[1], table[0], n)          # [n, Hk, 128]
    w = torch.full((n,), 2.0 ** -above, dtype=torch.float64)
    w[3] = 1
    ref = torch.einsum("n,nhd->hd", w / w.sum(), rows).repeat_interleave(H // Hk, 0)[None, None].expand(B, Sq, H, 128)
    out = kvcache.attend(q.expand(B, -1, -1, -1).to(cuda_dev), cache, table.expand(B, -1).contiguous().to(cuda_dev),
                         torch.full((B,), n, dtype=torch.int32, device=cuda_dev), sm_scale=scale).double().cpu()
    assert float(((out - ref).abs() / ref).max()) <= 2.0 ** -8 + 2.0 ** -11 + 1.2 * min(1, 2.0 ** (above - 37)) * 31 / (n - 1)  # (all values are positive)


@pytest.mark.parametrize("garbage", [-128, -127, -65, 65, 127])
@pytest.mark.parametrize("T", [16, 32])
def test_exponents_of_unwritten_pages(dsb, cuda_dev, garbage, T):
    """Pages need no preparation: their bytes and exponents may be anything until an append writes their first token."""
    from diffsynth_engine_b200 import kvcache
    lens = list(range(1, 2 * T + 2)) + [300, 333]
    B, W = len(lens), -(-max(lens) // T) + 1
    table = torch.arange(B * W, dtype=torch.int32).view(B, W)
    g = torch.Generator().manual_seed(T)
    k, v, q = (torch.randn(B, r, h, 128, generator=g).bfloat16() for r, h in ((max(lens), 1), (max(lens), 1), (2, 2)))
    pools = [torch.full((B * W, 1, T, 128), 0x7f, dtype=torch.uint8, device=cuda_dev).view(torch.float8_e4m3fn) for _ in range(2)]
    exps = [torch.full((B * W, 1), garbage, dtype=torch.int8, device=cuda_dev) for _ in range(2)]
    cache = kvcache.PagedKVCache(*pools, *exps)
    lt = torch.tensor(lens, dtype=torch.int32, device=cuda_dev)
    kvcache.append(cache, k.to(cuda_dev), v.to(cuda_dev), table.to(cuda_dev), 0, lt)
    kv, ex = _held(cache)
    ref = OK.attend(q, kv, ex, table, lens)
    out = kvcache.attend(q.to(cuda_dev), cache, table.to(cuda_dev), lt)
    _rows_near(out, ref, float(v.abs().max()) * 1.07)


def test_exponents_outside_their_range(dsb, cuda_dev):
    """A caller's exponents outside -64..64 count as the nearer end: for reads, attention and appends to the page."""
    from diffsynth_engine_b200 import kvcache
    g = torch.Generator().manual_seed(9)
    kv = [(torch.randn(4, 2, 16, 128, generator=g) * 90).clamp(-448, 448).to(torch.float8_e4m3fn) for _ in range(2)]
    ex = [torch.tensor([[-128, 3], [127, -65], [0, 65], [-64, 100]], dtype=torch.int8), torch.tensor([[5, -128], [-100, 64], [127, 2], [65, -65]], dtype=torch.int8)]
    q = torch.randn(1, 3, 2, 128, generator=g).bfloat16().to(cuda_dev)
    rows = [(torch.randn(1, 5, 2, 128, generator=g) * s).bfloat16().to(cuda_dev) for s in (1e-3, 1e6)]
    table = torch.arange(4, dtype=torch.int32, device=cuda_dev)[None]
    got = []
    for e in (ex, [t.clamp(-64, 64) for t in ex]):
        cache = kvcache.PagedKVCache(*(t.to(cuda_dev) for t in kv), *(t.to(cuda_dev) for t in e))
        out = [*kvcache.read(cache, table, 64), kvcache.attend(q, cache, table, 64)]
        kvcache.append(cache, *rows, table, 57)
        got.append(out + [cache.k[3].view(torch.uint8), cache.v[3].view(torch.uint8), cache.k_exp[3], cache.v_exp[3]])
    assert all(torch.equal(a.nan_to_num(nan=7.0) if a.is_floating_point() else a, b.nan_to_num(nan=7.0) if b.is_floating_point() else b)
               for a, b in zip(*got))
    assert bool(got[0][0].isfinite().all()) and bool(got[0][1].isfinite().all())


def test_pages_only(dsb, cuda_dev, monkeypatch):
    """Whatever the estimate says: the pages' own precision, and keys of entries that are no pages masked."""
    from diffsynth_engine_b200 import kvcache
    g = torch.Generator().manual_seed(4)
    B, Sq, H, T, W = 2, 600, 2, 64, 5
    kv = [(torch.randn(B * W, H, T, 128, generator=g) * 90).clamp(-448, 448).to(torch.float8_e4m3fn) for _ in range(2)]
    ex = [torch.full((B * W, H), -7, dtype=torch.int8) for _ in range(2)]
    cache = kvcache.PagedKVCache(*(t.to(cuda_dev) for t in kv), *(t.to(cuda_dev) for t in ex))
    q = torch.randn(B, Sq, H, 128, generator=g).bfloat16()
    table = torch.randperm(B * W, generator=g).view(B, W).int()
    monkeypatch.setattr(kvcache, "dense_pays", lambda *sizes: True)
    n = W * T - 3
    out = kvcache.attend(q.to(cuda_dev), cache, table.to(cuda_dev), n, pages_only=True)
    lens = torch.full((B,), n, dtype=torch.int32, device=cuda_dev)
    assert torch.equal(out, kvcache.attend(q.to(cuda_dev), cache, table.to(cuda_dev), lens))
    top = float(max((t.double().abs().max() for t in kv))) * 2.0 ** -7
    _rows_near(out, OK.attend(q, [t.double() for t in kv], ex, table, [n] * B), top)
    bad = table.clone()
    bad[1, 2] = B * W
    out = kvcache.attend(q.to(cuda_dev), cache, bad.to(cuda_dev), n, pages_only=True)
    with pytest.raises(dsb.DsbError, match="ERR_ARG"):
        dsb.ops.check_status(0)
    seen = torch.ones(B, n, dtype=torch.bool)
    seen[1, 2 * T:3 * T] = False
    _rows_near(out, OK.attend(q, [t.double() for t in kv], ex, table, [n] * B, ok=seen), top)

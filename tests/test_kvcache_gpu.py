"""The paged 8-bit key/value cache: appends bit for bit, reads exactly, attention against 64 bits.

Tolerance of the attention: the output is rounded to bf16, half a step is 2^-8 of a value at most (1.7e-3 rms), and the
probabilities may be rounded to 16 bits with at least 11 (2^-11 each, independent): 2^-8 + 2^-11 of the norm is asked, and per
value 2^-8 of the value plus 2^-10 of the largest |v| that it averages."""
import pytest
import torch

from oracle import kvcache as OK
from oracle import ops as O

pytestmark = pytest.mark.gpu
NAN8 = 0x7f


def _pool(P, H, T, seed, lo=-9, hi=-4):
    """A cache with random content: (k, v as e4m3, exponents)."""
    g = torch.Generator().manual_seed(seed)
    kv = [(torch.randn(P, H, T, 128, generator=g) * 90).clamp(-448, 448).to(torch.float8_e4m3fn) for _ in range(2)]
    return kv, [torch.randint(lo, hi, (P, H), generator=g, dtype=torch.int8) for _ in range(2)]


def _cache(dev, kv, ex):
    from diffsynth_engine_b200 import kvcache
    return kvcache.PagedKVCache(*(t.to(dev) for t in kv), *(t.to(dev) for t in ex))


def _table(B, W, P, seed):
    return torch.randperm(P, generator=torch.Generator().manual_seed(seed))[:B * W].view(B, W).int()


def _angles(n):
    f = 10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)
    a = torch.outer(torch.arange(n, dtype=torch.float64), f)
    return torch.stack([a.cos(), a.sin()], -1).float().contiguous()


def _same_bytes(cache, kv, ex):
    for got, want in zip((cache.k, cache.v), kv):
        assert torch.equal(got.cpu().view(torch.uint8), want.view(torch.uint8))
    for got, want in zip((cache.k_exp, cache.v_exp), ex):
        assert torch.equal(got.cpu(), want)


def _append_ref(kv, ex, table, start, counts, k, v, rope=None, row0=0):
    kv2, ex2 = [], []
    for pages, e, rows in zip(kv, ex, (k, v)):
        rows = rows.float()
        if rope is not None and rows is not None and pages is kv[0]:
            rows = torch.stack([torch.cat([OK.rotate(rows[b, :int(counts[b])], rope, row0 + int(start[b])), rows[b, int(counts[b]):]])
                                for b in range(rows.shape[0])])
        p, e = pages.double(), e.clone()
        raw = pages.clone().view(torch.uint8)
        OK.append(p, e, table, start, counts, rows)
        q = p.float().to(torch.float8_e4m3fn).view(torch.uint8)
        changed = ~(p == pages.double()) & ~p.isnan() | (p.isnan() & ~pages.double().isnan())
        kv2.append(torch.where(changed, q, raw).view(torch.float8_e4m3fn))
        ex2.append(e)
    return kv2, ex2


CASES = [
    # B, n, H, T, starts, counts, rotated
    (1, 1, 1, 16, [0], None, False), (1, 1, 2, 16, [5], None, True), (3, 1, 2, 64, [0, 63, 64], None, True),
    (2, 16, 1, 16, [0, 16], None, False), (2, 17, 3, 16, [15, 1], [17, 0], True), (1, 512, 2, 64, [0], None, False),
    (2, 130, 2, 32, [31, 7], [1, 130], True), (1, 200, 1, 128, [100], None, True), (4, 3, 5, 128, [125, 126, 0, 128], [3, 2, 1, 3], True),
]


@pytest.mark.parametrize("B,n,H,T,starts,counts,rot", CASES)
def test_append_is_exact(dsb, cuda_dev, B, n, H, T, starts, counts, rot):
    from diffsynth_engine_b200 import kvcache
    W = -(-(max(starts) + n) // T) + 1
    kv, ex = _pool(B * W + 3, H, T, seed=n)
    table = _table(B, W, B * W + 3, seed=n + 1)
    g = torch.Generator().manual_seed(n + T)
    k, v = torch.randn(B, n, H, 128, generator=g).bfloat16(), (torch.randn(B, n, H, 128, generator=g) * 3).bfloat16()
    if n > 2:
        k[0, 1] = 0
        v[0, 2] *= 1e-20
    rope = _angles(max(starts) + n + 9) if rot else None
    st, ct = torch.tensor(starts, dtype=torch.int32), torch.tensor(counts if counts else [n] * B, dtype=torch.int32)
    cache = _cache(cuda_dev, kv, ex)
    args = dict(rope=None if rope is None else rope.to(cuda_dev), rope_row0=2 if rot else 0)
    want = _append_ref(kv, ex, table, st, ct, k, v, rope, 2)
    kvcache.append(cache, k.to(cuda_dev), v.to(cuda_dev), table.to(cuda_dev), st.to(cuda_dev), ct.to(cuda_dev) if counts else None, **args)
    _same_bytes(cache, *want)
    # once more: the rows are the same, and their blocks have the exponent already
    kvcache.append(cache, k.to(cuda_dev), v.to(cuda_dev), table.to(cuda_dev), st.to(cuda_dev), ct.to(cuda_dev) if counts else None, **args)
    _same_bytes(cache, *want)
    if B == 1 and counts is None:      # a start that the host knows, rows inside a wider projection
        fused = torch.zeros(1, n, 3, H, 128, dtype=torch.bfloat16)
        fused[:, :, 1], fused[:, :, 2] = k, v
        fused = fused.to(cuda_dev)
        cache = _cache(cuda_dev, kv, ex)
        kvcache.append(cache, fused[:, :, 1], fused[:, :, 2], table.to(cuda_dev), starts[0], **args)
        _same_bytes(cache, *want)


def test_append_exponents(dsb, cuda_dev):
    """Magnitudes at the border of a power of two, beyond the exponents' range, and numbers that are not finite."""
    from diffsynth_engine_b200 import kvcache
    tops = [448.0, 450.0, 1.75, 1.7578125, 3.5, 2.0 ** -63, 2.0 ** -100, 3e38, 0.0, 7.0]
    H = len(tops)
    k = torch.zeros(1, 3, H, 128)
    for h, t in enumerate(tops):
        k[0, 1, h, 5], k[0, 2, h, 77] = -t, t / 3
    k[0, 0, 9, 0], k[0, 0, 9, 1], k[0, 0, 9, 2] = float("inf"), -float("inf"), float("nan")
    k = k.bfloat16()
    v = k.flip(2).contiguous()
    for slot in (0, 4):
        kv, ex = _pool(2, H, 16, seed=slot)
        want = _append_ref(kv, ex, torch.tensor([[1]]), [slot], [3], k, v)
        cache = _cache(cuda_dev, kv, ex)
        kvcache.append(cache, k.to(cuda_dev), v.to(cuda_dev), torch.tensor([[1]], dtype=torch.int32, device=cuda_dev), slot)
        assert torch.equal(cache.k_exp.cpu(), want[1][0]) and torch.equal(cache.v_exp.cpu(), want[1][1])
        for got, ref in zip((cache.k, cache.v), want[0]):
            a, b = got.cpu().float(), ref.float()
            assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(nan=0.0), b.nan_to_num(nan=0.0))
        if slot == 0:      # 448 = 448 * 2^0, 450 needs 2^1; 1.75 = 448 * 2^-8; zeros and what lies below take the least, 3e38 the most
            assert cache.k_exp[1].tolist() == [0, 1, -8, -7, -7, -64, -64, 64, -64, -6]
            assert float(cache.k[1, 9, 0, 0].float()) == 448.0 and float(cache.k[1, 9, 0, 1].float()) == -448.0


def test_read_is_exact(dsb, cuda_dev):
    from diffsynth_engine_b200 import kvcache
    kv, ex = _pool(9, 3, 32, seed=1, lo=-64, hi=65)
    cache, table = _cache(cuda_dev, kv, ex), _table(2, 4, 9, 2)
    for first, n in ((0, 1), (0, 128), (31, 2), (100, 28), (5, 0)):
        got = kvcache.read(cache, table.to(cuda_dev), n, first)
        for i in (0, 1):
            want = torch.stack([OK.held(kv[i].double(), ex[i], table[b], 128)[first:first + n] for b in (0, 1)])
            assert torch.equal(got[i].cpu().double(), want)


ATT = [
    # B, Sq, H, Hk, T, lens, causal
    (1, 1, 1, 1, 16, [1], False), (1, 1, 2, 2, 16, [77], False), (2, 1, 8, 2, 64, [0, 65], False), (3, 1, 5, 1, 32, [31, 32, 33], True),
    (2, 3, 8, 8, 128, [127, 2], True), (1, 5, 10, 2, 64, [300], True), (2, 16, 4, 4, 16, [16, 250], False), (2, 17, 16, 2, 64, [17, 500], True),
    (1, 70, 4, 2, 32, [64], True), (2, 130, 3, 3, 64, [129, 400], False), (1, 1, 64, 4, 64, [2100], False), (5, 2, 24, 3, 128, [1, 1300, 0, 257, 640], True),
    (1, 1, 2, 1, 64, [9000], False), (1, 300, 2, 1, 64, [40], True), (1, 20, 4, 2, 16, [45], True), (2, 3, 8, 1, 16, [700, 5], True),
    (1, 3, 10, 1, 64, [3000], False), (2, 33, 2, 1, 128, [2500, 1200], True), (70, 1, 3, 3, 16, [9 * i % 40 for i in range(70)], False),
]


@pytest.mark.parametrize("B,Sq,H,Hk,T,lens,causal", ATT)
@pytest.mark.parametrize("sharp", [1.0, 12.0])
def test_attention(dsb, cuda_dev, B, Sq, H, Hk, T, lens, causal, sharp):
    """Also: what lies behind a sequence's length is NaN, blocks of a head differ in scale, and rows of q in size."""
    from diffsynth_engine_b200 import kvcache
    W = -(-max(lens) // T) + 1
    kv, ex = _pool(B * W + 2, Hk, T, seed=B + Sq)
    table = _table(B, W, B * W + 2, seed=Sq)
    for t in kv:
        raw = t.view(torch.uint8)
        for b in range(B):
            for j in range(W):
                raw[int(table[b, j]), :, max(0, min(T, lens[b] - j * T)):] = NAN8
    g = torch.Generator().manual_seed(7)
    q = (torch.randn(B, Sq, H, 128, generator=g) * sharp).bfloat16()
    if Sq > 1:
        q[0, 1] = 0
    lt = torch.tensor(lens, dtype=torch.int32)
    ref = OK.attend(q, [t.double() for t in kv], ex, table, lens, causal)
    cache = _cache(cuda_dev, kv, ex)
    out = kvcache.attend(q.to(cuda_dev), cache, table.to(cuda_dev), lt.to(cuda_dev), causal=causal)
    _near(out, ref, kv, ex)
    assert torch.equal(out, kvcache.attend(q.to(cuda_dev), cache, table.to(cuda_dev), lt.to(cuda_dev), causal=causal))
    if len(set(lens)) == 1:
        one = kvcache.attend(q.to(cuda_dev), cache, table.to(cuda_dev), lens[0], causal=causal)
        _near(one, ref, kv, ex)
    # queries and results inside wider rows, another scale
    wide = torch.zeros(B, Sq, H + 2, 128, dtype=torch.bfloat16, device=cuda_dev)
    wide[:, :, 1:H + 1] = q.to(cuda_dev)
    into = torch.full((B, Sq, H + 1, 128), 5.0, dtype=torch.bfloat16, device=cuda_dev)
    kvcache.attend(wide[:, :, 1:H + 1], cache, table.to(cuda_dev), lt.to(cuda_dev), causal=causal, sm_scale=0.05, out=into[:, :, :H])
    _near(into[:, :, :H], OK.attend(q, [t.double() for t in kv], ex, table, lens, causal, 0.05), kv, ex)
    assert bool((into[:, :, H:] == 5).all())


@pytest.mark.parametrize("B,Sq,H,Hk,T,n,dense", [(1, 400, 4, 4, 64, 300, True), (2, 2100, 2, 1, 16, 513, True), (1, 257, 6, 1, 32, 90, False),
                                                 (1, 700, 8, 1, 64, 640, False), (3, 256, 2, 2, 128, 385, True),
                                                 (2, 900, 5, 1, 32, 200, False)])
def test_many_queries_by_either_route(dsb, cuda_dev, B, Sq, H, Hk, T, n, dense):
    """A known length: read back for the dense kernel where that is estimated to be less, the pages otherwise.  The dense kernel
    rounds a probability to bf16, at most 2^-8 of it: on a result at most 2^-8 of the largest value, on all of them half a step
    (2^-8 / sqrt 3 rms) as often as the result's own rounding, together less than 2^-8."""
    from diffsynth_engine_b200 import kvcache
    assert kvcache.dense_pays(B, Sq, H, Hk, n) == dense
    W = -(-n // T)
    kv, ex = _pool(B * W + 1, Hk, T, seed=n)
    table = _table(B, W, B * W + 1, seed=Sq)
    q = torch.randn(B, Sq, H, 128, generator=torch.Generator().manual_seed(7)).bfloat16()
    ref = OK.attend(q, [t.double() for t in kv], ex, table, [n] * B, False)
    cache = _cache(cuda_dev, kv, ex)
    out = torch.full((B, Sq, H + 1, 128), 5.0, dtype=torch.bfloat16, device=cuda_dev)
    kvcache.attend(q.to(cuda_dev), cache, table.to(cuda_dev), n, out=out[:, :, :H])
    assert bool((out[:, :, H:] == 5).all())
    whole = kvcache.attend(q.to(cuda_dev), cache, table.to(cuda_dev), n)     # (one cache head: its query heads as rows of one launch)
    top = float((kv[1].double().abs().amax(dim=(2, 3)) * 2.0 ** ex[1].double()).max())
    for got in (out[:, :, :H].double().cpu(), whole.double().cpu()):
        assert float(((got - ref).abs() - ref.abs() * 2.0 ** -8).max()) <= 2.0 ** -8 * top
        assert O.rel_l2(got, ref) < 2.0 ** -8 + 2.0 ** -11


def test_broadcast_queries(dsb, cuda_dev, monkeypatch):
    """Queries with a stride of 0 read the pages, where others would take the dense kernel."""
    from diffsynth_engine_b200 import kvcache
    kv, ex = _pool(9, 2, 64, seed=2)
    table, cache = _table(2, 4, 9, 3), _cache(cuda_dev, kv, ex)
    monkeypatch.setattr(kvcache, "dense_pays", lambda *sizes: True)
    q = torch.randn(2, 600, 2, 128, generator=torch.Generator().manual_seed(5)).bfloat16().to(cuda_dev)
    for x in (q[:1].expand(2, -1, -1, -1), q[:, :1].expand(-1, 600, -1, -1), q[:, :, :1].expand(-1, -1, 2, -1)):
        out = kvcache.attend(x, cache, table.to(cuda_dev), 250)
        _near(out, OK.attend(x.cpu(), [t.double() for t in kv], ex, table, [250, 250]), kv, ex)


def _near(out, ref, kv, ex):
    out = out.double().cpu()
    assert bool(out.isfinite().all())
    assert bool((out[ref.abs().amax(-1) == 0] == 0).all())
    top = float((kv[1].double().nan_to_num(nan=0.0).abs().amax(dim=(2, 3)) * 2.0 ** ex[1].double()).max())
    assert float(((out - ref).abs() - ref.abs() * 2.0 ** -8).max()) <= 2.0 ** -10 * top
    if float(ref.norm()) > 0:
        assert O.rel_l2(out, ref) < 2.0 ** -8 + 2.0 ** -11


def test_blocks_of_very_different_scale(dsb, cuda_dev):
    """Value blocks 2^40 apart, the probability on the small one: its rows come out with their own precision."""
    from diffsynth_engine_b200 import kvcache
    kv, ex = _pool(8, 1, 16, seed=3)
    ex[1][:, 0] = torch.tensor([-30, 10, -20, 0, -30, 5, -10, -30], dtype=torch.int8)
    table = torch.arange(8, dtype=torch.int32)[None]
    q = torch.randn(1, 4, 2, 128, generator=torch.Generator().manual_seed(1)).bfloat16()
    k = kv[0].float()
    k[0, 0, 3] = q[0, 0, 0].float() * 200 / q[0, 0, 0].float().abs().max()       # query 0 looks at a key of the smallest block
    kv[0] = k.to(torch.float8_e4m3fn)
    ex[0][0] = 0
    cache = _cache(cuda_dev, kv, ex)
    out = kvcache.attend(q.to(cuda_dev), cache, table.to(cuda_dev), 128).double().cpu()
    ref = OK.attend(q, [t.double() for t in kv], ex, table, [128])
    for i in range(4):
        for h in range(2):
            assert O.rel_l2(out[0, i, h], ref[0, i, h]) < 2.0 ** -8 + 2.0 ** -10


@pytest.mark.parametrize("T,n,Sq", [(16, 40, 20), (64, 100, 9), (64, 700, 5), (128, 1300, 40)])
def test_nan_stays_with_the_rows_that_see_it(dsb, cuda_dev, T, n, Sq):
    """A key, a value column or a query that is NaN reaches the rows that see it and no other; cut sequences too."""
    from diffsynth_engine_b200 import kvcache
    B, H, Hk = 2, 6, 2
    W = -(-n // T) + 1
    kv, ex = _pool(B * W, Hk, T, seed=T)
    table = _table(B, W, B * W, seed=1)
    q = torch.randn(B, Sq, H, 128, generator=torch.Generator().manual_seed(2)).bfloat16()

    def put(i, b, tok, head, cols):
        kv[i].view(torch.uint8)[int(table[b, tok // T]), head, tok % T, cols] = NAN8

    put(1, 0, n - 2, 0, slice(17, 18))          # a value that the last two queries of sequence 0 see
    put(0, 1, n - 3, 1, slice(5, 6))            # a key that the last three of sequence 1 see
    q[0, 2, 5, 7] = float("nan")                # one row of its own
    out = kvcache.attend(q.to(cuda_dev), _cache(cuda_dev, kv, ex), table.to(cuda_dev), torch.full((B,), n, dtype=torch.int32, device=cuda_dev),
                         causal=True).cpu()
    nan = out.isnan()
    want = torch.zeros_like(nan)
    want[0, Sq - 2:, :3, 17] = True
    want[1, Sq - 3:, 3:] = True
    want[0, 2, 5] = True
    assert torch.equal(nan, want)
    clean = [t.clone() for t in kv]
    for t in clean:
        t.view(torch.uint8)[t.view(torch.uint8) & 0x7f == 0x7f] = 0
    q[0, 2, 5, 7] = 0
    ref = OK.attend(q, [t.double() for t in clean], ex, table, [n] * B, True)
    rows = ~want.any(-1)
    assert O.rel_l2(out[rows], ref[rows]) < 2.0 ** -8 + 2.0 ** -11
    keep = ~want[0, Sq - 2:, :3]
    assert O.rel_l2(out[0, Sq - 2:, :3][keep], ref[0, Sq - 2:, :3][keep]) < 2.0 ** -8 + 2.0 ** -11


def test_sequences_share_pages(dsb, cuda_dev):
    """A prompt's pages, in the tables of several sequences."""
    from diffsynth_engine_b200 import kvcache
    kv, ex = _pool(8, 2, 32, seed=8)
    table = torch.tensor([[3, 1, 4], [3, 1, 7], [3, 3, 3]], dtype=torch.int32)
    q = torch.randn(3, 2, 4, 128, generator=torch.Generator().manual_seed(3)).bfloat16()
    lens = [70, 96, 65]
    out = kvcache.attend(q.to(cuda_dev), _cache(cuda_dev, kv, ex), table.to(cuda_dev), torch.tensor(lens, dtype=torch.int32, device=cuda_dev))
    _near(out, OK.attend(q, [t.double() for t in kv], ex, table, lens), kv, ex)


def test_pools_past_32_bits(dsb, cuda_dev):
    """Pools of 5.4 GB each: appends, reads and attention on their last pages."""
    from diffsynth_engine_b200 import kvcache
    P, H, T = 41000, 8, 128
    cache = kvcache.PagedKVCache.empty(P, H, T, cuda_dev)
    table = torch.tensor([[P - 1, 5, P - 3]], dtype=torch.int32, device=cuda_dev)
    g = torch.Generator(device=cuda_dev).manual_seed(0)
    k, v = (torch.randn(1, 300, H, 128, generator=g, device=cuda_dev).bfloat16() for _ in range(2))
    kvcache.append(cache, k, v, table, 0)
    small = kvcache.PagedKVCache.empty(3, H, T, cuda_dev)
    near = torch.tensor([[0, 1, 2]], dtype=torch.int32, device=cuda_dev)
    kvcache.append(small, k, v, near, 0)
    q = torch.randn(1, 4, 16, 128, generator=g, device=cuda_dev).bfloat16()
    assert torch.equal(kvcache.attend(q, cache, table, 300, causal=True), kvcache.attend(q, small, near, 300, causal=True))
    assert all(torch.equal(a, b) for a, b in zip(kvcache.read(cache, table, 300), kvcache.read(small, near, 300)))


def test_bad_pages_and_lengths_are_masked_and_reported(dsb, cuda_dev):
    from diffsynth_engine_b200 import kvcache
    kv, ex = _pool(6, 2, 16, seed=4)
    cache = _cache(cuda_dev, kv, ex)
    good = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32)
    q = torch.randn(2, 2, 4, 128, generator=torch.Generator().manual_seed(1)).bfloat16().to(cuda_dev)
    lens = torch.tensor([40, 48], dtype=torch.int32)

    def reported():
        with pytest.raises(dsb.DsbError, match="ERR_ARG"):
            dsb.ops.check_status(0)

    for wrong in (-1, 6, 1 << 30, -(1 << 31)):
        t = good.clone()
        t[0, 1] = wrong
        out = kvcache.attend(q, cache, t.to(cuda_dev), lens.to(cuda_dev))
        reported()
        ok = torch.ones(2, 48, dtype=torch.bool)
        ok[0, 16:32] = False
        _near(out, OK.attend(q.cpu(), [x.double() for x in kv], ex, good, [40, 48], ok=ok), kv, ex)
        k, _ = kvcache.read(cache, t.to(cuda_dev), 48)
        reported()
        assert bool((k[0, 16:32] == 0).all()) and not bool((k[1] == 0).all())
        rows = torch.ones(2, 20, 2, 128, dtype=torch.bfloat16, device=cuda_dev)
        mine = _cache(cuda_dev, kv, ex)
        kvcache.append(mine, rows, rows, t.to(cuda_dev), 10)
        reported()
        ref = _append_ref(kv, ex, good, [10, 10], [6, 20], rows.cpu(), rows.cpu())
        _same_bytes(mine, *ref)
    for wrong in (-1, 49, 1 << 30, -(1 << 31)):
        n = torch.tensor([wrong, 48], dtype=torch.int32)
        out = kvcache.attend(q, cache, good.to(cuda_dev), n.to(cuda_dev))
        reported()
        _near(out, OK.attend(q.cpu(), [x.double() for x in kv], ex, good, [max(0, min(48, wrong)), 48]), kv, ex)
    rows = torch.ones(2, 4, 2, 128, dtype=torch.bfloat16, device=cuda_dev)
    rope = _angles(40).to(cuda_dev)
    for start, counts, kw in (([-1, 0], [4, 0], {}), ([45, 0], [4, 0], {}), ([(1 << 31) - 2, 0], [4, 0], {}), ([0, 0], [5, 0], {}), ([0, 0], [-1, 0], {}),
                              ([37, 0], [4, 0], dict(rope=rope)), ([0, 20], [4, 0], dict(rope=rope, rope_row0=-1)),
                              ([4, 0], [4, 0], dict(rope=rope, rope_row0=(1 << 31) - 4))):
        mine = _cache(cuda_dev, kv, ex)
        kvcache.append(mine, rows, rows, good.to(cuda_dev), torch.tensor(start, dtype=torch.int32, device=cuda_dev),
                       torch.tensor(counts, dtype=torch.int32, device=cuda_dev), **kw)
        reported()
        _same_bytes(mine, kv, ex)


def test_refusals(dsb, cuda_dev):
    from diffsynth_engine_b200 import kvcache
    c = kvcache.PagedKVCache.empty(4, 2, 16, cuda_dev)
    t = torch.zeros(1, 2, dtype=torch.int32, device=cuda_dev)
    x = torch.zeros(1, 3, 2, 128, dtype=torch.bfloat16, device=cuda_dev)
    n = torch.ones(1, dtype=torch.int32, device=cuda_dev)
    for bad in (lambda: kvcache.PagedKVCache(c.k, c.v[:2], c.k_exp, c.v_exp), lambda: kvcache.PagedKVCache(c.k, c.v, c.k_exp.int(), c.v_exp),
                lambda: kvcache.PagedKVCache(c.k[..., :64], c.v[..., :64], c.k_exp, c.v_exp), lambda: kvcache.PagedKVCache.empty(4, 2, 48, cuda_dev),
                lambda: kvcache.PagedKVCache(c.k, c.v.cpu(), c.k_exp, c.v_exp), lambda: kvcache.PagedKVCache(c.k.transpose(0, 1), c.v.transpose(0, 1), c.k_exp.t(), c.v_exp.t()),
                lambda: kvcache.append(c, x, x[:, :2], t, 0), lambda: kvcache.append(c, x[:, :, :1], x[:, :, :1], t, 0),
                lambda: kvcache.append(c, x.half(), x.half(), t, 0), lambda: kvcache.append(c, x, x, t.long(), 0),
                lambda: kvcache.append(c, x, x, t, 30), lambda: kvcache.append(c, x, x, t, -1), lambda: kvcache.append(c, x, x, t, n.long()),
                lambda: kvcache.append(c, x, x, t, 0, n[:0]), lambda: kvcache.append(c, x, x, t, 0, rope=torch.zeros(9, 64, 2, dtype=torch.float16, device=cuda_dev)),
                lambda: kvcache.append(c, x.cpu(), x.cpu(), t.cpu(), 0), lambda: kvcache.attend(x, c, t, 33), lambda: kvcache.attend(x, c, t, -1),
                lambda: kvcache.attend(x[:, :, :1], c, t, 4), lambda: kvcache.attend(x[..., :64], c, t, 4), lambda: kvcache.attend(x.float(), c, t, 4),
                lambda: kvcache.attend(x, c, t[:, :0], 4), lambda: kvcache.attend(x, c, t.expand(2, 2), 4), lambda: kvcache.attend(x, c, t, n.long()),
                lambda: kvcache.attend(x, c, t, 4, out=x[:, :2]), lambda: kvcache.attend(x, c, t, 4, out=x[:, :1].expand(1, 3, 2, 128)),
                lambda: kvcache.read(c, t, 33), lambda: kvcache.read(c, t, 1, -1)):
        with pytest.raises(dsb.DsbError):
            bad()
    kvcache.append(c, x[:, :0], x[:, :0], t, 0)
    assert kvcache.attend(x[:, :0], c, t, 0).shape == (1, 0, 2, 128)
    assert bool((kvcache.attend(x, c, t, 0) == 0).all())

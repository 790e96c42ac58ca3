"""What the 4-bit weights and the paged cache check without a GPU: the index arithmetic of the cache's kernels, compiled for the
CPU and run against the obvious loops, and the refusals of the C entry points, which come before any launch."""
import ctypes
import os
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SHIM = """
#include "kv_index.h"
extern "C" {
int t_page(const int* row, int w, int n, int j) { return dsb::kv_page(row, w, n, j); }
int t_length(int len, long long cap) { return dsb::kv_length(len, cap); }
int t_length_ok(int len, long long cap) { return dsb::kv_length_ok(len, cap); }
int t_visible(int len, int sq, int i, int c) { return dsb::kv_visible(len, sq, i, c); }
void t_span(int start, int count, int T, int j, int* out) {
  const dsb::KvSpan s = dsb::kv_span(start, count, T, j);
  out[0] = s.index, out[1] = s.slot, out[2] = s.row, out[3] = s.rows;
}
int t_span_pages(int n, int T) { return dsb::kv_span_pages(n, T); }
int t_append_ok(int start, int count, int n, long long cap) { return dsb::kv_append_ok(start, count, n, cap); }
int t_exponent(unsigned bits) { return dsb::kv_exponent(bits); }
}
"""


@pytest.fixture(scope="module")
def idx(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv_index")
    (d / "shim.cpp").write_text(SHIM)
    so = d / "shim.so"
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-fsanitize=signed-integer-overflow", "-fsanitize-undefined-trap-on-error", "-I",
                    os.path.join(ROOT, "diffsynth-engine_b200", "csrc"), str(d / "shim.cpp"), "-o", str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    lib.t_length.argtypes = lib.t_length_ok.argtypes = [ctypes.c_int, ctypes.c_longlong]
    lib.t_append_ok.argtypes = [ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_longlong]
    lib.t_exponent.argtypes = [ctypes.c_uint]
    return lib


def test_pages_and_lengths(idx):
    row = (ctypes.c_int * 4)(2, -1, 7, 1 << 30)
    assert [idx.t_page(row, 4, 7, j) for j in (-1, 0, 1, 2, 3, 4, 1 << 30)] == [-1, 2, -1, -1, -1, -1, -1]
    assert idx.t_page(row, 4, 8, 2) == 7
    big = (1 << 31) - 1
    assert [idx.t_length(n, 64) for n in (-big - 1, -1, 0, 63, 64, 65, big)] == [0, 0, 0, 63, 64, 64, 64]
    assert [idx.t_length_ok(n, 64) for n in (-1, 0, 64, 65)] == [0, 1, 1, 0]
    assert [idx.t_visible(5, 3, i, 1) for i in range(3)] == [3, 4, 5] and idx.t_visible(5, 3, 0, 0) == 5
    assert [idx.t_visible(2, 4, i, 1) for i in range(4)] == [0, 0, 1, 2]
    assert [idx.t_append_ok(*a, 64) for a in ((0, 64, 64), (1, 64, 64), (-1, 1, 4), (0, 5, 4), (3, -1, 4), (big, 1, 4), (64, 0, 4))] == [1, 0, 0, 0, 0, 0, 1]


@pytest.mark.parametrize("T", [16, 32, 64, 128])
def test_spans_cover_every_row_once(idx, T):
    out = (ctypes.c_int * 4)()
    for start in (0, 1, T - 1, T, 5 * T + 3):
        for n in (1, 2, T - 1, T, T + 1, 3 * T + 5):
            for count in {0, 1, n // 2, n}:
                put = {}
                for j in range(idx.t_span_pages(n, T)):
                    idx.t_span(start, count, T, j, out)
                    index, slot, row, rows = out
                    assert rows == 0 or (0 <= slot and slot + rows <= T)
                    for r in range(rows):
                        assert row + r not in put
                        put[row + r] = index * T + slot + r
                assert put == {r: start + r for r in range(count)}


def test_exponents(idx):
    from oracle.kvcache import exponent
    vals = [0.0, 1e-45, 1e-38, 448.0, 448.00003, 447.99997, 1.75, 1.7500001, 2.0 ** -64 * 448, 3.0e38, 1.0, 3.5, 3.5000002, 5e21, 9e21]
    for v in vals:
        bits = torch.tensor(v, dtype=torch.float32).view(torch.int32).item()
        assert idx.t_exponent(bits) == exponent(float(torch.tensor(v, dtype=torch.float32))), v


def test_oracle_rounds_like_the_cast():
    from oracle.kvcache import round_e4m3
    x = torch.cat([torch.randn(20000) * 100, torch.randn(20000) * 0.01, torch.arange(-460, 460).float() / 2,
                   torch.arange(0, 256).to(torch.uint8).view(torch.float8_e4m3fn).float().nan_to_num(0.0)]).clamp(-448, 448)
    assert torch.equal(round_e4m3(x.double()).float(), x.to(torch.float8_e4m3fn).float())


def test_c_entries_refuse_before_any_launch(dsb):
    lib, P = dsb._lib.lib(), 1 << 20
    ARG, UNS = dsb._lib.ERR_ARG, dsb._lib.ERR_UNSUPPORTED

    def gemv(**kw):
        a = dict(p=P, s=P, m=None, N=16, K=64, group=32, x=P, ld_x=64, xb=0, bias=None, y=P, ld_y=16, yb=0, M=1, ai=0, ao=0, acc=0)
        a.update(kw)
        a = list(a.values())
        return lib.dsb_gemv_int4(ctypes.byref(dsb._lib.Int4Args(*a[:6])), *a[6:], None)

    for kw in (dict(p=None), dict(s=None), dict(x=None), dict(y=None), dict(N=0), dict(K=0), dict(K=63), dict(group=16), dict(M=33), dict(M=-1), dict(ai=1),
               dict(ao=4), dict(ao=-1), dict(p=P + 8), dict(s=P + 4), dict(x=P + 2), dict(M=2, ld_x=63), dict(M=2, ld_y=15), dict(y=P + 2)):
        assert gemv(**kw) == ARG, kw
    assert gemv(M=0, p=None) == 0
    assert lib.dsb_int4_pack(P, 31, P, None, 2, 16, 64, 32, P, P, None, None) == ARG
    assert lib.dsb_int4_pack(P, 32, P, P, 2, 16, 64, 32, P, P, None, None) == ARG
    assert lib.dsb_int4_from_gguf(14, P, 210, 1, 256, P, 128, P, P, None) == UNS
    assert lib.dsb_int4_from_gguf(2, P, 18, 1, 32, P, 16, P, P, None) == ARG          # Q4_0 has no minima
    assert lib.dsb_int4_from_gguf(3, P, 20, 1, 32, P, 16, P, None, None) == ARG       # Q4_1 has
    assert lib.dsb_int4_from_gguf(12, P, 143, 1, 256, P, 128, P, P, None) == ARG
    assert lib.dsb_int4_quantize(P, 63, 0, 1, 64, 32, P, 32, P, None, None) == ARG
    assert lib.dsb_int4_dequant(ctypes.byref(dsb._lib.Int4Args(P, P, None, 16, 64, 32)), P, 63, None) == ARG
    assert lib.dsb_gemv_int4(None, P, 64, 0, None, P, 16, 0, 1, 0, 0, 0, None) == ARG and lib.dsb_int4_dequant(None, P, 64, None) == ARG

    def cache(**kw):
        a = dict(k=P, v=P, k_exp=P, v_exp=P, n_pages=4, heads=2, page_tokens=16)
        a.update(kw)
        return ctypes.byref(dsb._lib.KVCacheArgs(**a))

    def attn(c=None, **kw):
        a = dict(q=P, qb=256, qs=256, qh=128, o=P, ob=256, os=256, oh=128, B=1, Sq=1, H=2, table=P, ld=2, width=2, lens=None, len_all=4, causal=0,
                 scale=0.1, ws=None, wsb=0, status=None)
        a.update(kw)
        return lib.dsb_kv_attn(c or cache(), *a.values(), None)

    for kw in (dict(q=None), dict(o=P + 8), dict(H=3), dict(H=0), dict(B=-1), dict(Sq=-1), dict(table=None), dict(width=0), dict(ld=1), dict(len_all=33),
               dict(len_all=-1), dict(qs=4), dict(oh=-8), dict(len_all=300, width=32, ld=32)):
        assert attn(**kw) == ARG, kw
    for c in (cache(k=None), cache(v_exp=None), cache(n_pages=0), cache(heads=0), cache(v=P + 16)):
        assert attn(c) == ARG
    for c in (cache(page_tokens=48), cache(page_tokens=256), cache(n_pages=1 << 27)):
        assert attn(c) == UNS
    assert lib.dsb_kv_attn(None, *([None] * 0), P, 256, 256, 128, P, 256, 256, 128, 1, 1, 2, P, 2, 2, None, 4, 0, 0.1, None, 0, None, None) == ARG
    assert attn(B=0, q=None) == 0 and attn(Sq=0, q=None) == 0

    def append(**kw):
        a = dict(k=P, kb=256, ks=256, kh=128, v=P, vb=256, vs=256, vh=128, B=1, n=3, table=P, ld=2, width=2, start=None, start_all=0, counts=None,
                 rope=None, rows=0, row0=0, status=None)
        a.update(kw)
        return lib.dsb_kv_append(cache(), *a.values(), None)

    for kw in (dict(k=None), dict(v=P + 2), dict(n=-1), dict(B=-1), dict(start_all=-1), dict(start_all=30), dict(table=P + 2), dict(ks=4), dict(rope=P + 4)):
        assert append(**kw) == ARG, kw
    assert append(n=0, k=None) == 0

    def read(**kw):
        a = dict(table=P, ld=2, width=2, B=1, first=0, n=4, k=P, kb=1024, ks=256, kh=128, v=P, vb=1024, vs=256, vh=128, status=None)
        a.update(kw)
        return lib.dsb_kv_read(cache(), *a.values(), None)

    for kw in (dict(k=None), dict(first=-1), dict(first=30), dict(n=33), dict(n=-1), dict(table=None)):
        assert read(**kw) == ARG, kw


def test_cpu_tensors_are_refused(dsb):
    from diffsynth_engine_b200 import int4, kvcache
    with pytest.raises(dsb.DsbError):
        int4.quantize(torch.zeros(16, 64))
    c = kvcache.PagedKVCache.empty(2, 1, 16, "cpu")
    x, t = torch.zeros(1, 1, 1, 128, dtype=torch.bfloat16), torch.zeros(1, 1, dtype=torch.int32)
    for call in (lambda: kvcache.append(c, x, x, t, 0), lambda: kvcache.attend(x, c, t, 1), lambda: kvcache.read(c, t, 1)):
        with pytest.raises(dsb.DsbError):
            call()


def test_which_attention_a_known_length_takes():
    """The gather and the dense kernel pay for many rows of a head; single tokens, empty sequences and many launches over little don't."""
    from diffsynth_engine_b200 import kvcache
    for args, dense in (((64, 1, 32, 8, 4096), False), ((1, 255, 24, 24, 4096), False), ((0, 300, 24, 24, 4096), False),
                        ((1, 300, 24, 24, 0), False), ((1, 4096, 24, 24, 4096), True), ((1, 4096, 32, 8, 4096), True),
                        ((1, 512, 32, 8, 512), False), ((1, 300, 1, 1, 100000), False), ((1, 32760, 4, 1, 512), True)):
        assert kvcache.dense_pays(*args) == dense, args

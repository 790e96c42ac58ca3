"""What the 4-bit weight functions hand to the library for rows that overlap in memory: one group of scales for all rows, one row of a
weight repeated, windows of a buffer.  The library is replaced by one that reads the rows where the arguments say they are."""
import ctypes

import pytest
import torch


class _Reads:
    """Takes the place of the loaded library: copies out the rows that a call would read, and checks that they are inside a tensor."""

    def __init__(self):
        self.seen = {}

    @staticmethod
    def rows(at, ld, n, cols, size):
        return torch.stack([torch.frombuffer(bytearray(ctypes.string_at(at + r * ld * size, cols * size)), dtype=torch.uint8) for r in range(n)])

    def dsb_int4_pack(self, codes, ld, scales, mins, ld_s, N, K, group, *rest):
        groups = -(-K // group)
        assert ld >= K // 2 and ld_s >= groups
        self.seen = dict(codes=(codes, ld, N, K // 2, 1), scales=(scales, ld_s, N, groups, 2))
        if mins:
            self.seen["mins"] = (mins, ld_s, N, groups, 2)
        return 0

    def dsb_int4_quantize(self, W, ld, bf16, N, K, *rest):
        assert ld >= K
        self.seen = dict(W=(W, ld, N, K, 2 if bf16 else 4))
        return 0

    def dsb_int4_from_gguf(self, qtype, raw, row_bytes, N, K, *rest):
        self.seen = dict(raw=(raw, row_bytes, N, K // 32 * 18, 1))
        return 0


@pytest.fixture
def fake(dsb, monkeypatch):
    from diffsynth_engine_b200 import int4
    lib, held = _Reads(), []
    monkeypatch.setattr(int4, "_require_cuda", lambda *ts: None)
    monkeypatch.setattr(int4, "_stream", lambda: 0)
    monkeypatch.setattr(int4._lib, "lib", lambda: lib)

    def ptr(t):          # (keeps what the call reads, and knows how far each goes)
        if t is None:
            return None
        held.append(t)
        return t.data_ptr()

    monkeypatch.setattr(int4, "_ptr", ptr)

    def read(name, want):
        at, ld, n, cols, size = lib.seen[name]
        t = next(t for t in held if t.data_ptr() == at and t.shape == want.shape)
        end = t.untyped_storage().data_ptr() + t.untyped_storage().nbytes()
        assert n == 1 or at + ((n - 1) * ld + cols) * size <= end, f"{name}: {n} rows {ld} apart pass the end of the tensor"
        assert torch.equal(lib.rows(at, ld, n, cols, size), want.contiguous().view(torch.uint8).view(n, -1))

    return int4, read


@pytest.mark.parametrize("overlap", ["expanded", "window", "one row", "plain"])
@pytest.mark.parametrize("mins", [False, True])
def test_rows_that_overlap(fake, overlap, mins):
    int4, read = fake
    N, K = (1, 128) if overlap == "one row" else (9, 128)

    def rows(n, cols, dtype):
        base = torch.arange(1, n * cols + 1).remainder(120).to(dtype)
        if overlap == "expanded":
            return base[:cols].clone()[None].expand(n, cols)
        if overlap == "window":
            return base[:cols + n - 1].clone().as_strided((n, cols), (1, 1))
        if overlap == "one row":
            return base[:cols].clone().as_strided((1, cols), (1, 1))
        return base.view(n, cols)

    codes, scales, m = rows(N, K // 2, torch.uint8), rows(N, K // 32, torch.float16), rows(N, K // 32, torch.float16) if mins else None
    int4.from_codes(codes, scales, m)
    read("codes", codes)
    read("scales", scales)
    if mins:
        read("mins", m)
    for dtype in (torch.float32, torch.bfloat16):
        W = rows(N, K, dtype)
        int4.quantize_codes(W)
        read("W", W)
    raw = rows(N, K // 32 * 18, torch.uint8)
    int4.gguf_codes(raw, "Q4_0")
    read("raw", raw)

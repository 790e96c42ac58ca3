"""The records by which the streams of kv_attn_kernel hand an item over to the combine pass, checked on the CPU: a record that a stream did
not write, because a wait of its ran out, is whatever the workspace held, and must not become an address."""
import ctypes
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "diffsynth-engine_b200", "csrc")
SHIM = """
#include "kv_index.h"
extern "C" int t_cut_ok(int pair, int h, int more, int slot, int stream, int pairs, int heads, int n_streams) {
  return dsb::kv_cut_ok(pair, h, more, slot, stream, pairs, heads, n_streams);
}
"""


@pytest.fixture(scope="module")
def ok(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv_records")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-fsanitize=signed-integer-overflow", "-fsanitize-undefined-trap-on-error", "-I", CSRC,
                    str(d / "shim.cpp"), "-o", str(d / "shim.so")], check=True)
    lib = ctypes.CDLL(str(d / "shim.so"))
    return lambda *a: bool(lib.t_cut_ok(*a))


def test_records_name_items_and_streams_that_there_are(ok):
    pairs, heads, streams = 7, 3, 50
    for rec in ((0, 0, 1, 0), (6, 2, 1, 1), (3, 1, 48, 0)):
        assert ok(*rec, 1, pairs, heads, streams)
    big = (1 << 31) - 1
    for rec in ((-1, 0, 0, 0), (7, 0, 1, 0), (0, 3, 1, 0), (0, -1, 1, 0), (0, 0, 0, 0), (0, 0, -1, 0), (0, 0, 49, 0), (0, 0, 1, 2), (0, 0, 1, -1),
                (big, big, big, big), (-big - 1,) * 4, (0, 0, big, 1)):
        assert not ok(*rec, 1, pairs, heads, streams), rec
    rng = random.Random(0)
    for _ in range(20000):
        pair, h, more, slot = (rng.randrange(-(1 << 31), 1 << 31) if rng.random() < 0.3 else rng.randrange(-2, 60) for _ in range(4))
        stream = rng.randrange(streams)
        if ok(pair, h, more, slot, stream, pairs, heads, streams):
            assert 0 <= pair < pairs and 0 <= h < heads and slot in (0, 1) and 1 <= more and stream + more < streams


def test_every_stream_has_a_record_before_its_first_wait():
    """In the kernel's source: the empty record stands behind the CTA's barrier and ahead of the consumers' first wait."""
    with open(os.path.join(CSRC, "kvcache.cu")) as f:
        body = f.read().split("kv_attn_kernel(", 1)[1].split("kv_combine_kernel", 1)[0]
    body = body[body.index("- consumers"):]
    first = body.index("cuts[stream0 + st] = {-1, 0, 0, 0}")
    assert body.index("__syncthreads()") < first < body.index("mbar_wait_all(")

"""The work split over the 4-bit cache (csrc/s14_attn_plan.h), compiled for the
host: the limits of the 8-bit cache's, with room for the chunk's word at the
workspace's end, and a balanced plan's chunks whatever the lengths are."""

from __future__ import annotations

import ctypes as C
import itertools
import random
import shutil
import subprocess
from pathlib import Path

import pytest

from test_attention_plan import LAYOUTS, REACH, cut

ROOT = Path(__file__).resolve().parents[1]


class Plan:
    def __init__(self, v):
        self.row_tiles, self.rec_rows, self.chunk, self.chunks, self.fused, self.blocks, self.fill, self.least = v


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    if not shutil.which("g++"):
        pytest.skip("g++ not available")
    out = tmp_path_factory.mktemp("attnplan4") / "libattnplan4.so"
    subprocess.run(
        ["g++", "-O2", "-std=c++17", "-Wall", "-Werror", "-fPIC", "-shared", f"-I{ROOT / 'colormlm_amd' / 'csrc'}",
         str(ROOT / "tests" / "native" / "attention_plan4_check.cpp"), "-o", str(out)],
        check=True,
    )
    return C.CDLL(str(out))


def plan(lib, seqs, heads, kv, dim, max_new, max_len, window=0, reach=REACH):
    out = (C.c_uint64 * 8)()
    lib.attn_plan((C.c_uint32 * 8)(seqs, heads, kv, dim, max_new, max_len, window, reach), out)
    return Plan(list(out))


@pytest.mark.parametrize("heads,kv,dim", LAYOUTS)
def test_split_of_every_promise(lib, heads, kv, dim):
    rng = random.Random(heads * dim)
    part, counters = C.c_uint64(), C.c_uint32()
    lib.attn_limits(C.byref(part), C.byref(counters))
    balanced = 0
    for seqs, new, most in itertools.product((1, 2, 8, 100, 256, 257), (1, 2, 8, 33, 64, 200), (0, 1, 63, 500, 9000, 70000, REACH)):
        p = plan(lib, seqs, heads, kv, dim, new, most, rng.choice((0, 0, 64, 4096)))
        what = (seqs, heads, kv, dim, new, most, vars(p))
        rows = new * (heads // kv)
        tiles = -(-rows // (16 * p.row_tiles))
        assert p.chunk >= 64 and p.chunk % 64 == 0 and p.chunks >= 1, what
        assert p.blocks == tiles * kv * seqs * p.chunks, what
        if p.chunks > 1:
            assert p.blocks * p.rec_rows * (dim + 4) + 4 <= part.value, what
        if p.fused:
            assert p.row_tiles == 1 and p.rec_rows <= 4 and p.chunks <= 64 and tiles * kv * seqs <= counters.value, what
        if not p.fill:
            continue
        balanced += 1
        assert p.chunks > 1 and 1 < seqs <= 256 and p.least >= 64 and p.least % 64 == 0, what
        # the chunk that the device takes: 64 times the steps in all over fill, `least` at least
        for _ in range(20):
            lengths = [rng.choice((0, 1, rng.randrange(1, max(2, min(most, 1 << 30))), min(REACH, 2 * most))) for _ in range(seqs)]
            steps = [-(-n // 64) for n in lengths]
            each = min(-(-sum(steps) // p.fill), 1 << 24) if sum(steps) >> 31 == 0 else 1 << 24
            size = 64 * max(p.least // 64, each)
            work = 0
            for n in lengths:
                out = (C.c_uint32 * 2)()
                lib.attn_cut(C.c_uint32(n), C.c_uint32(size), C.c_uint32(p.chunks), out)
                chunk, chunks = out
                assert chunk % 64 == 0 and chunk >= size and chunks <= p.chunks and chunk * chunks >= n, what
                work += chunks
            assert work <= p.fill + seqs, what  # one each more than the card holds, at the most
    assert balanced > 0 or dim in (64, 256) or heads // kv == 1

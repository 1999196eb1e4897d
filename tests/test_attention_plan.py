"""paged_attention's work split (csrc/s14_attn_plan.h), compiled for the host:
whatever a call promises about its lengths, every chunk is a whole number of
64-token steps, the partial results and the arrival counters stay in the
context's, a launch without partial results has one chunk, and the chunks of
any sequence cover it, the one that nothing of is seen too."""

from __future__ import annotations

import ctypes as C
import itertools
import random
import shutil
import subprocess
from dataclasses import dataclass
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
REACH = (1 << 31) - (1 << 16)  # the longest sequence a page table may have


@dataclass
class Plan:
    row_tiles: int
    rec_rows: int
    chunk: int
    chunks: int
    fused: int
    blocks: int


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    if not shutil.which("g++"):
        pytest.skip("g++ not available")
    out = tmp_path_factory.mktemp("attnplan") / "libattnplan.so"
    subprocess.run(
        ["g++", "-O2", "-std=c++17", "-Wall", "-Werror", "-fPIC", "-shared", f"-I{ROOT / 'colormlm_amd' / 'csrc'}",
         str(ROOT / "tests" / "native" / "attention_plan_check.cpp"), "-o", str(out)],
        check=True,
    )
    return C.CDLL(str(out))


def plan(lib, seqs, heads, kv, dim, max_new, max_len, window=0, reach=REACH):
    out = (C.c_uint64 * 6)()
    lib.attn_plan((C.c_uint32 * 8)(seqs, heads, kv, dim, max_new, max_len, window, reach), out)
    return Plan(*out)


def cut(lib, p, span):
    out = (C.c_uint32 * 2)()
    lib.attn_cut(C.c_uint32(span), C.c_uint32(p.chunk), C.c_uint32(p.chunks), out)
    return list(out)


LAYOUTS = [(32, 8, 128), (64, 8, 64), (16, 16, 64), (12, 2, 256), (64, 1, 512), (7, 1, 64), (128, 1, 512)]


def check(lib, seqs, heads, kv, dim, max_new, max_len, window=0, reach=REACH):
    p = plan(lib, seqs, heads, kv, dim, max_new, max_len, window, reach)
    part, counters = C.c_uint64(), C.c_uint32()
    lib.attn_limits(C.byref(part), C.byref(counters))
    what = (seqs, heads, kv, dim, max_new, max_len, window, p)
    assert p.chunk >= 64 and p.chunk % 64 == 0 and p.chunks >= 1, what
    rows = max_new * (heads // kv)
    tiles = -(-rows // (16 * p.row_tiles))
    assert p.blocks == tiles * kv * seqs * p.chunks, what
    if p.chunks > 1:
        assert p.blocks * p.rec_rows * (dim + 4) <= part.value, what
        if p.fused:  # only the kernels of one row tile join their own chunks
            assert p.row_tiles == 1 and p.rec_rows <= 4, what
            assert p.chunks <= 64 and tiles * kv * seqs <= counters.value, what
    for span in (0, 1, 63, 64, 65, max_len, 5 * max_len, p.chunk, p.chunk * p.chunks, 1_000_003, REACH):
        if span > REACH:
            continue
        chunk, chunks = cut(lib, p, span)
        assert chunk >= 64 and chunk % 64 == 0 and chunks <= p.chunks, (what, span)
        assert chunks * chunk >= span and (chunks - 1) * chunk < max(span, 1), (what, span)
        # each chunk's end, in the kernels' 31 bits, where the span starts at position 0 and as late as it may
        for lo in (0, (REACH - span) & ~63):
            for i in {0, chunks - 1} if chunks else ():
                begin = lo + i * chunk
                assert lib.attn_end(begin, lo + span, C.c_uint32(chunk)) == min(lo + span, begin + chunk), (what, span, lo)
    return p


@pytest.mark.parametrize("heads,kv,dim", LAYOUTS)
def test_split_of_every_promise(lib, heads, kv, dim):
    rng = random.Random(heads * dim)
    for seqs, new, most in itertools.product((1, 2, 8, 100), (1, 2, 8, 33, 64, 200), (1, 63, 64, 500, 9000, 70000)):
        check(lib, seqs, heads, kv, dim, new, most)
        check(lib, seqs, heads, kv, dim, new, most, rng.choice((1, 64, 500, 4096)))


@pytest.mark.parametrize("heads,kv,dim", LAYOUTS)
@pytest.mark.parametrize("window", [0, 1, 500])
def test_split_without_cached_tokens(lib, heads, kv, dim, window):
    """max_len 0, the longest of a batch of empty sequences: their rows see
    nothing, which is one chunk of no tokens."""
    for seqs, new in itertools.product((1, 3, 128), (1, 4, 8, 40)):
        p = check(lib, seqs, heads, kv, dim, new, 0, window)
        assert p.chunks == 1 and cut(lib, p, 0)[1] <= 1


@pytest.mark.parametrize("heads,kv,dim", LAYOUTS)
@pytest.mark.parametrize("max_len", [REACH, (1 << 31) - 256, (1 << 31) - 255, (1 << 31) - 1])
@pytest.mark.parametrize("window", [0, 1 << 30])
def test_split_of_the_longest_promise(lib, heads, kv, dim, max_len, window):
    """A max_len that promises nothing, up to the largest that is accepted: the
    page table's reach sets the split, and no chunk passes 31 bits."""
    for seqs, new, reach in itertools.product((1, 4, 96, 256), (1, 8, 64, 512, 2048, 1 << 20), (64, 12_000, REACH)):
        p = check(lib, seqs, heads, kv, dim, new, max_len, window, reach)
        assert p.chunk < 1 << 31 and p.chunk * p.chunks < reach + 256 * p.chunks
        assert p == plan(lib, seqs, heads, kv, dim, new, reach, window, reach)

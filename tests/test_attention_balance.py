"""The chunks of balanced launches over the 4-bit cache (csrc/s14_attn_plan.h),
compiled for the host: what the device makes of the sequences' lengths."""

from __future__ import annotations

import ctypes as C
import random
import shutil
import subprocess
from pathlib import Path

import pytest

from test_attention_plan import REACH
from test_attention_plan4 import lib, plan  # noqa: F401

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def steps(tmp_path_factory):
    """Steps of a chunk by the steps held in all, the workgroups and the least chunk."""
    if not shutil.which("g++"):
        pytest.skip("g++ not available")
    out = tmp_path_factory.mktemp("attnbalance") / "libattnbalance.so"
    subprocess.run(
        ["g++", "-O2", "-std=c++17", "-Wall", "-Werror", "-fPIC", "-shared", f"-I{ROOT / 'colormlm_amd' / 'csrc'}",
         str(ROOT / "tests" / "native" / "attention_balance_check.cpp"), "-o", str(out)],
        check=True,
    )
    host = C.CDLL(str(out))
    f = host.attn_balanced
    f.argtypes, f.restype = (C.c_uint64, C.c_uint32, C.c_uint32), C.c_uint32
    f.may = host.attn_may_balance
    return f


def test_steps_of_a_chunk(steps):
    rng = random.Random(1)
    for _ in range(3000):
        fill, least = rng.randrange(1, 1025), rng.randrange(1, 17)
        total = rng.choice((0, 1, fill, rng.randrange(2 * fill), rng.randrange(1 << 20), rng.randrange(1 << 33)))
        got = steps(total, fill, least)
        each = min(-(-total // fill), 1 << 24) if total < 1 << 31 else 1 << 24
        root = least * min(1.0, total / fill) ** 0.5
        if each > least:
            assert got == each, (total, fill, least)
        else:  # the root to the nearest, or what fills the workgroups
            assert got == max(1, each) or abs(got - root) <= 0.5 + 1e-9, (total, fill, least)
            assert got >= each and got >= root - 0.5 - 1e-9 and 1 <= got <= max(least, each), (total, fill, least)


# sequences, heads, key heads, head size, new tokens, longest: launches that balance
BALANCED = [(256, 32, 1, 512, 1, 3000), (8, 64, 1, 512, 1, 2048), (4, 64, 1, 512, 4, 5000), (31, 64, 1, 512, 1, 1000),
            (12, 16, 8, 128, 64, 4000), (40, 4, 1, 128, 70, 3000)]


@pytest.mark.parametrize("seqs,heads,kv,dim,new,most", BALANCED)
def test_balanced_launches(lib, seqs, heads, kv, dim, new, most):  # noqa: F811
    assert plan(lib, seqs, heads, kv, dim, new, most).fill
    assert not plan(lib, 257, heads, kv, dim, new, most).fill


@pytest.mark.parametrize("heads,kv,dim,balances", [(64, 1, 512, True), (16, 8, 128, True), (8, 2, 256, False), (8, 8, 64, False)])
def test_which_heads_balance(lib, heads, kv, dim, balances):  # noqa: F811
    found = any(plan(lib, seqs, heads, kv, dim, new, most).fill for seqs in (2, 8, 30, 100, 256) for new in (1, 16, 64, 200)
                for most in (500, 3000, 70000, REACH))
    assert found == balances


@pytest.mark.parametrize("heads,kv,dim", [(64, 1, 512), (9, 1, 512), (16, 8, 128), (125, 1, 128), (31, 1, 128), (8, 2, 256), (8, 8, 64)])
def test_plans_balance_only_for_kernels_that_do(lib, steps, heads, kv, dim):  # noqa: F811
    """A plan with a chunk of the device's for a kernel that was compiled without would
    be joined by another chunk than the one it ran by; a kernel that was compiled with
    has plans that use it."""
    used, may = set(), set()
    for seqs in (2, 3, 8, 30, 100, 256):
        for new in range(1, 300, 3 if dim < 512 else 1):
            for most in (500, 3000, 70000, REACH):
                p = plan(lib, seqs, heads, kv, dim, new, most)
                if steps.may(dim, p.row_tiles):
                    may.add(p.row_tiles)
                if p.fill:
                    used.add(p.row_tiles)
                    assert steps.may(dim, p.row_tiles), (seqs, new, most)
    assert used == may


@pytest.mark.parametrize("heads", [32, 64, 128])
def test_chunks_do_not_jump_with_the_lengths(lib, steps, heads):  # noqa: F811
    """Heads of 512, one token each: a step more of every sequence makes a chunk a
    step longer at the most, from short sequences to long ones."""
    for seqs in (2, 3, 4, 7, 8, 15, 16, 31, 32, 64, 100, 127):
        before = None
        for n in range(192, 20000, 64):
            p = plan(lib, seqs, heads, 1, 512, 1, n)
            assert p.chunks > 1 and (p.fill or p.chunk == 64), (seqs, n)
            size = steps(seqs * n // 64, p.fill, p.least // 64) if p.fill else 1
            assert before is None or 0 <= size - before <= 1, (seqs, n, before, size)
            before = size


@pytest.mark.parametrize("heads,kv,dim,new", [(64, 1, 512, 1), (64, 1, 512, 4), (16, 8, 128, 64)])
def test_chunks_of_a_balanced_launch_are_the_sequence(lib, steps, heads, kv, dim, new):  # noqa: F811
    """End to end, whatever the lengths are: no token left out or taken twice, no
    more chunks than the workspace and the grid have."""
    rng = random.Random(dim + new)
    balanced = 0
    for _ in range(300):
        seqs, most = rng.randrange(2, 65), rng.choice((900, 4096, 20000, REACH))
        p = plan(lib, seqs, heads, kv, dim, new, most)
        if not p.fill:
            continue
        balanced += 1
        lengths = [min(REACH, rng.choice((1, rng.randrange(1, most + 1), most, 2 * most))) for _ in range(seqs)]
        size = 64 * steps(sum(-(-n // 64) for n in lengths), p.fill, p.least // 64)
        for n in lengths:
            out = (C.c_uint32 * 2)()
            lib.attn_cut(C.c_uint32(n), C.c_uint32(size), C.c_uint32(p.chunks), out)
            chunk, chunks = out
            assert chunks <= p.chunks and chunk % 64 == 0
            begin = 0
            for i in range(chunks):
                end = lib.attn_end(C.c_int32(begin), C.c_int32(n), C.c_uint32(chunk))
                assert begin < end <= n and (end == n) == (i == chunks - 1), (n, chunk, i)
                begin = end
    assert balanced > 100

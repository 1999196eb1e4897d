"""Whether two attention operands share memory (csrc/s14_attn_share.h), compiled
for the host, against sets of bytes; and the calls that refuse it."""

from __future__ import annotations

import ctypes as C
import random
import shutil
import subprocess
from pathlib import Path

import pytest

from colormlm_amd import _native as N

ROOT = Path(__file__).resolve().parents[1]
CTX = C.c_void_p(16)  # never read: every call below is refused first
AT = 1 << 20
NONE = N.Buffer(None, 0)
BIG = N.Buffer(1 << 45, 1 << 44)


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    if not shutil.which("g++"):
        pytest.skip("g++ not available")
    out = tmp_path_factory.mktemp("attnshare") / "libattnshare.so"
    subprocess.run(
        ["g++", "-O2", "-std=c++17", "-Wall", "-Werror", "-fPIC", "-shared", f"-I{ROOT / 'colormlm_amd' / 'csrc'}",
         str(ROOT / "tests" / "native" / "attention_share_check.cpp"), "-o", str(out)],
        check=True,
    )
    return C.CDLL(str(out))


def share(lib, a, b, tokens, own):
    return bool(lib.attn_share((C.c_uint64 * 5)(*a), (C.c_uint64 * 5)(*b), C.c_uint32(tokens), int(own)))


def rows_of(x, tokens):
    at, token, head, row, heads = x
    return {(t, h): range(at + t * token + h * head, at + t * token + h * head + row) for t in range(tokens) for h in range(heads)}


def want(a, b, tokens, own):
    ra, rb = rows_of(a, tokens), rows_of(b, tokens)
    return any(max(x[0], y[0]) <= min(x[-1], y[-1]) for i, x in ra.items() for j, y in rb.items()
               if not (own and i == j and a[0] == b[0]))


def test_overlap_against_sets_of_bytes(lib):
    rng = random.Random(5)
    seen = {True: 0, False: 0}
    for _ in range(6000):
        tokens, ha, hb = rng.randint(1, 5), rng.randint(1, 4), rng.randint(1, 4)
        row = rng.choice([4, 8])
        head = rng.choice([row, row, 2 * row, 3 * row, 20])
        token = rng.choice([row, head * 4, head * 8, 3 * head, 9 * row])
        swap = rng.random() < 0.2  # heads outermost
        if swap:
            head, token = max(head, 6 * token), token
        a = (100 + rng.choice([0, 0, row, -row, 4 * head, 2, -40, 500]), token, head, row, ha)
        b = (100, token, head, rng.choice([row, row // 2, 2 * row]), hb)
        own = ha == hb and rng.random() < 0.6
        w = want(a, b, tokens, own)
        assert share(lib, a, b, tokens, own) == w, (a, b, tokens, own)
        seen[w] += 1
    assert min(seen.values()) > 1000


def test_operands_of_other_steps_share_where_their_extents_do(lib):
    a, b = (100, 40, 4, 4, 3), (104, 50, 4, 4, 3)
    assert share(lib, a, b, 2, False) and not share(lib, a, (100 + 40 + 12, 50, 4, 4, 3), 2, False)
    assert share(lib, a, a, 2, False) and not share(lib, a, a, 2, True)


def rows(at, heads, token, head=128, dtype=N.S14_X_BF16):
    return N.Rows(N.Buffer(at, 1 << 40), dtype, heads, token, head)


def refused(rc, text):
    assert rc == N.S14_ERR_INVALID and text in N.last_error(), (rc, N.last_error())


def norm_rope(native, q, k, qo, ko):
    r = C.byref
    return native.s14_qk_norm_rope(CTX, None, 5, 128, r(q), r(k), r(qo), r(ko), NONE, NONE, 1e-6, None, NONE)


F32 = N.S14_X_F32


@pytest.mark.parametrize("text,q,k,qo,ko", [
    # one projection of 4 + 2 heads, 512 and 256 values of its 768: outputs that are not their inputs' rows
    ("q output", (AT, 4, 768), (AT + 1024, 2, 768), (AT + 256, 4, 768), (AT + 1024, 2, 768)),
    ("k output", (AT, 4, 768), (AT + 1024, 2, 768), (AT, 4, 768), (AT + 512, 2, 768)),
    ("q output", (AT, 4, 768), (AT + 1024, 2, 768), (AT + 1024 - 16, 4, 768), (AT + 1024, 2, 768)),
    # bf16 packed into the f32 rows' place
    ("q output", (AT, 4, 512, 128, F32), (1 << 30, 2, 256), (AT, 4, 512), (1 << 31, 2, 256)),
    # both outputs in one place
    ("outputs", (AT, 4, 512), (1 << 30, 4, 512), (1 << 31, 4, 512), (1 << 31, 4, 512)),
])
def test_norm_rope_refuses_outputs_over_other_rows(native, text, q, k, qo, ko):
    refused(norm_rope(native, *(rows(*x) for x in (q, k, qo, ko))), text)


def test_attention_refuses_outputs_over_its_inputs(native):
    r = C.byref
    q, k, v = rows(AT, 4, 1024), rows(AT + 1024, 2, 1024), rows(AT + 1536, 2, 1024)

    def prompt(out):
        return native.s14_prompt_attention(CTX, None, 128, r(q), r(k), r(v), 5, 2, BIG, r(out), NONE, 0.1, 0)

    refused(prompt(rows(AT + 512, 4, 1024)), "shares memory")
    refused(prompt(rows(AT + 1024, 4, 1024)), "shares memory")
    refused(prompt(rows(AT + 1536 - 2048, 4, 1024)), "shares memory")
    cache = N.KvCache(BIG, BIG, BIG, BIG, 10, 2, 64, 128)

    def paged(out):
        return native.s14_paged_attention(CTX, None, r(q), r(cache), 5, 2, 3, 100, BIG, 4, BIG, BIG, r(out), NONE, 0.1, 0)

    refused(paged(rows(AT + 256, 4, 1024)), "shares memory")
    refused(paged(rows(AT, 4, 512)), "shares memory")

"""Refusals of the attention entry points, before any device call: the C ABI
with addresses that are never followed, and the Python layer with CPU tensors."""

from __future__ import annotations

import ctypes as C
import math

import pytest

torch = pytest.importorskip("torch")

from colormlm_amd import _native as N  # noqa: E402
from colormlm_amd import attention as A  # noqa: E402

CTX = C.c_void_p(16)  # never read: every call below is refused first
AT = 1 << 20
HUGE = 1 << 50
BIG = N.Buffer(AT, HUGE)
NONE = N.Buffer(None, 0)


def rows(heads=4, dtype=N.S14_X_BF16, token=512, head=128, buf=BIG):
    return N.Rows(buf, dtype, heads, token, head)


def cache(pages=10, heads=2, page=64, dim=128, **bufs):
    b = dict(k=BIG, v=BIG, k_scale=BIG, v_scale=BIG) | bufs
    return N.KvCache(b["k"], b["v"], b["k_scale"], b["v_scale"], pages, heads, page, dim)


def rope(positions=100, rot=128, start=0, layout=0, table=BIG):
    return N.Rope(table, positions, rot, start, layout)


def ref(x):
    return None if x is None else C.byref(x)


def refused(code, rc, text=""):
    assert rc == code, (rc, N.last_error())
    assert text in N.last_error()


def norm_rope(native, ctx=CTX, tokens=3, dim=128, q=rows(), k=rows(2, token=256), qo=rows(), ko=rows(2, token=256),
              qw=NONE, kw=NONE, eps=1e-6, rp=None, pos=NONE):
    return native.s14_qk_norm_rope(ctx, None, tokens, dim, ref(q), ref(k), ref(qo), ref(ko), qw, kw, eps, ref(rp), pos)


@pytest.mark.parametrize("code,text,kw", [
    (N.S14_ERR_INVALID, "context", dict(ctx=None)),
    (N.S14_ERR_SHAPE, "head size", dict(dim=96)),
    (N.S14_ERR_SHAPE, "tokens", dict(tokens=(1 << 30) + 1)),
    (N.S14_ERR_INVALID, "q rows", dict(q=None)),
    (N.S14_ERR_INVALID, "k rows", dict(k=None)),
    (N.S14_ERR_INVALID, "k output rows", dict(ko=None)),
    (N.S14_ERR_INVALID, "dtype", dict(q=rows(dtype=2))),
    (N.S14_ERR_SHAPE, "heads", dict(q=rows(0))),
    (N.S14_ERR_SHAPE, "heads", dict(qo=rows(5, token=640))),
    (N.S14_ERR_SHAPE, "multiples of 8", dict(q=rows(token=513))),
    (N.S14_ERR_SHAPE, "multiples of 8", dict(q=rows(head=132))),
    (N.S14_ERR_SHAPE, "multiples of 8", dict(q=rows(token=1 << 25))),
    (N.S14_ERR_SHAPE, "below the head size", dict(q=rows(head=64))),
    (N.S14_ERR_SHAPE, "below the head size", dict(q=rows(token=0))),
    (N.S14_ERR_SHAPE, "overlap", dict(qo=rows(token=256))),
    (N.S14_ERR_CAPACITY, "q buffer", dict(q=rows(buf=N.Buffer(AT, 2 * (2 * 512 + 3 * 128 + 128) - 1)))),
    (N.S14_ERR_SHAPE, "aligned", dict(q=rows(buf=N.Buffer(AT + 8, HUGE)))),
    (N.S14_ERR_INVALID, "NULL", dict(q=rows(buf=NONE))),
    (N.S14_ERR_CAPACITY, "weight", dict(qw=N.Buffer(AT, 508))),
    (N.S14_ERR_INVALID, "eps", dict(kw=BIG, eps=-1.0)),
    (N.S14_ERR_INVALID, "eps", dict(kw=BIG, eps=math.nan)),
    (N.S14_ERR_INVALID, "layout", dict(rp=rope(layout=2), pos=BIG)),
    (N.S14_ERR_SHAPE, "rotation", dict(rp=rope(rot=0), pos=BIG)),
    (N.S14_ERR_SHAPE, "rotation", dict(rp=rope(rot=12), pos=BIG)),
    (N.S14_ERR_SHAPE, "rotation", dict(rp=rope(rot=64, start=72), pos=BIG)),
    (N.S14_ERR_SHAPE, "rotation", dict(rp=rope(rot=64, start=4), pos=BIG)),
    (N.S14_ERR_SHAPE, "rotation", dict(rp=rope(rot=8, start=0xFFFFFFF8), pos=BIG)),
    (N.S14_ERR_SHAPE, "positions", dict(rp=rope(positions=0), pos=BIG)),
    (N.S14_ERR_CAPACITY, "rotation table", dict(rp=rope(table=N.Buffer(AT, 100 * 128 * 4 - 1)), pos=BIG)),
    (N.S14_ERR_INVALID, "positions", dict(rp=rope())),
    (N.S14_ERR_CAPACITY, "positions", dict(rp=rope(), pos=N.Buffer(AT, 8))),
])
def test_norm_rope_refusals(native, code, text, kw):
    refused(code, norm_rope(native, **kw), text)


def test_norm_rope_without_tokens_is_no_launch(native):
    assert norm_rope(native, tokens=0) == N.S14_OK


def test_norm_rope_without_tokens_asks_for_no_positions(native):
    """An empty tensor has no address."""
    assert norm_rope(native, tokens=0, rp=rope(), pos=NONE) == N.S14_OK


def append(native, ctx=CTX, c=cache(), tokens=5, seqs=2, most=3, k=rows(2, token=256), v=rows(2, token=256), table=BIG,
           width=4, cu=BIG, past=BIG, kw=NONE, eps=1e-6, rp=None):
    return native.s14_kv_append(ctx, None, ref(c), tokens, seqs, most, ref(k), ref(v), table, width, cu, past, kw, eps,
                                ref(rp))


@pytest.mark.parametrize("code,text,kw", [
    (N.S14_ERR_INVALID, "context", dict(ctx=None)),
    (N.S14_ERR_INVALID, "cache", dict(c=None)),
    (N.S14_ERR_SHAPE, "head size", dict(c=cache(dim=32))),
    (N.S14_ERR_SHAPE, "pages of", dict(c=cache(page=48))),
    (N.S14_ERR_SHAPE, "pages of", dict(c=cache(page=8))),
    (N.S14_ERR_SHAPE, "0 pages", dict(c=cache(pages=0))),
    (N.S14_ERR_SHAPE, "0 heads", dict(c=cache(heads=0))),
    (N.S14_ERR_CAPACITY, "k codes", dict(c=cache(k=N.Buffer(AT, 10 * 2 * 64 * 128 - 1)))),
    (N.S14_ERR_CAPACITY, "v codes", dict(c=cache(v=N.Buffer(AT, 10 * 2 * 64 * 128 - 1)))),
    (N.S14_ERR_CAPACITY, "k scales", dict(c=cache(k_scale=N.Buffer(AT, 19)))),
    (N.S14_ERR_INVALID, "v scales", dict(c=cache(v_scale=NONE))),
    (N.S14_ERR_SHAPE, "aligned", dict(c=cache(v=N.Buffer(AT + 4, HUGE)))),
    (N.S14_ERR_SHAPE, "sequences", dict(seqs=65536)),
    (N.S14_ERR_INVALID, "longest", dict(most=6)),
    (N.S14_ERR_SHAPE, "heads", dict(k=rows(4))),
    (N.S14_ERR_SHAPE, "heads", dict(v=rows(1, token=128))),
    (N.S14_ERR_SHAPE, "page table", dict(width=0)),
    (N.S14_ERR_CAPACITY, "page table", dict(table=N.Buffer(AT, 31))),
    (N.S14_ERR_CAPACITY, "cu", dict(cu=N.Buffer(AT, 11))),
    (N.S14_ERR_CAPACITY, "past", dict(past=N.Buffer(AT, 7))),
    (N.S14_ERR_SHAPE, "aligned", dict(past=N.Buffer(AT + 2, HUGE))),
    (N.S14_ERR_INVALID, "past", dict(past=NONE)),
    (N.S14_ERR_INVALID, "eps", dict(kw=BIG, eps=math.inf)),
    (N.S14_ERR_SHAPE, "rotation", dict(rp=rope(rot=256))),
])
def test_append_refusals(native, code, text, kw):
    refused(code, append(native, **kw), text)


def test_append_without_tokens_is_no_launch(native):
    assert append(native, tokens=0, most=0) == N.S14_OK
    assert append(native, seqs=0) == N.S14_OK


def paged(native, ctx=CTX, q=rows(), c=cache(), tokens=5, seqs=2, most=3, length=100, table=BIG, width=4, cu=BIG,
          lens=BIG, out=rows(), lse=NONE, scale=0.1, window=0):
    return native.s14_paged_attention(ctx, None, ref(q), ref(c), tokens, seqs, most, length, table, width, cu, lens,
                                      ref(out), lse, scale, window)


@pytest.mark.parametrize("code,text,kw", [
    (N.S14_ERR_INVALID, "context", dict(ctx=None)),
    (N.S14_ERR_INVALID, "q rows", dict(q=None)),
    (N.S14_ERR_INVALID, "bf16", dict(q=rows(dtype=N.S14_X_F32))),
    (N.S14_ERR_SHAPE, "divide", dict(q=rows(3), out=rows(3))),
    (N.S14_ERR_INVALID, "out rows", dict(out=None)),
    (N.S14_ERR_SHAPE, "heads", dict(out=rows(2))),
    (N.S14_ERR_CAPACITY, "lse", dict(lse=N.Buffer(AT, 79))),
    (N.S14_ERR_INVALID, "scale", dict(scale=0.0)),
    (N.S14_ERR_INVALID, "scale", dict(scale=-1.0)),
    (N.S14_ERR_INVALID, "scale", dict(scale=math.nan)),
    (N.S14_ERR_INVALID, "scale", dict(scale=math.inf)),
    (N.S14_ERR_SHAPE, "longest", dict(length=1 << 31)),
    (N.S14_ERR_INVALID, "longest", dict(most=6)),
    (N.S14_ERR_CAPACITY, "lens", dict(lens=N.Buffer(AT, 4))),
    (N.S14_ERR_SHAPE, "positions", dict(width=1 << 24, c=cache(page=128))),
    (N.S14_ERR_SHAPE, "one launch", dict(tokens=1 << 29, most=1 << 29, q=rows(32, token=4096), out=rows(32, token=4096),
                                         seqs=64)),
])
def test_paged_refusals(native, code, text, kw):
    refused(code, paged(native, **kw), text)


def prompt(native, ctx=CTX, dim=128, q=rows(), k=rows(2, token=256), v=rows(2, token=256), tokens=5, seqs=2, cu=BIG,
           out=rows(), lse=NONE, scale=0.1, window=0):
    return native.s14_prompt_attention(ctx, None, dim, ref(q), ref(k), ref(v), tokens, seqs, cu, ref(out), lse, scale,
                                       window)


@pytest.mark.parametrize("code,text,kw", [
    (N.S14_ERR_INVALID, "context", dict(ctx=None)),
    (N.S14_ERR_SHAPE, "head size", dict(dim=512)),
    (N.S14_ERR_INVALID, "bf16", dict(k=rows(2, dtype=N.S14_X_F32, token=256))),
    (N.S14_ERR_SHAPE, "below the head size", dict(k=rows(1, token=0))),
    (N.S14_ERR_SHAPE, "k has", dict(v=rows(1, token=256))),
    (N.S14_ERR_SHAPE, "divide", dict(k=rows(3), v=rows(3))),
    (N.S14_ERR_CAPACITY, "cu", dict(cu=N.Buffer(AT, 8))),
    (N.S14_ERR_CAPACITY, "out", dict(out=rows(buf=N.Buffer(AT, 64)))),
    (N.S14_ERR_INVALID, "scale", dict(scale=0.0)),
    (N.S14_ERR_SHAPE, "one launch", dict(tokens=1 << 30, q=rows(64, token=8192), out=rows(64, token=8192))),
])
def test_prompt_refusals(native, code, text, kw):
    refused(code, prompt(native, **kw), text)


def test_prompt_without_tokens_is_no_launch(native):
    assert prompt(native, tokens=0) == N.S14_OK
    assert prompt(native, seqs=0) == N.S14_OK


@pytest.mark.parametrize("code,text,args", [
    (N.S14_ERR_SHAPE, "rotation table", (0, 64, 1e4, None, BIG)),
    (N.S14_ERR_SHAPE, "rotation table", (8, 12, 1e4, None, BIG)),
    (N.S14_ERR_SHAPE, "rotation table", (8, 1024, 1e4, None, BIG)),
    (N.S14_ERR_INVALID, "base", (8, 64, 1.0, None, BIG)),
    (N.S14_ERR_INVALID, "base", (8, 64, math.nan, None, BIG)),
    (N.S14_ERR_INVALID, "scaling", (8, 64, 1e4, (0.0, 0.0, 0.0, 0.0, 1.0), BIG)),
    (N.S14_ERR_INVALID, "scaling", (8, 64, 1e4, (2.0, -1.0, 32.0, 1.0, 1.0), BIG)),
    (N.S14_ERR_INVALID, "turns", (8, 64, 1e4, (2.0, 4096.0, 1.0, 32.0, 1.0), BIG)),
    (N.S14_ERR_CAPACITY, "rotation table", (8, 64, 1e4, None, N.Buffer(AT, 8 * 64 * 4 - 1))),
])
def test_rope_table_refusals(native, code, text, args):
    positions, rot, theta, scaling, table = args
    s = None if scaling is None else C.byref(N.RopeScaling(*scaling))
    refused(code, native.s14_rope_table(CTX, None, positions, rot, theta, s, table), text)


class FakeContext:
    device, handle, _h = 0, CTX, CTX


def test_python_layer_refuses_cpu_tensors_and_bad_caches():
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)  # noqa: E731
    k, v, s = u8(3, 2, 16, 64), u8(3, 2, 64, 16), u8(3, 2)
    A.KvCache(k, s, v, s.clone())
    for bad in ((k, s, k, s), (k, s, v, u8(3, 1)), (k[0], s, v, s), (k.float(), s, v, s), (k, s, v.transpose(2, 3), s)):
        with pytest.raises(N.S14Error):
            A.KvCache(*bad)
    with pytest.raises(N.S14Error, match="layout"):
        A.Rope(torch.zeros(4, 8), "pairs")
    with pytest.raises(N.S14Error):
        A.Rope(torch.zeros(4, 8, dtype=torch.float64))
    with pytest.raises(N.S14Error):
        A.Rope(torch.zeros(4, 8), start=-8)
    x = torch.zeros(2, 2, 64)
    with pytest.raises(N.S14Error, match="context's device"):
        A.qk_norm_rope(FakeContext(), x, None, x, None)
    with pytest.raises(N.S14Error, match="context's device"):
        A.prompt_attention(FakeContext(), x, x, x, torch.zeros(2, dtype=torch.int32), x)


class CpuContext:
    """A context of no GPU: its calls end at the tensors' checks."""

    device, handle, _h = -1, CTX, CTX


@pytest.mark.parametrize("swap", [lambda t: t.resize_(2 * t.shape[0], *t.shape[1:]), lambda t: t.set_(torch.zeros_like(t)),
                                  lambda t: setattr(t, "data", torch.zeros_like(t))])
@pytest.mark.parametrize("which", range(5))
def test_other_memory_behind_a_cache_or_rotation_is_refused(swap, which):
    """A cache and a rotation are made of addresses: a tensor that has other
    memory since would leave calls writing to what was freed."""
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)  # noqa: E731
    tensors = [u8(3, 2, 16, 64), u8(3, 2), u8(3, 2, 64, 16), u8(3, 2)]
    cache, table = A.KvCache(*tensors), torch.zeros(4, 64)
    rope = A.Rope(table)
    swap([*tensors, table][which])
    x, i = torch.zeros(2, 2, 64), torch.zeros(2, dtype=torch.int32)
    ctx, pages = CpuContext(), torch.zeros(1, 1, dtype=torch.int32)
    what = "rotation" if which == 4 else "cache"
    with pytest.raises(N.S14Error, match=f"the {what} was made of other memory"):
        A.kv_append(ctx, cache, x, x, pages, i, i, rope=rope)
    with pytest.raises(N.S14Error, match=f"the {what} was made of other memory"):
        if which == 4:
            A.qk_norm_rope(ctx, x, None, x, None, rope=rope, positions=i)
        else:
            A.paged_attention(ctx, x.bfloat16(), cache, pages, i, i, x)


@pytest.mark.parametrize("start", [1 << 32, (1 << 32) + 8, 1 << 40, -(1 << 32)])
def test_rotation_start_past_32_bits_is_refused(start):
    """It would be another one in the call's 32 bits."""
    with pytest.raises(N.S14Error, match="start"):
        A.Rope(torch.zeros(4, 8), start=start)


@pytest.mark.parametrize("dim,tokens,heads", [(512, 1 << 26, 1), (256, 1 << 27, 1), (64, 1 << 23, 64), (128, 1 << 23, 32)])
def test_more_rows_than_a_launch_has_threads_are_refused(native, dim, tokens, heads):
    x = rows(heads, token=heads * dim, head=dim)
    refused(N.S14_ERR_SHAPE, norm_rope(native, tokens=tokens, dim=dim, q=x, k=rows(0), qo=x, ko=rows(0)), "one launch")


def test_a_table_past_a_launch_is_refused(native):
    refused(N.S14_ERR_SHAPE, native.s14_rope_table(CTX, None, 1 << 27, 64, 1e4, None, BIG), "one launch")


def test_strides_of_single_heads_are_not_asked_for():
    """torch may give a dimension of one any stride: such a call ends at the next
    thing that is wrong with it, here its eps."""
    x = torch.zeros(2, 64).as_strided((2, 1, 64), (64, 1 << 33, 1))
    with pytest.raises(N.S14Error, match="eps"):
        A.qk_norm_rope(CpuContext(), x, None, x, None, q_weight=torch.ones(64), eps=-1.0, stream=0)

"""Refusals of the 4-bit cache's entry points and of add_rms_norm, before any
device call: the C ABI with addresses that are never followed, and the Python
layer with CPU tensors."""

from __future__ import annotations

import ctypes as C
import math

import pytest

torch = pytest.importorskip("torch")

from test_attention_args import AT, BIG, CTX, HUGE, NONE, CpuContext, FakeContext, ref, refused, rope, rows  # noqa: E402

from colormlm_amd import _native as N  # noqa: E402
from colormlm_amd import attention as A  # noqa: E402


def cache(pages=10, heads=2, page=64, dim=128, **bufs):
    b = dict(k=BIG, v=BIG, k_scale=BIG, v_scale=BIG) | bufs
    return N.Kv4Cache(b["k"], b["v"], b["k_scale"], b["v_scale"], pages, heads, page, dim)


def append(native, ctx=CTX, c=cache(), tokens=5, seqs=2, most=3, k=rows(2, token=256), v=rows(2, token=256), table=BIG,
           width=4, cu=BIG, past=BIG, kw=NONE, eps=1e-6, rp=None):
    return native.s14_kv4_append(ctx, None, ref(c), tokens, seqs, most, ref(k), ref(v), table, width, cu, past, kw, eps,
                                 ref(rp))


def paged(native, ctx=CTX, q=rows(), c=cache(), tokens=5, seqs=2, most=3, length=100, table=BIG, width=4, cu=BIG,
          lens=BIG, out=rows(), lse=NONE, scale=0.1, window=0):
    return native.s14_paged4_attention(ctx, None, ref(q), ref(c), tokens, seqs, most, length, table, width, cu, lens,
                                       ref(out), lse, scale, window)


@pytest.mark.parametrize("call", [append, paged])
@pytest.mark.parametrize("code,text,kw", [
    (N.S14_ERR_INVALID, "context", dict(ctx=None)),
    (N.S14_ERR_INVALID, "cache", dict(c=None)),
    (N.S14_ERR_SHAPE, "head size", dict(c=cache(dim=32))),
    (N.S14_ERR_SHAPE, "head size", dict(c=cache(dim=192))),
    (N.S14_ERR_SHAPE, "pages of", dict(c=cache(page=48))),
    (N.S14_ERR_SHAPE, "pages of", dict(c=cache(page=256))),
    (N.S14_ERR_SHAPE, "0 pages", dict(c=cache(pages=0))),
    (N.S14_ERR_SHAPE, "heads", dict(c=cache(heads=0))),
    (N.S14_ERR_CAPACITY, "k codes", dict(c=cache(k=N.Buffer(AT, 10 * 2 * 64 * 64 - 1)))),
    (N.S14_ERR_CAPACITY, "v codes", dict(c=cache(v=N.Buffer(AT, 10 * 2 * 64 * 64 - 1)))),
    (N.S14_ERR_CAPACITY, "k scales", dict(c=cache(k_scale=N.Buffer(AT, 10 * 2 * 64 * 4 - 1)))),
    (N.S14_ERR_CAPACITY, "v scales", dict(c=cache(v_scale=N.Buffer(AT, 10 * 2 * 64 - 1)))),
    (N.S14_ERR_INVALID, "v scales", dict(c=cache(v_scale=NONE))),
    (N.S14_ERR_SHAPE, "aligned", dict(c=cache(v=N.Buffer(AT + 8, HUGE)))),
    (N.S14_ERR_SHAPE, "aligned", dict(c=cache(k_scale=N.Buffer(AT + 4, HUGE)))),
    (N.S14_ERR_SHAPE, "sequences", dict(seqs=65536)),
    (N.S14_ERR_INVALID, "longest", dict(most=6)),
    (N.S14_ERR_SHAPE, "page table", dict(width=0)),
    (N.S14_ERR_CAPACITY, "page table", dict(table=N.Buffer(AT, 31))),
    (N.S14_ERR_CAPACITY, "cu", dict(cu=N.Buffer(AT, 11))),
])
def test_cache_refusals(native, call, code, text, kw):
    refused(code, call(native, **kw), text)


@pytest.mark.parametrize("code,text,kw", [
    (N.S14_ERR_SHAPE, "heads", dict(k=rows(4))),
    (N.S14_ERR_SHAPE, "heads", dict(v=rows(1, token=128))),
    (N.S14_ERR_CAPACITY, "past", dict(past=N.Buffer(AT, 7))),
    (N.S14_ERR_INVALID, "past", dict(past=NONE)),
    (N.S14_ERR_INVALID, "eps", dict(kw=BIG, eps=math.inf)),
    (N.S14_ERR_SHAPE, "rotation", dict(rp=rope(rot=256))),
    (N.S14_ERR_SHAPE, "one launch", dict(tokens=1 << 30, c=cache(heads=1), k=rows(1, token=128), v=rows(1, token=128))),
])
def test_append_refusals(native, code, text, kw):
    refused(code, append(native, **kw), text)


@pytest.mark.parametrize("code,text,kw", [
    (N.S14_ERR_INVALID, "bf16", dict(q=rows(dtype=N.S14_X_F32))),
    (N.S14_ERR_SHAPE, "divide", dict(q=rows(3), out=rows(3))),
    (N.S14_ERR_SHAPE, "heads", dict(out=rows(2))),
    (N.S14_ERR_CAPACITY, "lse", dict(lse=N.Buffer(AT, 79))),
    (N.S14_ERR_INVALID, "scale", dict(scale=0.0)),
    (N.S14_ERR_INVALID, "scale", dict(scale=math.nan)),
    (N.S14_ERR_SHAPE, "longest", dict(length=1 << 31)),
    (N.S14_ERR_CAPACITY, "lens", dict(lens=N.Buffer(AT, 4))),
    (N.S14_ERR_SHAPE, "positions", dict(width=1 << 24, c=cache(page=128))),
    (N.S14_ERR_SHAPE, "one launch", dict(tokens=1 << 29, most=1 << 29, q=rows(32, token=4096), out=rows(32, token=4096),
                                         seqs=64)),
])
def test_paged_refusals(native, code, text, kw):
    refused(code, paged(native, **kw), text)


def test_no_tokens_are_no_launch(native):
    assert append(native, tokens=0, most=0) == N.S14_OK and append(native, seqs=0) == N.S14_OK
    assert paged(native, tokens=0, most=0) == N.S14_OK and paged(native, seqs=0) == N.S14_OK


def flat(k=512, dtype=N.S14_X_F32, at=AT, stride=None, heads=1, size=HUGE):
    return N.Rows(N.Buffer(at, size), dtype, heads, k if stride is None else stride, 0)


FAR = [AT + (i << 32) for i in range(8)]


def norm(native, ctx=CTX, n=4, k=512, x=flat(at=FAR[0]), r=flat(at=FAR[1]), ro=flat(at=FAR[2]), y=flat(at=FAR[3]),
         w=N.Buffer(FAR[4], HUGE), eps=1e-6, group=128, q=N.Buffer(FAR[5], HUGE), s=N.Buffer(FAR[6], HUGE)):
    return native.s14_add_rms_norm(ctx, None, n, k, ref(x), ref(r), ref(ro), ref(y), w, eps, group, q, s)


ROW = 4 * 512 * 4  # bytes of four f32 rows


@pytest.mark.parametrize("code,text,kw", [
    (N.S14_ERR_INVALID, "context", dict(ctx=None)),
    (N.S14_ERR_SHAPE, "rows", dict(n=(1 << 30) + 1)),
    (N.S14_ERR_SHAPE, "multiples of 8", dict(k=0)),
    (N.S14_ERR_SHAPE, "multiples of 8", dict(k=516, group=0)),
    (N.S14_ERR_SHAPE, "multiples of 8", dict(k=65544, group=0)),
    (N.S14_ERR_SHAPE, "group", dict(group=16)),
    (N.S14_ERR_SHAPE, "whole groups", dict(k=448)),
    (N.S14_ERR_INVALID, "asked for", dict(y=None, group=0)),
    (N.S14_ERR_INVALID, "x rows", dict(x=None)),
    (N.S14_ERR_INVALID, "dtype", dict(x=flat(dtype=7))),
    (N.S14_ERR_SHAPE, "heads", dict(r=flat(heads=2, stride=1024, at=FAR[1]))),
    (N.S14_ERR_SHAPE, "multiples of 8", dict(y=flat(stride=516, at=FAR[3]))),
    (N.S14_ERR_SHAPE, "below", dict(ro=flat(stride=504, at=FAR[2]))),
    (N.S14_ERR_CAPACITY, "residual buffer", dict(r=flat(at=FAR[1], size=ROW - 1))),
    (N.S14_ERR_SHAPE, "aligned", dict(x=flat(at=FAR[0] + 8))),
    (N.S14_ERR_INVALID, "weight", dict(w=NONE)),
    (N.S14_ERR_CAPACITY, "weight", dict(w=N.Buffer(FAR[4], 2047))),
    (N.S14_ERR_INVALID, "eps", dict(eps=-1.0)),
    (N.S14_ERR_INVALID, "eps", dict(eps=math.nan)),
    (N.S14_ERR_INVALID, "codes", dict(q=NONE)),
    (N.S14_ERR_CAPACITY, "codes", dict(q=N.Buffer(FAR[5], 2047))),
    (N.S14_ERR_SHAPE, "aligned", dict(q=N.Buffer(FAR[5] + 4, HUGE))),
    (N.S14_ERR_CAPACITY, "scales", dict(s=N.Buffer(FAR[6], 15))),
    (N.S14_ERR_SHAPE, "one launch", dict(n=1 << 30)),
    # rows in another row's place, and in another operand's
    (N.S14_ERR_INVALID, "share", dict(y=flat(at=FAR[0] + 2048))),
    (N.S14_ERR_INVALID, "share", dict(ro=flat(at=FAR[1], stride=1024))),
    (N.S14_ERR_INVALID, "share", dict(y=flat(at=FAR[1], dtype=N.S14_X_BF16))),
    (N.S14_ERR_INVALID, "share", dict(y=flat(at=FAR[2]))),
    (N.S14_ERR_INVALID, "norm weight", dict(y=flat(at=FAR[4]))),
    (N.S14_ERR_INVALID, "codes or scales", dict(q=N.Buffer(FAR[0], HUGE))),
    (N.S14_ERR_INVALID, "codes or scales", dict(s=N.Buffer(FAR[5] + 16, HUGE))),
    (N.S14_ERR_INVALID, "codes or scales", dict(s=N.Buffer(FAR[4] + 100, HUGE))),
    (N.S14_ERR_INVALID, "codes or scales", dict(q=N.Buffer(FAR[2] + ROW - 8, HUGE))),
])
def test_norm_refusals(native, code, text, kw):
    refused(code, norm(native, **kw), text)


def test_norm_without_rows_is_no_launch(native):
    assert norm(native, n=0) == N.S14_OK
    assert norm(native, n=0, q=NONE, s=NONE) == N.S14_OK


def test_python_layer_refuses_other_shapes():
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)  # noqa: E731
    good = [u8(3, 2, 16, 64), u8(3, 2, 4, 16), u8(3, 2, 4, 1, 16, 16), u8(3, 2, 1, 16)]
    c = A.KvCache4(*good)
    assert (c.pages, c.heads, c.page_tokens, c.dim) == (3, 2, 16, 128)
    wide = A.KvCache4.empty(3, 1, 32, 512, device="cpu")
    assert wide.v_scales.shape == (3, 1, 4, 32) and wide.k_scales.shape == (3, 1, 16, 32)
    for i, bad in ((0, good[0][0]), (0, good[0].float()), (1, u8(3, 2, 16, 4)), (2, u8(3, 2, 128, 8)), (3, u8(3, 2)),
                   (3, u8(3, 2, 2, 16)), (2, u8(3, 2, 4, 1, 16, 32)[..., ::2])):
        with pytest.raises(N.S14Error):
            A.KvCache4(*good[:i], bad, *good[i + 1:])
    x, i = torch.zeros(2, 2, 128), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(N.S14Error, match="context's device"):
        A.kv_append(FakeContext(), c, x, x, i, i, i)
    with pytest.raises(N.S14Error, match="context's device"):
        A.paged_attention(FakeContext(), x, c, i, i, i, x)


@pytest.mark.parametrize("which", range(4))
def test_other_memory_behind_a_cache_is_refused(which):
    c = A.KvCache4.empty(3, 2, 16, 64, device="cpu")
    c._tensors[which].set_(torch.zeros_like(c._tensors[which]))
    x, i = torch.zeros(2, 2, 64), torch.zeros(2, dtype=torch.int32)
    ctx, pages = CpuContext(), torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(N.S14Error, match="the cache was made of other memory"):
        A.kv_append(ctx, c, x, x, pages, i, i)
    with pytest.raises(N.S14Error, match="the cache was made of other memory"):
        A.paged_attention(ctx, x.bfloat16(), c, pages, i, i, x)


@pytest.mark.parametrize("text,kw", [
    ("x is required", dict(x=None)),
    ("x must be", dict(x=torch.zeros(2, 2, 256))),
    ("float32 or bfloat16", dict(x=torch.zeros(2, 256, dtype=torch.float16))),
    ("last dimension contiguous", dict(x=torch.zeros(256, 2).T)),
    ("residual must have", dict(residual=torch.zeros(3, 256))),
    ("y must have", dict(y=torch.zeros(2, 128))),
    ("norm weight", dict(weight=torch.zeros(128))),
    ("norm weight", dict(weight=torch.zeros(256, dtype=torch.bfloat16))),
    ("go together", dict(q=torch.zeros(2, 256, dtype=torch.uint8))),
    ("codes must be", dict(q=torch.zeros(2, 256), scales=torch.zeros(2, 2, dtype=torch.uint8))),
    ("codes must be", dict(q=torch.zeros(2, 255, dtype=torch.uint8), scales=torch.zeros(2, 2, dtype=torch.uint8))),
    ("scales must be", dict(q=torch.zeros(2, 256, dtype=torch.uint8), scales=torch.zeros(3, 2, dtype=torch.uint8))),
    ("scales of a row", dict(q=torch.zeros(2, 256, dtype=torch.uint8), scales=torch.zeros(2, 3, dtype=torch.uint8))),
    ("scales of a row", dict(q=torch.zeros(2, 256, dtype=torch.uint8), scales=torch.zeros(2, 1, dtype=torch.uint8))),
    ("scales of a row", dict(q=torch.zeros(2, 256, dtype=torch.uint8), scales=torch.zeros(2, 0, dtype=torch.uint8))),
])
def test_python_norm_refusals(text, kw):
    args = dict(x=torch.zeros(2, 256), weight=torch.ones(256), y=torch.zeros(2, 256)) | kw
    with pytest.raises(N.S14Error, match=text):
        A.add_rms_norm(CpuContext(), stream=0, **args)
    with pytest.raises(N.S14Error, match="context's device|required"):
        A.add_rms_norm(FakeContext(), stream=0, **args)


@pytest.mark.parametrize("row", range(4))
@pytest.mark.parametrize("which", ["ro", "y"])
def test_norm_refuses_a_weight_in_any_row_of_an_output(native, which, row):
    out = flat(at=FAR[7], stride=1024)
    last = row * 4096 + 2048 - 16
    refused(N.S14_ERR_INVALID, norm(native, **{which: out}, w=N.Buffer(FAR[7] + last, HUGE)), "norm weight")
    refused(N.S14_ERR_INVALID, norm(native, **{which: out}, q=N.Buffer(FAR[7] + last, HUGE)), "codes or scales")


@pytest.mark.parametrize("row", range(3))
def test_norm_takes_a_weight_between_an_outputs_rows(native, row):
    out = flat(at=FAR[7], stride=1024)
    weight = N.Buffer(FAR[7] + row * 4096 + 2048, HUGE)
    refused(N.S14_ERR_INVALID, norm(native, y=out, ro=out, w=weight), "the residual output and y share")

"""Attention between the FP8 projections and the expert layer — Python face of
the C ABI's attention entry points (include/s14_hip.h).

A decode or verify step of a layer, around ``s14.fp8_linear`` and
``s14.moe_block_route``::

    qk_norm_rope(ctx, q, None, q16, None, q_weight=wq, rope=rope, positions=pos)
    kv_append(ctx, cache, k, v, table, cu, past, k_weight=wk, rope=rope, max_new=n)
    paged_attention(ctx, q16, cache, table, cu, lens, out, max_new=n, max_len=longest)

and a whole prompt: ``qk_norm_rope`` of q and k, ``prompt_attention``, and
``kv_append`` of the rotated keys for the steps that follow.

Operands are torch tensors on the context's device, packed [tokens, heads,
dim] with any strides that are multiples of 8 elements and a contiguous last
dimension; index tensors are contiguous int32.  The work goes to that device's
current torch stream unless ``stream`` is given.  The reference's GPU code has
no counterpart.
"""

from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from typing import Optional

import torch

from . import _native as N
from ._native import S14Error, check, lib
from .s14 import Context

PAGE_TOKENS = (16, 32, 64, 128)
_DTYPES = {torch.float32: (N.S14_X_F32, 4), torch.bfloat16: (N.S14_X_BF16, 2)}
_LAYOUTS = {"half": N.S14_ROPE_HALF, "interleaved": N.S14_ROPE_INTERLEAVED}
_NO_BUFFER, _NO_ROWS = N.Buffer(None, 0), N.Rows()


def _raw_stream():
    """torch's current stream of a device, without the object where this torch
    has the raw call."""
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return raw if raw is not None else lambda device: torch.cuda.current_stream(device).cuda_stream


_RAW_STREAM = _raw_stream()


def _refuse(code: int, message: str):
    raise S14Error(code, message)


def _here(ctx: Context, t, label: str):
    if not isinstance(t, torch.Tensor) or t.get_device() != ctx.device:
        _refuse(N.S14_ERR_INVALID, f"{label} must be a tensor on the context's device {ctx.device}")


def _rows(ctx: Context, t, label: str, dim: Optional[int] = None):
    """The s14_rows of a [tokens, heads, dim] tensor.  (On the path of a
    single token's calls: each tensor is asked for each property once.)"""
    try:
        code, size = _DTYPES[t.dtype]
        tokens, heads, width = t.shape
        token_stride, head_stride, one = t.stride()
        if t.get_device() != ctx.device or (one != 1 and width > 1) or (dim is not None and width != dim):
            raise ValueError
    except (AttributeError, KeyError, ValueError):
        _here(ctx, t, label)
        if t.dtype not in _DTYPES:
            _refuse(N.S14_ERR_INVALID, f"{label} must be float32 or bfloat16, not {t.dtype}")
        _refuse(N.S14_ERR_SHAPE, f"{label} must be [tokens, heads, {dim or 'dim'}] with a contiguous last dimension")
    # strides of a dimension of one are not used; what torch gives there may be anything
    if tokens < 2:
        token_stride = 0
    if heads < 2:
        head_stride = 0
    reach = ((tokens - 1) * token_stride + (heads - 1) * head_stride + width) * size if tokens and heads else 0
    return N.Rows(t.data_ptr(), reach, code, heads, token_stride, head_stride)


def _flat(ctx: Context, t, dtype, label: str, size: int = 0):
    """The buffer of a contiguous tensor of one dtype, of `size` values at least."""
    if t is None:
        return _NO_BUFFER
    if not isinstance(t, torch.Tensor) or t.get_device() != ctx.device:
        _here(ctx, t, label)
    if t.dtype is not dtype or not t.is_contiguous():
        _refuse(N.S14_ERR_INVALID, f"{label} must be a contiguous {dtype} tensor")
    if size and t.numel() < size:
        _refuse(N.S14_ERR_CAPACITY, f"{label} has {t.numel()} values, {size} are required")
    return N.Buffer(t.data_ptr(), t.nbytes)


class Rope:
    """A rotation: its table (f32 [positions, rot], ``rope_table``), the pairs'
    layout ("half": i with i + rot / 2; "interleaved": 2 i with 2 i + 1) and the
    first rotated dimension of a head."""

    def __init__(self, table, layout: str = "half", start: int = 0):
        if layout not in _LAYOUTS:
            _refuse(N.S14_ERR_INVALID, f"unknown rotation layout {layout!r}")
        if table.dim() != 2 or table.dtype != torch.float32 or not table.is_contiguous():
            _refuse(N.S14_ERR_SHAPE, "a rotation table is contiguous float32 [positions, rot]")
        if start < 0:
            _refuse(N.S14_ERR_SHAPE, f"rotation start {start}")
        self.table, self.layout, self.start = table, layout, start
        self._c = N.Rope(N.Buffer(table.data_ptr(), table.nbytes), table.shape[0], table.shape[1], start,
                         _LAYOUTS[layout])


def _rope(ctx: Context, rope: Optional[Rope]):
    if rope is None:
        return None
    if rope.table.get_device() != ctx.device:
        _here(ctx, rope.table, "rotation table")
    return C.byref(rope._c)


@dataclass(frozen=True)
class RopeScaling:
    """Stretching of a rotation for long contexts (s14_rope_scaling)."""

    factor: float
    original: float = 0.0
    beta_fast: float = 32.0
    beta_slow: float = 1.0
    amplitude: float = 1.0


class KvCache:
    """The paged 8-bit cache: uint8 E4M3 codes k [pages, heads, page_tokens,
    dim] and v [pages, heads, dim, page_tokens], uint8 E8M0 scales [pages,
    heads] of each."""

    def __init__(self, k_pages, k_scales, v_pages, v_scales):
        for t, label in ((k_pages, "k codes"), (k_scales, "k scales"), (v_pages, "v codes"), (v_scales, "v scales")):
            if t.dtype != torch.uint8 or not t.is_contiguous():
                _refuse(N.S14_ERR_INVALID, f"{label} must be contiguous uint8")
            if t.device != k_pages.device:
                _refuse(N.S14_ERR_INVALID, "the cache's tensors are on different devices")
        if k_pages.dim() != 4:
            _refuse(N.S14_ERR_SHAPE, "k codes must be [pages, heads, page_tokens, dim]")
        pages, heads, page, dim = k_pages.shape
        if tuple(v_pages.shape) != (pages, heads, dim, page):
            _refuse(N.S14_ERR_SHAPE, f"v codes must be [{pages}, {heads}, {dim}, {page}]")
        if tuple(k_scales.shape) != (pages, heads) or tuple(v_scales.shape) != (pages, heads):
            _refuse(N.S14_ERR_SHAPE, f"scales must be [{pages}, {heads}]")
        self.k_pages, self.k_scales, self.v_pages, self.v_scales = k_pages, k_scales, v_pages, v_scales
        self.pages, self.heads, self.page_tokens, self.dim = pages, heads, page, dim
        buf = [N.Buffer(t.data_ptr(), t.nbytes) for t in (k_pages, v_pages, k_scales, v_scales)]
        self._c = N.KvCache(*buf, pages, heads, page, dim)

    @classmethod
    def empty(cls, pages: int, heads: int, page_tokens: int, dim: int, device="cuda") -> "KvCache":
        """An uninitialised cache: every slot is written before it is read."""
        new = lambda *shape: torch.empty(shape, dtype=torch.uint8, device=device)  # noqa: E731
        return cls(new(pages, heads, page_tokens, dim), new(pages, heads), new(pages, heads, dim, page_tokens),
                   new(pages, heads))


def _cache(ctx: Context, cache: KvCache):
    if cache.k_pages.get_device() != ctx.device:
        _here(ctx, cache.k_pages, "cache")
    return C.byref(cache._c)


def rope_table(ctx: Context, table, theta: float = 10000.0, scaling: Optional[RopeScaling] = None, stream=None) -> None:
    """Fill table (f32 [positions, rot]) with cos | sin of each position's
    rot / 2 angles, computed in 64 bits."""
    buf = _flat(ctx, table, torch.float32, "rotation table")
    if table.dim() != 2:
        _refuse(N.S14_ERR_SHAPE, "a rotation table is [positions, rot]")
    s = None
    if scaling is not None:
        s = C.byref(N.RopeScaling(scaling.factor, scaling.original, scaling.beta_fast, scaling.beta_slow,
                                  scaling.amplitude))
    check(lib().s14_rope_table(ctx._h, _RAW_STREAM(ctx.device) if stream is None else stream, table.shape[0], table.shape[1], theta, s, buf))


def qk_norm_rope(ctx: Context, q, k, q_out, k_out, q_weight=None, k_weight=None, eps: float = 1e-6,
                 rope: Optional[Rope] = None, positions=None, stream=None) -> None:
    """Per-head RMS norm (where a weight is given) and rotation (where `rope`
    is) of q [tokens, heads, dim] and k (or None) in one launch, in f32; f32 or
    bf16 in and out, outputs may be their inputs."""
    rq, ro = _rows(ctx, q, "q"), _rows(ctx, q_out, "q output")
    tokens, _, dim = q.shape
    if q_out.shape != q.shape:
        _refuse(N.S14_ERR_SHAPE, "q output must have q's shape")
    if k is None:
        rk = ko = _NO_ROWS
    else:
        rk, ko = _rows(ctx, k, "k", dim), _rows(ctx, k_out, "k output", dim)
        if k.shape[0] != tokens or k_out.shape != k.shape:
            _refuse(N.S14_ERR_SHAPE, "k must have q's tokens, and k output k's shape")
    check(lib().s14_qk_norm_rope(
        ctx._h, _RAW_STREAM(ctx.device) if stream is None else stream, tokens, dim, C.byref(rq), C.byref(rk), C.byref(ro), C.byref(ko),
        _flat(ctx, q_weight, torch.float32, "q norm weight"), _flat(ctx, k_weight, torch.float32, "k norm weight"),
        eps, _rope(ctx, rope), _flat(ctx, positions, torch.int32, "positions")))


def _table(ctx: Context, page_table, cu, lens, label: str):
    """Buffers of the index tensors, sequences and table width."""
    table = _flat(ctx, page_table, torch.int32, "page table")
    if page_table.dim() != 2:
        _refuse(N.S14_ERR_SHAPE, "a page table is [sequences, pages]")
    seqs, width = page_table.shape
    return table, width, _flat(ctx, cu, torch.int32, "cu", seqs + 1), _flat(ctx, lens, torch.int32, label, seqs), seqs


def kv_append(ctx: Context, cache: KvCache, k, v, page_table, cu, past, k_weight=None, eps: float = 1e-6,
              rope: Optional[Rope] = None, max_new: Optional[int] = None, stream=None) -> None:
    """Rows cu[i] .. cu[i + 1] - 1 of k and v [tokens, heads, dim] (f32 or
    bf16) become positions past[i] .. of sequence i in the cache, K with the
    norm and rotation of ``qk_norm_rope`` on the way.  max_new: at least the
    most new tokens of a sequence (all of them if left out)."""
    rk, rv = _rows(ctx, k, "k", cache.dim), _rows(ctx, v, "v", cache.dim)
    if k.shape[0] != v.shape[0]:
        _refuse(N.S14_ERR_SHAPE, "k and v have different token counts")
    table, width, cub, lenb, seqs = _table(ctx, page_table, cu, past, "past")
    tokens = k.shape[0]
    check(lib().s14_kv_append(
        ctx._h, _RAW_STREAM(ctx.device) if stream is None else stream, _cache(ctx, cache), tokens, seqs, tokens if max_new is None else max_new,
        C.byref(rk), C.byref(rv), table, width, cub, lenb, _flat(ctx, k_weight, torch.float32, "k norm weight"), eps,
        _rope(ctx, rope)))


def paged_attention(ctx: Context, q, cache: KvCache, page_table, cu, lens, out, lse=None, scale: Optional[float] = None,
                    window: int = 0, max_new: Optional[int] = None, max_len: Optional[int] = None, stream=None) -> None:
    """Attention of q's rows (bf16 [tokens, heads, dim]; cu[i] .. cu[i + 1] - 1
    are the last tokens of sequence i) over the sequences' lens[i] cached
    tokens, causal, with `window` > 0 over the last `window` positions only.
    out: q's shape, bf16 or f32; lse: f32 [tokens, heads] or None.  max_new: at
    least the most rows of a sequence; max_len: about the longest sequence (it
    sets how the work is split; the page table's reach if left out)."""
    rq, ro = _rows(ctx, q, "q", cache.dim), _rows(ctx, out, "out", cache.dim)
    tokens, heads, dim = q.shape
    if out.shape != q.shape:
        _refuse(N.S14_ERR_SHAPE, "out must have q's shape")
    table, width, cub, lenb, seqs = _table(ctx, page_table, cu, lens, "lens")
    check(lib().s14_paged_attention(
        ctx._h, _RAW_STREAM(ctx.device) if stream is None else stream, C.byref(rq), _cache(ctx, cache), tokens, seqs,
        tokens if max_new is None else max_new, width * cache.page_tokens if max_len is None else max_len, table, width,
        cub, lenb, C.byref(ro), _flat(ctx, lse, torch.float32, "lse", tokens * heads),
        dim ** -0.5 if scale is None else scale, window))


def prompt_attention(ctx: Context, q, k, v, cu, out, lse=None, scale: Optional[float] = None, window: int = 0,
                     stream=None) -> None:
    """Causal attention over packed prompts, sequence i the rows cu[i] .. cu[i
    + 1] - 1 of q [tokens, heads, dim] and k, v [tokens, key heads, dim] (all
    bf16).  out, lse and window as in ``paged_attention``."""
    rq, ro = _rows(ctx, q, "q"), _rows(ctx, out, "out")
    tokens, heads, dim = q.shape
    rk, rv = _rows(ctx, k, "k", dim), _rows(ctx, v, "v", dim)
    if out.shape != q.shape or k.shape != v.shape or k.shape[0] != tokens:
        _refuse(N.S14_ERR_SHAPE, "out must have q's shape, v k's, and k q's tokens")
    cub = _flat(ctx, cu, torch.int32, "cu", 1)
    check(lib().s14_prompt_attention(
        ctx._h, _RAW_STREAM(ctx.device) if stream is None else stream, dim, C.byref(rq), C.byref(rk), C.byref(rv), tokens, cu.numel() - 1, cub,
        C.byref(ro), _flat(ctx, lse, torch.float32, "lse", tokens * heads), dim ** -0.5 if scale is None else scale,
        window))


__all__ = [
    "KvCache",
    "Rope",
    "RopeScaling",
    "kv_append",
    "paged_attention",
    "prompt_attention",
    "qk_norm_rope",
    "rope_table",
]

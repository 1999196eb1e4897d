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
import importlib.util
from dataclasses import dataclass
from typing import Optional

import torch

from . import _native as N
from ._native import S14Error, check, lib
from .s14 import Context

PAGE_TOKENS = (16, 32, 64, 128)
_LAYOUTS = {"half": N.S14_ROPE_HALF, "interleaved": N.S14_ROPE_INTERLEAVED}


def _raw_stream():
    """torch's current stream of a device, without the object where this torch
    has the raw call."""
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return raw if raw is not None else lambda device: torch.cuda.current_stream(device).cuda_stream


def _refuse(code: int, message: str):
    raise S14Error(code, message)


def _load():
    """The calls' C side (csrc/s14_attn_py.cpp) with the library's entry points."""
    path = N.LIB_DIR / "_s14attn.so"
    if not path.exists():
        raise ImportError(f"{path} is not built; run `python -m colormlm_amd.build` (there is no fallback path)")
    spec = importlib.util.spec_from_file_location("_s14attn", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    names = ("s14_qk_norm_rope", "s14_kv_append", "s14_paged_attention", "s14_prompt_attention")
    module.bind(tuple(C.cast(getattr(lib(), n), C.c_void_p).value for n in names), _refuse, check, _raw_stream())
    return module


_call = _load()


def _here(device: int, t, label: str):
    if not isinstance(t, torch.Tensor) or t.get_device() != device:
        _refuse(N.S14_ERR_INVALID, f"{label} must be a tensor on the context's device {device}")


class Rope:
    """A rotation: its table (f32 [positions, rot], ``rope_table``), the pairs'
    layout ("half": i with i + rot / 2; "interleaved": 2 i with 2 i + 1) and the
    first rotated dimension of a head."""

    def __init__(self, table, layout: str = "half", start: int = 0):
        if layout not in _LAYOUTS:
            _refuse(N.S14_ERR_INVALID, f"unknown rotation layout {layout!r}")
        if table.dim() != 2 or table.dtype != torch.float32 or not table.is_contiguous():
            _refuse(N.S14_ERR_SHAPE, "a rotation table is contiguous float32 [positions, rot]")
        if not 0 <= start < 1 << 32:
            _refuse(N.S14_ERR_SHAPE, f"rotation start {start}")
        self._tensors, self.layout, self.start = (table,), layout, start
        self._c = N.Rope(N.Buffer(table.data_ptr(), table.nbytes), table.shape[0], table.shape[1], start,
                         _LAYOUTS[layout])
        self._at, self._device = C.addressof(self._c), table.get_device()

    # its address is held: not to be replaced, and a call refuses other memory behind it
    table = property(lambda self: self._tensors[0])


def _rope(ctx: Context, rope: Optional[Rope]):
    """The address of a rotation's s14_rope on the context's device."""
    if rope is None:
        return None
    if rope._device != ctx.device:
        _here(ctx.device, rope.table, "rotation table")
    return rope._at


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
        self._tensors = (k_pages, k_scales, v_pages, v_scales)
        self.pages, self.heads, self.page_tokens, self.dim = pages, heads, page, dim
        buf = [N.Buffer(t.data_ptr(), t.nbytes) for t in (k_pages, v_pages, k_scales, v_scales)]
        self._c = N.KvCache(*buf, pages, heads, page, dim)
        self._at, self._device = C.addressof(self._c), k_pages.get_device()

    # their addresses are held: not to be replaced, and a call refuses other memory behind them
    k_pages = property(lambda self: self._tensors[0])
    k_scales = property(lambda self: self._tensors[1])
    v_pages = property(lambda self: self._tensors[2])
    v_scales = property(lambda self: self._tensors[3])

    @classmethod
    def empty(cls, pages: int, heads: int, page_tokens: int, dim: int, device="cuda") -> "KvCache":
        """An uninitialised cache: every slot is written before it is read."""
        new = lambda *shape: torch.empty(shape, dtype=torch.uint8, device=device)  # noqa: E731
        return cls(new(pages, heads, page_tokens, dim), new(pages, heads), new(pages, heads, dim, page_tokens),
                   new(pages, heads))


def _cache(ctx: Context, cache: KvCache):
    if cache._device != ctx.device:
        _here(ctx.device, cache.k_pages, "cache")
    return cache._at


def rope_table(ctx: Context, table, theta: float = 10000.0, scaling: Optional[RopeScaling] = None, stream=None) -> None:
    """Fill table (f32 [positions, rot]) with cos | sin of each position's
    rot / 2 angles, computed in 64 bits."""
    _here(ctx.device, table, "rotation table")
    if table.dim() != 2 or table.dtype != torch.float32 or not table.is_contiguous():
        _refuse(N.S14_ERR_SHAPE, "a rotation table is contiguous float32 [positions, rot]")
    s = None
    if scaling is not None:
        s = C.byref(N.RopeScaling(scaling.factor, scaling.original, scaling.beta_fast, scaling.beta_slow,
                                  scaling.amplitude))
    stream = _raw_stream()(ctx.device) if stream is None else stream
    check(lib().s14_rope_table(ctx.handle, stream, table.shape[0], table.shape[1], theta, s,
                               N.Buffer(table.data_ptr(), table.nbytes)))


def qk_norm_rope(ctx: Context, q, k, q_out, k_out, q_weight=None, k_weight=None, eps: float = 1e-6,
                 rope: Optional[Rope] = None, positions=None, stream=None) -> None:
    """Per-head RMS norm (where a weight is given) and rotation (where `rope`
    is) of q [tokens, heads, dim] and k (or None) in one launch, in f32; f32 or
    bf16 in and out.  An output may be its own input; outputs that share memory
    with other rows are refused, here and below."""
    _call.qk_norm_rope(ctx._h.value, ctx.device, stream, q, k, q_out, k_out, q_weight, k_weight, eps, _rope(ctx, rope),
                       positions, None if rope is None else rope._tensors)


def kv_append(ctx: Context, cache: KvCache, k, v, page_table, cu, past, k_weight=None, eps: float = 1e-6,
              rope: Optional[Rope] = None, max_new: Optional[int] = None, stream=None) -> None:
    """Rows cu[i] .. cu[i + 1] - 1 of k and v [tokens, heads, dim] (f32 or
    bf16) become positions past[i] .. of sequence i in the cache, K with the
    norm and rotation of ``qk_norm_rope`` on the way.  max_new: at least the
    most new tokens of a sequence, and at most the call's (which it is if left
    out); rows past it are not stored."""
    _call.kv_append(ctx._h.value, ctx.device, stream, _cache(ctx, cache), cache.dim, k, v, page_table, cu, past, k_weight,
                    eps, _rope(ctx, rope), max_new, cache._tensors, None if rope is None else rope._tensors)


def paged_attention(ctx: Context, q, cache: KvCache, page_table, cu, lens, out, lse=None, scale: Optional[float] = None,
                    window: int = 0, max_new: Optional[int] = None, max_len: Optional[int] = None, stream=None) -> None:
    """Attention of q's rows (bf16 [tokens, heads, dim]; cu[i] .. cu[i + 1] - 1
    are the last tokens of sequence i) over the sequences' lens[i] cached
    tokens, causal, with `window` > 0 over the last `window` positions only.
    out: q's shape, bf16 or f32, q itself at will; lse: f32 [tokens, heads] or
    None.  max_new: at least the most rows of a sequence, and at most the call's
    tokens, which it is if left out (the work is split for one sequence that has
    them all: give it for a batch); max_len: about the longest sequence (it
    sets how the work is split; the page table's reach if left out)."""
    _call.paged_attention(ctx._h.value, ctx.device, stream, q, _cache(ctx, cache), cache.dim, page_table, cu, lens, out,
                          lse, scale, window, max_new, max_len, cache.page_tokens, cache._tensors)


def prompt_attention(ctx: Context, q, k, v, cu, out, lse=None, scale: Optional[float] = None, window: int = 0,
                     stream=None) -> None:
    """Causal attention over packed prompts, sequence i the rows cu[i] .. cu[i
    + 1] - 1 of q [tokens, heads, dim] and k, v [tokens, key heads, dim] (all
    bf16).  out, lse and window as in ``paged_attention``."""
    _call.prompt_attention(ctx._h.value, ctx.device, stream, q, k, v, cu, out, lse, scale, window)


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

"""The paged 4-bit cache (append and attention) against plain 64-bit
implementations.

Tolerances, from the operators' own roundings:

  append     without a norm or rotation none: codes and scales are those of the
             definition, bit for bit (scales and quotients by powers of two are
             exact).  With them a value is off by (D + 16) 2^-24 of the pair's
             magnitudes before it is rounded: within half an E2M1 step (1/4, 1/2 or
             1 of the scale) and that, by the scale that the cache holds, which is
             the definition's of a value within the same error
  attention  a weight, multiplied by its token's power of two, is rounded to bf16
             once, 2^-8 of it, as with the 8-bit cache: that module's tolerance
"""

from __future__ import annotations

import itertools
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import test_gpu_attention as T  # noqa: E402
from test_gpu_attention import BF16, F32, I32, U8, check_attention, cumulative, gen, ints, norm_rope64, rand, say, table64  # noqa: E402

from colormlm_amd import attention as A  # noqa: E402
from colormlm_amd import s14  # noqa: E402

pytestmark = pytest.mark.gpu

E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


@pytest.fixture(scope="module")
def ctx():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    c = s14.Context(0)
    yield c
    torch.cuda.synchronize()
    c.destroy()


# ---------------------------------------------------------------------------
# the format, by its places: code and scale of (page, head, slot, dimension)
# ---------------------------------------------------------------------------


def block_of(dim, side):
    return 32 if side == 0 else min(dim, 128)


def k_codes(k):
    """uint8 [pages, heads, slots, dim] of a cache's bytes."""
    return torch.stack([k & 15, k >> 4], -1).flatten(-2)


def v_codes(v):
    x = torch.stack([v & 15, v >> 4], -1)  # [pages, heads, dim / 32, slots / 16, 16, 16, 2]
    pages, heads, u, b = x.shape[:4]
    x = x.view(pages, heads, u, b, 16, 2, 8, 2)  # unit, block, d, half, j, parity
    return x.permute(0, 1, 3, 6, 7, 2, 5, 4).reshape(pages, heads, 16 * b, 32 * u)


def k_scales(s):
    """uint8 [pages, heads, slots, dim / 32]."""
    slot = torch.arange(s.shape[-1])
    return s[..., slot - slot % 16 + 4 * (slot % 4) + slot % 16 // 4].transpose(-1, -2)


def v_scales(s):
    return s.transpose(-1, -2)


def value64(codes, scales):
    """[..., dim] values of codes [..., dim] and scales [..., blocks]."""
    v = E2M1[(codes & 7).long()] * (1.0 - 2.0 * (codes >> 3).double())
    p = (scales.double() - 127.0).exp2()
    p[scales == 255] = math.nan
    return (v.unflatten(-1, (scales.shape[-1], -1)) * p[..., None]).flatten(-2)


def scale64(amax):
    """E8M0 codes of blocks' largest magnitudes (f64, finite)."""
    e = torch.where(amax > 0, (amax.clamp(min=2.0 ** -140) / 6.0).log2().ceil(), -100.0)
    e = torch.where(6.0 * (e - 1).exp2() >= amax, e - 1, e)  # the logarithm's rounding
    return (e.clamp(-100, 100) + 127).to(U8)


def codes64(x, scales, block):
    """Codes of x [..., dim] (f64, finite), to nearest, ties to even."""
    a = x.unflatten(-1, (-1, block)) / (scales.double() - 127.0).exp2()[..., None]
    step = torch.where(a.abs() < 2.0, 0.5, torch.where(a.abs() < 4.0, 1.0, 2.0))
    near = ((a / step).round() * step).abs().clamp(max=6.0)
    code = torch.searchsorted(E2M1, near.contiguous())
    return (code + 8 * (a < 0)).to(U8).flatten(-2)


class Paged4:
    """A random cache whose pages lie in random order, with spare pages, and the
    sequences' K and V as 64-bit rows."""

    def __init__(self, seed, lengths, kv, dim, page, width=None, lo=122, hi=129):
        g = gen(seed)
        need = [-(-n // page) for n in lengths]
        pages = sum(need) + 3
        self.cache = A.KvCache4.empty(pages, kv, page, dim)
        c = self.cache
        byte = lambda t: torch.randint(0, 256, t.shape, generator=g, dtype=U8)  # noqa: E731
        scale = lambda t: torch.randint(lo, hi, t.shape, generator=g, dtype=U8)  # noqa: E731
        self.k, self.v, self.ks, self.vs = byte(c.k_pages), byte(c.v_pages), scale(c.k_scales), scale(c.v_scales)
        order = torch.randperm(pages, generator=g)
        self.table = torch.full((len(lengths), max([1, *need]) if width is None else width), 0x7FFFFFFF, dtype=I32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n].int()
            at += n
        self.lengths, self.page, self.need = lengths, page, need
        self.upload()

    def upload(self):
        c = self.cache
        for dst, src in ((c.k_pages, self.k), (c.v_pages, self.v), (c.k_scales, self.ks), (c.v_scales, self.vs)):
            dst.copy_(src)
        self.dev_table = self.table.cuda()
        self.lens = ints(self.lengths)

    def download(self):
        c = self.cache
        self.k, self.v, self.ks, self.vs = (x.cpu() for x in (c.k_pages, c.v_pages, c.k_scales, c.v_scales))

    def rows(self, i, length=None):
        length = self.lengths[i] if length is None else length
        ids = self.table[i, :-(-length // self.page)].long()
        k = value64(k_codes(self.k[ids]), k_scales(self.ks[ids])).permute(0, 2, 1, 3).flatten(0, 1)
        v = value64(v_codes(self.v[ids]), v_scales(self.vs[ids])).permute(0, 2, 1, 3).flatten(0, 1)
        return k[:length], v[:length]

    def place(self, i, j):
        """Page and slot of position j of sequence i."""
        return int(self.table[i, j // self.page]), j % self.page

    def set_scale(self, side, i, j, code, block=None):
        """The scales of a token (one block of it, or all) in the host's copy."""
        page, slot = self.place(i, j)
        s = self.vs if side else self.ks
        at = slot if side else slot - slot % 16 + 4 * (slot % 4) + slot % 16 // 4
        if block is None:
            s[page, :, :, at] = code
        else:
            s[page, :, block, at] = code


run_paged, paged_want = T.run_paged, T.paged_want  # by the cache that they are given


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------

APPEND = [  # lengths before, new counts, kv heads, dim, page
    ([0], [1], 1, 64, 16), ([0, 5, 64, 63], [1, 1, 1, 1], 8, 128, 64), ([299], [8], 1, 512, 64),
    ([7, 0, 31, 16], [40, 0, 1, 17], 2, 128, 16), ([100, 3], [300, 129], 1, 256, 128), ([130], [200], 3, 64, 32),
    ([10, 120], [128, 9], 1, 512, 128), ([15, 14, 2], [3, 4, 2], 2, 64, 32), ([13, 1], [2, 4], 1, 512, 16),
    ([3] * 70, [1] * 70, 2, 256, 16), ([5] * 40, [20, 1] * 20, 2, 64, 64)]


def changed(p, past, new):
    """Places (page, slot) of the new tokens, in packed order."""
    return [p.place(i, a + j) for i, (a, b) in enumerate(zip(past, new)) for j in range(b)]


@pytest.mark.parametrize("past,new,kv,dim,page", APPEND)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_append_is_the_definition(ctx, past, new, kv, dim, page, dtype):
    say(f"append4 past={past} new={new} kv={kv} dim={dim} page={page} {dtype}")
    g = gen(sum(past) + 7 * sum(new) + dim)
    p = Paged4(dim + page, [a + b for a, b in zip(past, new)], kv, dim, page)
    tokens = sum(new)
    k, v = (rand(g, tokens, kv, dim, dtype=dtype) * torch.exp(4 * rand(g, tokens, 1, 1)).to(dtype) for _ in range(2))
    # ties, values at the border of a scale, zeros
    k[0, 0, :16] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 2).to(dtype)
    k[0, 0, 16:32], v[-1, -1] = 0.0, 0.0
    A.kv_append(ctx, p.cache, k.cuda(), v.cuda(), p.dev_table, cumulative(new), ints(past), max_new=max(new))
    torch.cuda.synchronize()
    ctx.launch_status()
    was = [k_codes(p.k), v_codes(p.v), k_scales(p.ks).contiguous(), v_scales(p.vs).contiguous()]
    p.download()
    got = [k_codes(p.k), v_codes(p.v), k_scales(p.ks), v_scales(p.vs)]
    for side, x in enumerate((k.double(), v.double())):
        block = block_of(dim, side)
        s = scale64(x.unflatten(-1, (-1, block)).abs().amax(-1))
        c = codes64(x, s, block)
        for at, (pg, slot) in enumerate(changed(p, past, new)):
            was[side][pg, :, slot], was[2 + side][pg, :, slot] = c[at], s[at]
    for side in range(2):
        assert torch.equal(got[2 + side], was[2 + side]), ("scales", side)
        # a zero has either sign
        assert torch.equal(torch.where(got[side] == 8, 0, got[side]), torch.where(was[side] == 8, 0, was[side])), ("codes", side)


@pytest.mark.parametrize("past,new,kv,dim,page", APPEND[:9])
@pytest.mark.parametrize("dtype,norm,rot,start,layout", [(F32, True, 64, 0, "half"), (BF16, True, 0, 0, "half"),
                                                         (F32, False, 32, 24, "interleaved"), (F32, True, 40, 8, "half"),
                                                         (BF16, False, 0, 0, "full")])
def test_append_norm_and_rotation(ctx, past, new, kv, dim, page, dtype, norm, rot, start, layout):
    if layout == "full":
        rot, layout = dim, "half"
    say(f"append4 past={past} new={new} kv={kv} dim={dim} page={page} {dtype} norm={norm} rot={rot}@{start} {layout}")
    g = gen(sum(past) + 7 * sum(new) + dim)
    p = Paged4(dim + page, [a + b for a, b in zip(past, new)], kv, dim, page)
    tokens = sum(new)
    k, v = (rand(g, tokens, kv, dim, dtype=dtype) * torch.exp(rand(g, tokens, 1, 1)).to(dtype) for _ in range(2))
    w = rand(g, dim).abs() + 0.5 if norm else None
    table = table64(1024, rot).float() if rot else None
    rope = A.Rope(table.cuda(), layout, start) if rot else None
    before = [k_codes(p.k), v_codes(p.v)]
    A.kv_append(ctx, p.cache, k.cuda(), v.cuda(), p.dev_table, cumulative(new), ints(past), k_weight=w.cuda() if norm else None,
                rope=rope, max_new=max(new))
    torch.cuda.synchronize()
    ctx.launch_status()
    p.download()
    pos = torch.cat([torch.arange(a, a + b) for a, b in zip(past, new)])
    y, mag = norm_rope64(k, w, 1e-6, table, pos, layout, start)
    err = (dim + 16) * 2.0 ** -24 * mag
    places = changed(p, past, new)
    pg, slot = (torch.tensor(x) for x in zip(*places))
    codes, scales = k_codes(p.k)[pg, :, slot], k_scales(p.ks)[pg, :, slot]
    part, slack = y.unflatten(-1, (-1, 32)).abs().amax(-1), err.unflatten(-1, (-1, 32)).amax(-1)
    lo, hi = scale64((part - slack).clamp(min=0)), scale64(part + slack)
    assert bool(((scales >= lo) & (scales <= hi)).all())
    power = (scales.double() - 127).exp2().repeat_interleave(32, -1)
    a = y.abs() / power
    half = torch.where(a < 2.0, 0.25, torch.where(a < 4.0, 0.5, 1.0))
    # at 2 and 4 the step grows: a value just below may round within the larger one
    half = torch.where((a + err / power >= 2.0) & (a < 2.0), 0.5, torch.where((a + err / power >= 4.0) & (a < 4.0), 1.0, half))
    assert bool(((value64(codes, scales) - y).abs() <= half * power * (1 + 2.0 ** -20) + err).all())
    # V takes neither
    s = scale64(v.double().unflatten(-1, (-1, block_of(dim, 1))).abs().amax(-1))
    assert torch.equal(v_scales(p.vs)[pg, :, slot], s)
    for was, got in zip(before, (k_codes(p.k), v_codes(p.v))):
        keep = torch.ones(got.shape[0], got.shape[2], dtype=torch.bool)
        keep[pg, slot] = False
        assert torch.equal(got.transpose(1, 2)[keep], was.transpose(1, 2)[keep])


def test_append_special_values(ctx):
    say("append4: NaN blocks, infinities, denormals and the ends of the scales")
    big = 3.0e38
    k = torch.zeros(9, 1, 128)
    k[0, 0, 5], k[1, 0, 40], k[2, 0, 70] = math.nan, math.inf, -math.inf
    k[1, 0, 41], k[3, 0, :] = 1.0, big
    k[4, 0, :], k[5, 0, 100] = 2.0 ** -140, 2.0 ** -149
    k[6, 0, :32] = torch.tensor([6.0, -6.0, 5.0, 0.24] * 8) * 2.0 ** 100
    k[7, 0, :32] = torch.tensor([6.0, -6.0, 5.0, 0.24] * 8) * 2.0 ** -100
    k[8, 0, :32] = torch.tensor([6.0000005, -6.0, 5.0, 0.24] * 8)
    for page, most in ((16, 9), (64, 9)):
        p = Paged4(3, [9], 1, 128, page)
        A.kv_append(ctx, p.cache, k.cuda(), k.cuda(), p.dev_table, cumulative([9]), ints([0]), max_new=most)
        torch.cuda.synchronize()
        p.download()
        kk, vv = p.rows(0)
        top = 6.0 * 2.0 ** 100
        assert kk[0, 0, :32].isnan().all() and not kk[0, 0, 32:].any() and vv[0].isnan().all()
        assert kk[1, 0, 40] == top and kk[1, 0, 41] == 0 and kk[2, 0, 70] == -top and vv[2, 0, 70] == -top
        assert bool((kk[3] == top).all()) and bool((vv[3] == top).all())
        assert not kk[4:6].any() and not vv[4:6].any()
        want = torch.tensor([6.0, -6.0, 4.0, 0.0] * 8, dtype=torch.float64)
        assert torch.equal(kk[6, 0, :32], want * 2.0 ** 100) and torch.equal(kk[7, 0, :32], want * 2.0 ** -100)
        # one step past 6: the scale doubles
        assert torch.equal(kk[8, 0, :32], torch.tensor([6.0, -6.0, 4.0, 0.0] * 8, dtype=torch.float64))
        pg, slot = p.place(0, 8)
        assert int(k_scales(p.ks)[pg, 0, slot, 0]) == 128
    ctx.launch_status()


@pytest.mark.parametrize("dim,kv,page", [(64, 2, 16), (128, 1, 64), (512, 1, 128)])
@pytest.mark.parametrize("past,counts,most", [([5, 0], [40, 3], 3), ([0, 15], [2, 1], 1), ([100, 7], [130, 200], 129),
                                              ([-1, 9], [3, 5], 5), ([-2 ** 31, 4], [2, 2], 2)])
def test_append_more_rows_than_planned_and_a_past_below_0(ctx, dim, kv, page, past, counts, most):
    say(f"append4 dim={dim} past={past} counts={counts} max_new={most}")
    stored = [min(b, most) if a >= 0 else 0 for a, b in zip(past, counts)]
    p, w = (Paged4(dim, [max(0, a) + b for a, b in zip(past, counts)], kv, dim, page) for _ in range(2))
    x = rand(gen(7), sum(counts), kv, dim).cuda()
    A.kv_append(ctx, p.cache, x, x, p.dev_table, cumulative(counts), ints(past), max_new=most)
    with pytest.raises(s14.S14Error, match="past" if min(past) < 0 else "max_new|new rows|length"):
        ctx.launch_status()
    at, keep = 0, []
    for n, b in zip(counts, stored):
        keep += range(at, at + b)
        at += n
    y = x[keep].contiguous()
    A.kv_append(ctx, w.cache, y, y, w.dev_table, cumulative(stored), ints([max(0, a) for a in past]), max_new=max(stored))
    ctx.launch_status()
    for t in ("k_pages", "v_pages", "k_scales", "v_scales"):
        assert torch.equal(getattr(p.cache, t), getattr(w.cache, t)), t


def test_append_bad_pages_and_positions(ctx):
    say("append4: pages outside the cache and the table take nothing, positions outside the rotation table are NaN")
    p = Paged4(4, [40, 40, 40], 2, 128, 16)
    before = [x.clone() for x in (p.k, p.v, p.ks, p.vs)]
    p.table[0, 2], p.table[1, 2] = p.k.shape[0], -1
    p.upload()
    x = rand(gen(1), 6, 2, 128).cuda()
    A.kv_append(ctx, p.cache, x, x, p.dev_table, cumulative([2, 2, 2]), ints([38, 38, 60]), max_new=2)
    with pytest.raises(s14.S14Error, match="cache page"):
        ctx.launch_status()
    p.download()
    for a, b in zip(before, (p.k, p.v, p.ks, p.vs)):
        assert torch.equal(a, b)
    p = Paged4(4, [40], 2, 128, 16)
    rope = A.Rope(table64(39, 64).float().cuda())
    A.kv_append(ctx, p.cache, x[:2], x[:2], p.dev_table, cumulative([2]), ints([38]), rope=rope, max_new=2)
    with pytest.raises(s14.S14Error, match="rotation table"):
        ctx.launch_status()
    p.download()
    k, v = p.rows(0)
    assert k[39].isnan().all() and k[38].isfinite().all() and v[38:].isfinite().all()


def test_append_slices_of_one_projection(ctx):
    say("append4 of slices, heads outermost, and without tokens")
    fused = rand(gen(5), 21, 12 * 128 + 16).cuda()
    k, v = fused[:, :256].view(21, 2, 128), fused[:, 1024:1280].view(21, 2, 128)
    swapped = rand(gen(6), 2, 21, 128).cuda().transpose(0, 1)
    for a, b in ((k, v), (swapped, k)):
        p, w = (Paged4(5, [30], 2, 128, 32) for _ in range(2))
        A.kv_append(ctx, p.cache, a, b, p.dev_table, cumulative([21]), ints([9]))
        A.kv_append(ctx, w.cache, a.contiguous(), b.contiguous(), w.dev_table, cumulative([21]), ints([9]))
        A.kv_append(ctx, w.cache, a[:0], b[:0], w.dev_table, cumulative([0]), ints([9]))
        for t in ("k_pages", "v_pages", "k_scales", "v_scales"):
            assert torch.equal(getattr(p.cache, t), getattr(w.cache, t)), t


@pytest.mark.parametrize("new", [[1, 1], [40, 9]])
def test_append_operands_of_different_types(ctx, new):
    say("append4 of f32 keys with bf16 values and the other way round")
    for kt, vt in ((F32, BF16), (BF16, F32)):
        p, w = (Paged4(5, [5 + n for n in new], 2, 128, 32) for _ in range(2))
        x, y = rand(gen(1), sum(new), 2, 128, dtype=BF16).to(kt).cuda(), rand(gen(2), sum(new), 2, 128, dtype=BF16).to(vt).cuda()
        A.kv_append(ctx, p.cache, x, y, p.dev_table, cumulative(new), ints([5, 5]), max_new=max(new))
        A.kv_append(ctx, w.cache, x.float(), y.float(), w.dev_table, cumulative(new), ints([5, 5]), max_new=max(new))
        for t in ("k_pages", "v_pages", "k_scales", "v_scales"):
            assert torch.equal(getattr(p.cache, t), getattr(w.cache, t)), t


@pytest.mark.parametrize("seqs,counts", [(256, 1), (257, 1), (70, 20), (2, 300), (5, 40)])
def test_balanced_and_planned_splits(ctx, seqs, counts):
    """Chunks set by the lengths (up to 256 sequences) and by max_len, with
    sequences without tokens, without rows, and one far longer than the rest."""
    say(f"paged4 {seqs} sequences of {counts} rows, ragged")
    g = gen(seqs)
    lengths = [int(x) for x in torch.randint(0, 200, (seqs,), generator=g)]
    lengths[0], lengths[1], lengths[-1] = 6000, 0, 700
    new = [counts] * seqs
    new[seqs // 2] = 0 if seqs > 2 else counts
    for heads, kv, dim in ((64, 1, 512), (8, 1, 128)):
        p = Paged4(seqs, lengths, kv, dim, 64)
        q = rand(gen(4), sum(new), heads, dim, dtype=BF16).cuda()
        for window in (0, 1000):
            out, lse = run_paged(ctx, p, q, new, heads, dim, window)
            for i in (0, 1, seqs // 2, seqs - 1):
                at, m = sum(new[:i]), new[i]
                k, v = p.rows(i)
                for n, end in ((min(m, 2), len(k) - m + min(m, 2)), (min(m, 1), len(k))):  # its first and last rows
                    first = at if end < len(k) else at + m - n
                    rows = slice(first, first + n)
                    want = T.attention64(q[rows].cpu(), k[:max(end, 0)], v[:max(end, 0)], dim ** -0.5, window) if n else None
                    if n:
                        check_attention(out[rows], lse[rows], want, f"sequence {i}")
    ctx.launch_status()


def test_appends_in_pieces_are_one(ctx):
    say("append4: a token's codes do not depend on how the tokens came")
    x, y = rand(gen(8), 75, 2, 64).cuda(), rand(gen(9), 75, 2, 64).cuda()
    p, w = (Paged4(5, [80], 2, 64, 32) for _ in range(2))
    A.kv_append(ctx, w.cache, x, y, w.dev_table, cumulative([75]), ints([5]))
    at = 0
    for n in (1, 1, 3, 4, 16, 2, 33, 1, 14):
        A.kv_append(ctx, p.cache, x[at:at + n], y[at:at + n], p.dev_table, cumulative([n]), ints([5 + at]))
        at += n
    assert at == 75
    for t in ("k_pages", "v_pages", "k_scales", "v_scales"):
        assert torch.equal(getattr(p.cache, t), getattr(w.cache, t)), t


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

# query heads, key heads, head size, new tokens: rows of one wavefront, of one
# workgroup through LDS in each tile size, and wide heads
EVERY_TILE = [*T.EVERY_TILE, (4, 1, 128, 8), (32, 1, 64, 1), (8, 1, 64, 40), (6, 1, 128, 24), (2, 2, 256, 5), (64, 1, 512, 4)]


@pytest.mark.parametrize("lengths,new,heads,kv,dim,page", T.PAGED)
@pytest.mark.parametrize("window,dtype", [(0, BF16), (50, F32), (1, BF16)])
def test_paged(ctx, lengths, new, heads, kv, dim, page, window, dtype):
    say(f"paged4 lens={lengths} new={new} heads={heads}/{kv} dim={dim} page={page} window={window} {dtype}")
    p = Paged4(sum(lengths) + dim, lengths, kv, dim, page)
    q = rand(gen(3), sum(new), heads, dim, dtype=BF16).cuda()
    out, lse = run_paged(ctx, p, q, new, heads, dim, window, dtype)
    check_attention(out, lse, paged_want(p, q, new, window), "paged4")
    ctx.launch_status()


@pytest.mark.parametrize("lengths,new,heads,kv,dim,page", T.ROWS)
@pytest.mark.parametrize("window,dtype", [(0, F32), (90, BF16), (1, BF16)])
def test_paged_rows(ctx, lengths, new, heads, kv, dim, page, window, dtype):
    say(f"paged4 lens={lengths} new={new} heads={heads}/{kv} dim={dim} page={page} window={window} {dtype}")
    p = Paged4(sum(lengths) + dim, lengths, kv, dim, page)
    q = rand(gen(3), sum(new), heads, dim, dtype=BF16).cuda()
    out, lse = run_paged(ctx, p, q, new, heads, dim, window, dtype)
    check_attention(out, lse, paged_want(p, q, new, window), "paged4 rows")
    ctx.launch_status()


@pytest.mark.parametrize("lengths,new,heads,kv,dim,page,window", T.CUT)
def test_paged_cut_windows_and_large_tiles(ctx, lengths, new, heads, kv, dim, page, window):
    say(f"paged4 lens={lengths} new={new} heads={heads}/{kv} dim={dim} page={page} window={window}")
    p = Paged4(sum(lengths) + dim, lengths, kv, dim, page)
    q = rand(gen(3), sum(new), heads, dim, dtype=BF16).cuda()
    out, lse = run_paged(ctx, p, q, new, heads, dim, window)
    check_attention(out, lse, paged_want(p, q, new, window), "paged4 cut")


@pytest.mark.parametrize("heads,kv,dim,new", [(32, 8, 128, 1), (4, 1, 64, 8), (64, 1, 512, 2), (8, 4, 256, 6), (16, 1, 512, 1)])
def test_paged_split_axis(ctx, heads, kv, dim, new):
    """A long sequence is cut; the result does not depend on what max_len
    promises, to the tolerance, and is the same each time."""
    say(f"paged4 split heads={heads}/{kv} dim={dim} new={new}")
    p = Paged4(9, [9001, 130], kv, dim, 64)
    q = rand(gen(4), 2 * new, heads, dim, dtype=BF16).cuda()
    want = paged_want(p, q, [new, new])
    for max_len in (9001, 64, 1, 1 << 20):
        out, lse = run_paged(ctx, p, q, [new, new], heads, dim, max_len=max_len)
        check_attention(out, lse, want, f"max_len {max_len}")
        again, _ = run_paged(ctx, p, q, [new, new], heads, dim, max_len=max_len)
        assert torch.equal(out, again)


@pytest.mark.parametrize("heads,kv,dim,new", EVERY_TILE)
def test_paged_without_cached_tokens_and_rows_that_see_nothing(ctx, heads, kv, dim, new):
    say(f"paged4 nothing to see heads={heads}/{kv} dim={dim} new={new}")
    p = Paged4(2, [0, max(1, new // 2), 40 + new], kv, dim, 16)
    q = rand(gen(4), 3 * new, heads, dim, dtype=BF16).cuda()
    out, lse = run_paged(ctx, p, q, [new] * 3, heads, dim)
    check_attention(out, lse, paged_want(p, q, [new] * 3), "few tokens")
    blind = new + new - max(1, new // 2)
    assert not out[:blind].any() and bool((lse[:blind] == -math.inf).all())
    p = Paged4(2, [0, 0], kv, dim, 16)
    out, lse = run_paged(ctx, p, q[:2 * new], [new] * 2, heads, dim)
    assert not out.any() and bool((lse == -math.inf).all())
    ctx.launch_status()


@pytest.mark.parametrize("heads,kv,dim,new", EVERY_TILE)
def test_rows_behind_the_last_sequence_stay(ctx, heads, kv, dim, new):
    """A padded batch: sequences without rows and packed rows of no sequence, on
    another stream than the current one, over a page that two sequences share."""
    say(f"paged4 padded heads={heads}/{kv} dim={dim} new={new}")
    p = Paged4(dim + new, [40 + new, 70 + new, 33], kv, dim, 32)
    p.table[1, 0] = p.table[0, 0]
    p.upload()
    counts, rows = [new, new, 0], 2 * new + 5
    x, y = (rand(gen(i), rows, kv, dim).cuda() for i in (5, 6))
    q = rand(gen(4), rows, heads, dim, dtype=BF16).cuda()
    out, lse = torch.full((rows, heads, dim), 7.0, device="cuda"), torch.full((rows, heads), 7.0, device="cuda")
    cu = ints([0, new, 2 * new, 2 * new])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    A.kv_append(ctx, p.cache, x, y, p.dev_table, cu, ints([40, 70, 33]), max_new=new, stream=stream.cuda_stream)
    A.paged_attention(ctx, q, p.cache, p.dev_table, cu, p.lens, out, lse=lse, max_new=new, max_len=70 + new,
                      stream=stream.cuda_stream)
    stream.synchronize()
    before = [t.clone() for t in (p.k, p.v, p.ks, p.vs)]
    p.download()
    new_pages = {int(p.table[i, j // 32]) for i, n in ((0, 40), (1, 70)) for j in range(n, n + new)}
    kept = [i for i in range(p.cache.pages) if i not in new_pages]
    for a, b in zip(before, (p.k, p.v, p.ks, p.vs)):
        assert torch.equal(a[kept], b[kept])
    assert bool((out[2 * new:] == 7.0).all()) and bool((lse[2 * new:] == 7.0).all())
    check_attention(out[:2 * new], lse[:2 * new], paged_want(p, q[:2 * new], counts), "padded")
    ctx.launch_status()


@pytest.mark.parametrize("heads,kv,dim,new", EVERY_TILE)
@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("window", [0, 60])
def test_paged_hidden_places_may_hold_anything(ctx, heads, kv, dim, new, page, window):
    """NaN scales, the largest and 0 behind the last token, after a row's own
    position and before its window; rows that see a NaN are NaN, and no other."""
    say(f"paged4 hidden NaN heads={heads}/{kv} dim={dim} new={new} page={page} window={window}")
    lengths = [150 + new, 97 + new]
    p = Paged4(dim + page, lengths, kv, dim, page, lo=124, hi=128)
    for i, n in enumerate(lengths):
        for j in range(n, p.need[i] * page):  # behind the sequence
            for side in range(2):
                p.set_scale(side, i, j, (255, 254, 0)[j % 3])
    # the last token's, which only the last new token sees, and one before the windows of most
    p.set_scale(0, 0, lengths[0] - 1, 255, 0)
    p.set_scale(1, 1, lengths[1] - 1, 255, 0)
    page1, slot1 = p.place(1, lengths[1] - 1)
    if window:
        for j in range(0, 60):
            p.set_scale(0, 0, j, 255)
            p.set_scale(1, 1, min(j, 30), 255)
    p.upload()
    q = rand(gen(4), 2 * new, heads, dim, dtype=BF16).cuda()
    out, lse = run_paged(ctx, p, q, [new, new], heads, dim, window=window, dtype=F32)
    want = paged_want(p, q, [new, new], window)
    assert bool(want[0][new - 1].isnan().all()) and bool(want[0][2 * new - 1, :, :min(dim, 128)].isnan().all())
    if dim > 128:
        assert not want[0][2 * new - 1, :, 128:].isnan().any() or window
    check_attention(out, None, want, "hidden")
    fin = want[1].isfinite()
    assert torch.equal(lse.cpu().isnan(), want[1].isnan())
    assert bool(((lse.cpu().double() - want[1]).abs()[fin] <= 1e-4 * (1 + want[1].abs()[fin])).all())
    ctx.launch_status()


@pytest.mark.parametrize("heads,kv,dim,new", EVERY_TILE)
def test_paged_bad_pages(ctx, heads, kv, dim, new):
    say(f"paged4 bad pages heads={heads}/{kv} dim={dim} new={new}")
    p = Paged4(9, [90 + new, 70 + new, 33 + new], kv, dim, 16)
    good = p.table.clone()
    q = rand(gen(4), 3 * new, heads, dim, dtype=BF16).cuda()
    want = paged_want(p, q, [new] * 3)
    for bad in (-1, p.k.shape[0], 0x7FFFFFFF):
        p.table = good.clone()
        p.table[1, 2] = bad
        p.upload()
        out, lse = run_paged(ctx, p, q, [new] * 3, heads, dim)
        assert bool(out[new:2 * new].isnan().all())
        for s in (slice(0, new), slice(2 * new, None)):
            check_attention(out[s], lse[s], [x[s] for x in want], "beside a bad page")
        with pytest.raises(s14.S14Error, match="cache page"):
            ctx.launch_status()


@pytest.mark.parametrize("heads,kv,dim,counts,most", [(4, 2, 128, [3, 1], 1), (8, 1, 64, [2, 9], 8), (4, 1, 128, [50, 3], 40),
                                                      (16, 1, 512, [3, 1], 2), (4, 1, 256, [9, 2], 4)])
def test_paged_more_rows_than_planned_and_lengths_outside_the_table(ctx, heads, kv, dim, counts, most):
    say(f"paged4 counts={counts} max_new={most}")
    p = Paged4(3, [100 + n for n in counts], kv, dim, 32)
    q = rand(gen(4), sum(counts), heads, dim, dtype=BF16).cuda()
    want = paged_want(p, q, counts)
    out = torch.full((sum(counts), heads, dim), 7.0, dtype=BF16, device="cuda")
    A.paged_attention(ctx, q, p.cache, p.dev_table, cumulative(counts), p.lens, out, max_new=most, max_len=150)
    with pytest.raises(s14.S14Error, match="length"):
        ctx.launch_status()
    at = 0
    for n in counts:
        m = min(n, most)
        check_attention(out[at:at + m], None, [x[at:at + m] for x in want], "planned rows")
        assert bool((out[at + m:at + n] == 7.0).all())
        at += n
    reach = p.table.shape[1] * 32
    p.table[:] = p.table[0, 0]
    p.upload()
    p.lens = ints([-5, 1 << 30])
    out, lse = run_paged(ctx, p, q, counts, heads, dim, max_len=150)
    assert not out[:counts[0]].any()
    p.lengths = [0, reach]
    check_attention(out[counts[0]:], None, [x[counts[0]:] for x in paged_want(p, q, counts)], "held to the table")
    with pytest.raises(s14.S14Error, match="length"):
        ctx.launch_status()


@pytest.mark.parametrize("heads,kv,dim,new", EVERY_TILE)
@pytest.mark.parametrize("lo", [30, 90, 160])
def test_paged_far_scales(ctx, heads, kv, dim, new, lo):
    """Scales near the ends of what the append stores, and scales of V far apart
    within a row's tokens."""
    say(f"paged4 far scales heads={heads}/{kv} dim={dim} new={new} lo={lo}")
    p = Paged4(dim, [200 + new], kv, dim, 64, lo=lo, hi=lo + 60)
    g = gen(lo)
    p.ks = torch.randint(120, 124, p.ks.shape, generator=g, dtype=U8)
    p.upload()
    q = rand(g, new, heads, dim, dtype=BF16).cuda()
    out, lse = run_paged(ctx, p, q, [new], heads, dim, dtype=F32)
    check_attention(out, lse, paged_want(p, q, [new]), "far V scales")
    p.ks, p.vs = torch.randint(lo, lo + 4, p.ks.shape, generator=g, dtype=U8), torch.full_like(p.vs, 126)
    p.upload()
    power = 2.0 ** (124 - lo)  # scores of ordinary size again
    out, lse = run_paged(ctx, p, q, [new], heads, dim, dtype=F32, scale=power / 8)
    check_attention(out, lse, paged_want(p, q, [new], scale=power / 8), "far K scales")


@pytest.mark.parametrize("heads,kv,dim,new", [(4, 1, 128, 1), (8, 1, 64, 2), (2, 1, 256, 3), (4, 1, 128, 20), (16, 1, 512, 2)])
def test_paged_extreme_scores_strides_and_places(ctx, heads, kv, dim, new):
    say(f"paged4 extreme scores, strides, output in q's place heads={heads} dim={dim}")
    p = Paged4(7, [333], kv, dim, 64, lo=127, hi=131)
    wide = rand(gen(1), new, heads + 2, dim + 16, dtype=BF16).cuda()
    q = wide[:, 1:heads + 1, 8:dim + 8] * 40  # weights of one token, most 0
    view = wide[:, 1:heads + 1, 8:dim + 8]
    view.copy_(q)
    want = paged_want(p, q, [new])
    around = wide.clone()
    out = torch.zeros(new, 2 * heads, dim, device="cuda")[:, ::2]
    A.paged_attention(ctx, view, p.cache, p.dev_table, cumulative([new]), p.lens, out, max_new=new, max_len=333)
    check_attention(out, None, want, "strided")
    A.paged_attention(ctx, view, p.cache, p.dev_table, cumulative([new]), p.lens, view, max_new=new, max_len=333)
    check_attention(view, None, want, "in place")
    around[:, 1:heads + 1, 8:dim + 8] = view
    assert torch.equal(around, wide)


@pytest.mark.parametrize("heads,kv,dim,new", [(4, 2, 128, 1), (8, 2, 128, 8), (8, 1, 64, 6), (4, 1, 128, 40), (16, 1, 512, 1),
                                              (4, 1, 256, 3), (2, 1, 256, 20)])
@pytest.mark.parametrize("page", [16, 32])
def test_paged_pages_behind_the_window_may_be_gone(ctx, heads, kv, dim, new, page):
    p = Paged4(11, [500, 203], kv, dim, page)
    q = rand(gen(4), 2 * new, heads, dim, dtype=BF16).cuda()
    want = paged_want(p, q, [new, new], 70)
    for i, n in enumerate(p.lengths):
        first = max(0, n - new - 70 + 1)
        p.table[i, :first // page] = -7
    p.upload()
    out, lse = run_paged(ctx, p, q, [new, new], heads, dim, window=70)
    check_attention(out, lse, want, "window")
    ctx.launch_status()


def test_offsets_past_32_bits(ctx):
    say("paged4 and append4: a cache of more than 2^32 bytes a side")
    pages = 70_000  # 8 heads of 128, pages of 128 tokens: 65,536 bytes of codes a page
    cache = A.KvCache4.empty(pages, 8, 128, 128)
    assert cache.k_pages.nbytes > 1 << 32
    ids = [pages - 1, 3, pages - 2]
    p = Paged4(5, [300], 8, 128, 128)
    for new_id, old in zip(ids, p.table[0, :3].tolist()):
        for t in ("k_pages", "v_pages", "k_scales", "v_scales"):
            getattr(cache, t)[new_id] = getattr(p.cache, t)[old]
    want_cache, p.cache, p.dev_table = p.cache, cache, ints([ids])
    for new in (1, 12):
        q = rand(gen(4), new, 32, 128, dtype=BF16).cuda()
        out, lse = run_paged(ctx, p, q, [new], 32, 128)
        check_attention(out, lse, paged_want(p, q, [new]), "far pages")
    x = rand(gen(6), 1, 8, 128).cuda()
    A.kv_append(ctx, cache, x, x, p.dev_table, ints([0, 1]), ints([300]))
    A.kv_append(ctx, want_cache, x, x, p.table.cuda(), ints([0, 1]), ints([300]))
    for t in ("k_pages", "v_pages", "k_scales", "v_scales"):
        assert torch.equal(getattr(cache, t)[ids[2]], getattr(want_cache, t)[int(p.table[0, 2])]), t


def test_most_sequences_of_a_call(ctx):
    say("paged4 and append4: 65,535 sequences")
    n = 65535
    cache = A.KvCache4.empty(n, 1, 16, 64)
    for t in (cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales):
        t.zero_()
    table = torch.randperm(n, generator=gen(1)).int().view(n, 1).cuda()
    cu = torch.arange(n + 1, dtype=I32, device="cuda")
    x = rand(gen(2), n, 1, 64).cuda()
    zero, one = torch.zeros(n, dtype=I32, device="cuda"), torch.ones(n, dtype=I32, device="cuda")
    A.kv_append(ctx, cache, x, x, table, cu, zero, max_new=1)
    out = torch.empty(n, 1, 64, device="cuda")
    A.paged_attention(ctx, x.to(BF16), cache, table, cu, one, out, max_new=1, max_len=1)
    torch.cuda.synchronize()
    y = x.cpu().double()
    s, ks = (scale64(y.unflatten(-1, (-1, b)).abs().amax(-1)) for b in (64, 32))
    want, key = value64(codes64(y, s, 64), s), value64(codes64(y, ks, 32), ks)
    # one token: its weight 2^d, d the rounding of its score t (in powers of two),
    # at most 2^-24 |t|, is rounded to 1, and the output is divided by it: off by
    # 2^-24 |t| ln 2, and 2^-22 for the power's and the quotient's own roundings
    score = (x.to(BF16).cpu().double() * key).sum(-1, keepdim=True).abs() / 8 * math.log2(math.e)
    assert bool(((out.cpu().double() - want).abs() <= (2.0 ** -24 * score + 2.0 ** -22) * want.abs()).all())
    with pytest.raises(s14.S14Error):
        A.kv_append(ctx, cache, x, x, torch.zeros(n + 1, 1, dtype=I32, device="cuda"), torch.arange(n + 2, dtype=I32, device="cuda"),
                    torch.zeros(n + 1, dtype=I32, device="cuda"), max_new=1)
    ctx.launch_status()


# ---------------------------------------------------------------------------
# as they are used
# ---------------------------------------------------------------------------


class Layer(T.Layer):
    """The projections and attention of a layer over the 4-bit cache, with the
    residual norm before and after."""

    def __init__(self, ctx, n):
        super().__init__(ctx, n)
        self.cache = A.KvCache4.empty(12, self.kv, 64, self.dim)
        g = gen(77)
        self.wn = [(1 + 0.1 * rand(g, self.hidden)).cuda() for _ in range(2)]
        self.h = torch.zeros(n, self.hidden, device="cuda")
        self.y2 = torch.empty(n, self.hidden, device="cuda")

    def step(self, x, cu, past, lens, pos, most, stream=None):
        """x, the layer before's output, joins the residual stream h; y2 is what the experts take."""
        A.add_rms_norm(self.ctx, x, self.wn[0], residual=self.h, residual_out=self.h, q=self.xq, scales=self.xs, stream=stream)
        for name, (w, ws) in self.w.items():
            s14.fp8_linear(self.ctx, self.xq, self.xs, w, ws, self.rows[name], round_bf16=True, stream=stream)
        q, k, v = (self.rows[n].view(self.n, -1, self.dim) for n in ("q", "k", "v"))
        A.qk_norm_rope(self.ctx, q, None, self.q16, None, q_weight=self.norm[0], rope=self.rope, positions=pos, stream=stream)
        A.kv_append(self.ctx, self.cache, k, v, self.pages, cu, past, k_weight=self.norm[1], rope=self.rope,
                    max_new=most, stream=stream)
        A.paged_attention(self.ctx, self.q16, self.cache, self.pages, cu, lens, self.out, max_new=most, max_len=200,
                          stream=stream)
        s14.act_quant_e4m3(self.ctx, self.out.view(self.n, -1), self.oq, self.os, stream=stream)
        s14.fp8_linear(self.ctx, self.oq, self.os, *self.wo, self.y, stream=stream)
        A.add_rms_norm(self.ctx, self.y, self.wn[1], residual=self.h, residual_out=self.h, y=self.y2, stream=stream)


def test_layer_prefill_then_decode(ctx):
    """Chunks of two prompts, then verify blocks and single tokens; the stages
    against 64 bits from their own inputs."""
    say("residual norm -> projections -> norm, rotation -> 4-bit cache -> attention -> projection -> residual norm")
    g = gen(21)
    past, cache = [0, 0], None
    for new in ([70, 9], [8, 1], [1, 1], [1, 8], [20, 30], [1, 1]):
        n = sum(new)
        L = Layer(ctx, n)
        L.cache = cache = cache or L.cache
        L.h.copy_(3 * rand(g, n, L.hidden))
        x = rand(g, n, L.hidden).cuda()
        h0 = L.h.cpu().double() + x.cpu().double()
        pos = ints([p + j for p, c in zip(past, new) for j in range(c)])
        lens = [p + c for p, c in zip(past, new)]
        L.step(x, cumulative(new), ints(past), ints(lens), pos, max(new))
        torch.cuda.synchronize()
        view = Paged4.__new__(Paged4)
        view.table, view.page, view.lengths, view.cache = L.pages.cpu(), 64, lens, cache
        view.download()
        check_attention(L.out, None, paged_want(view, L.q16, new), f"step {new}")
        # the newest tokens' values in the cache are the projections'
        v = L.rows["v"].view(n, -1, L.dim).cpu().double()
        s = scale64(v.unflatten(-1, (-1, L.dim)).abs().amax(-1))
        got = torch.cat([view.rows(i)[1][p:] for i, p in enumerate(past)])
        assert torch.equal(got, value64(codes64(v, s, L.dim), s))
        h1 = h0 + L.y.cpu().double()
        want = h1 / (h1.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * L.wn[1].cpu().double()
        # two additions' roundings in h, the sum of squares and three products
        tol = (L.hidden ** 0.5 + 16) * 2.0 ** -24 * want.abs() + 2.0 ** -22 * h0.abs().amax()
        assert bool(((L.y2.cpu().double() - want).abs() <= tol).all())
        past = lens
    ctx.launch_status()


def test_layer_captured_and_replayed(ctx):
    """A decode step captured into a graph, replayed with new inputs in its
    buffers between eager steps of the same context: each replay equals an
    eager run of the same step bit for bit."""
    say("graph capture of a layer's step over the 4-bit cache")
    g = gen(22)
    L, E = Layer(ctx, 2), Layer(ctx, 2)
    x, cu, past, lens, pos = torch.empty(2, L.hidden, device="cuda"), cumulative([1, 1]), ints([0, 0]), ints([1, 1]), ints([0, 0])
    for c in (L.cache, E.cache):
        for t in (c.k_pages, c.v_pages, c.k_scales, c.v_scales):
            t.zero_()
    x.copy_(rand(g, 2, L.hidden))
    L.step(x, cu, past, lens, pos, 1)  # warm
    torch.cuda.synchronize()
    L.h.zero_()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        L.step(x, cu, past, lens, pos, 1)
    for step in range(5):
        x.copy_(rand(g, 2, L.hidden))
        for t, v in ((past, [step, 2 * step]), (lens, [step + 1, 2 * step + 1]), (pos, [step, 2 * step])):
            t.copy_(torch.tensor(v, dtype=I32))
        graph.replay()
        torch.cuda.synchronize()
        E.step(x, cu, past, lens, pos, 1)
        torch.cuda.synchronize()
        for a, b in ((L.out, E.out), (L.y2, E.y2), (L.h, E.h), (L.cache.k_pages, E.cache.k_pages),
                     (L.cache.v_pages, E.cache.v_pages), (L.cache.v_scales, E.cache.v_scales)):
            assert torch.equal(a, b), step


def test_both_caches_on_one_context_and_two_contexts(ctx):
    say("split calls over caches of 8 and 4 bits in turn on one context, and two contexts on two streams")
    p8, p4 = T.Paged(9, [5000], 2, 128, 64), Paged4(9, [5000], 2, 128, 64)
    q = rand(gen(4), 1, 4, 128, dtype=BF16).cuda()
    want8, want4 = paged_want(p8, q, [1]), paged_want(p4, q, [1])
    for _ in range(3):
        for p, want in ((p8, want8), (p4, want4)):
            out, lse = run_paged(ctx, p, q, [1], 4, 128)
            check_attention(out, lse, want, "in turn")
    other = s14.Context(0)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.zeros(1, 4, 128, dtype=BF16, device="cuda") for _ in range(8)] for _ in range(2)]
    cu = cumulative([1])
    torch.cuda.synchronize()
    for i in range(8):
        for c, s, o in zip((ctx, other), streams, outs):
            with torch.cuda.stream(s):
                A.paged_attention(c, q, p4.cache, p4.dev_table, cu, p4.lens, o[i], max_new=1, max_len=5000)
    torch.cuda.synchronize()
    for o in itertools.chain(*outs):
        check_attention(o, None, want4, "two contexts")
    other.destroy()

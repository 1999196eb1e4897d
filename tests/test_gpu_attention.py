"""The attention operators against plain 64-bit implementations.

Tolerances, all from the operators' own roundings (half a step is eps / 2:
bf16 2^-8, f32 2^-24, e4m3 2^-4 relative):

  attention  a weight is rounded to bf16 once (half a step of it; 1/16 more
             covers the f32 sums and exp2), so an output is within 2^-8 * 17/16
             * sum_j w_j |v_j|, and a bf16 output's own rounding adds 2^-8 |o|;
             lse: f32 sums of D products of magnitude L in all, (D + 8) 2^-24 L,
             and the log's own 2^-20 (1 + |lse|)
  norm/rope  a sum of D squares, a root, three products and the rotation's two:
             (D + 16) 2^-24 of the pair's magnitudes; 2^-8 |y| for bf16 outputs
  append     half an e4m3 step of the page's scale: max(2^-4 |x|, 2^-10 scale),
             with the norm's and rotation's error before it
"""

from __future__ import annotations

import math
import sys

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from colormlm_amd import _native as N  # noqa: E402
from colormlm_amd import attention as A  # noqa: E402
from colormlm_amd import s14  # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F32, I32, U8 = torch.bfloat16, torch.float32, torch.int32, torch.uint8
E4M3 = torch.float8_e4m3fn


def say(msg: str) -> None:
    print(f"[gpu-test] {msg}", file=sys.stderr, flush=True)


@pytest.fixture(scope="module")
def ctx():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    c = s14.Context(0)
    yield c
    torch.cuda.synchronize()
    c.destroy()


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rand(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g).to(dtype)


def ints(values):
    return torch.tensor(values, dtype=I32, device="cuda")


def cumulative(lengths):
    return ints([0, *np.cumsum(lengths).tolist()])


def table64(positions, rot, theta=10000.0):
    inv = theta ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    a = torch.arange(positions, dtype=torch.float64)[:, None] * inv
    return torch.cat([a.cos(), a.sin()], 1)


# ---------------------------------------------------------------------------
# plain implementations
# ---------------------------------------------------------------------------


def norm_rope64(x, weight, eps, table, positions, layout, start):
    """y, and the magnitude that each y's error is relative to."""
    y = x.double()
    if weight is not None:
        y = y / (y.pow(2).mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    mag = y.abs()
    if table is not None:
        rot = table.shape[1]
        row = table.double()[positions.long()]
        c, s = row[:, None, :rot // 2], row[:, None, rot // 2:]
        i = torch.arange(rot // 2)
        a, b = (start + i, start + i + rot // 2) if layout == "half" else (start + 2 * i, start + 2 * i + 1)
        ya, yb = y[..., a], y[..., b]
        y = y.clone()
        y[..., a], y[..., b] = ya * c - yb * s, yb * c + ya * s
        mag[..., a] = mag[..., b] = ya.abs() + yb.abs()
    return y, mag


def attention64(q, k, v, scale, window):
    """q [t, heads, d], the last tokens of k, v [l, kv, d]: outputs, lse, sum w
    |v| and the largest sum |q k| scale of each row.  Keys a row does not see
    take no part, whatever they hold."""
    t, heads, d = q.shape
    length, kv = k.shape[:2]
    out, lse, mass, big = (torch.zeros(t, heads, d, dtype=torch.float64), torch.full((t, heads), -math.inf).double(),
                           torch.zeros(t, heads, d, dtype=torch.float64), torch.zeros(t, heads, dtype=torch.float64))
    qd, kd, vd = q.double(), k.double(), v.double()
    for i in range(t):
        pos = length - t + i
        lo = max(0, pos - window + 1) if window else 0
        if pos < 0 or lo > pos:
            continue
        for h in range(heads):
            kk, vv = kd[lo:pos + 1, h // (heads // kv)], vd[lo:pos + 1, h // (heads // kv)]
            s = kk @ qd[i, h] * scale
            lse[i, h] = torch.logsumexp(s, 0)
            w = (s - lse[i, h]).exp()
            out[i, h] = (w[:, None] * vv).sum(0)
            mass[i, h] = (w[:, None] * vv.abs()).sum(0)
            big[i, h] = (kk.abs() @ qd[i, h].abs()).max() * abs(scale)
    return out, lse, mass, big


def check_attention(out, lse, want, what):
    o, l, mass, big = want
    got = out.cpu().double()
    assert torch.equal(got.isnan(), o.isnan()), what
    fin = o.isfinite()
    assert torch.equal(got[~fin & ~o.isnan()], o[~fin & ~o.isnan()]), what
    tol = 2.0 ** -8 * 17 / 16 * mass + (2.0 ** -8 * o.abs() if out.dtype == BF16 else 0) + 1e-30
    err = ((got - o).abs() / tol)[fin]
    worst = float(err.max()) if err.numel() else 0.0
    say(f"  {what}: worst error {worst:.3f} of the tolerance")
    assert worst <= 1.0, what
    if lse is not None:
        got = lse.cpu().double()
        assert torch.equal(got == -math.inf, l == -math.inf), what
        ok = l.isfinite()
        tol = (out.shape[-1] + 8) * 2.0 ** -24 * big + 2.0 ** -20 * (1 + l.abs())
        assert bool(((got - l).abs() <= tol)[ok].all()), what


def quantized(g, *shape, lo=-12, hi=4):
    """Random codes (no NaN) and their values."""
    c = torch.randint(0, 256, shape, generator=g, dtype=U8)
    c[(c & 0x7F) == 0x7F] = 0x40
    return c


class Paged:
    """A random cache whose pages lie in random order, with spare pages, and
    the sequences' K and V as 64-bit rows."""

    def __init__(self, seed, lengths, kv, dim, page, width=None, lo=118, hi=122):
        g = gen(seed)
        need = [-(-n // page) for n in lengths]
        pages = sum(need) + 3
        self.cache = A.KvCache.empty(pages, kv, page, dim)
        c = self.cache
        self.k, self.v = quantized(g, pages, kv, page, dim), quantized(g, pages, kv, dim, page)
        # values of a trained size: codes of [-448, 448] with scales near 2^-7
        self.ks = torch.randint(lo, hi, (pages, kv), generator=g, dtype=U8)
        self.vs = torch.randint(lo, hi, (pages, kv), generator=g, dtype=U8)
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

    def rows(self, i, length=None):
        length = self.lengths[i] if length is None else length
        ids = self.table[i, :-(-length // self.page)].long()
        ks, vs = ((x[ids].double() - 127).exp2()[..., None, None] for x in (self.ks, self.vs))
        k = (self.k[ids].view(E4M3).double() * ks).permute(0, 2, 1, 3).flatten(0, 1)
        v = (self.v[ids].view(E4M3).double() * vs).permute(0, 3, 1, 2).flatten(0, 1)
        return k[:length], v[:length]


def run_paged(ctx, p, q, new, heads, dim, window=0, dtype=BF16, lse=True, stream=None, **kw):
    out = torch.full((q.shape[0], heads, dim), 7.0, dtype=dtype, device="cuda")
    l = torch.full((q.shape[0], heads), 7.0, device="cuda") if lse else None
    A.paged_attention(ctx, q, p.cache, p.dev_table, cumulative(new), p.lens, out, lse=l, window=window,
                      max_new=max(new), max_len=kw.pop("max_len", max(p.lengths)), stream=stream, **kw)
    torch.cuda.synchronize()
    return out, l


def paged_want(p, q, new, window=0, scale=None):
    at, parts = 0, []
    for i, n in enumerate(new):
        k, v = p.rows(i)
        parts.append(attention64(q[at:at + n].cpu(), k, v, q.shape[-1] ** -0.5 if scale is None else scale, window))
        at += n
    return [torch.cat(x) for x in zip(*parts)]


# ---------------------------------------------------------------------------
# norm and rotation
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dim,rot,start,layout,heads,kv,tokens", [
    (128, 128, 0, "half", 32, 8, 1), (64, 64, 0, "half", 3, 1, 37), (512, 64, 448, "interleaved", 5, 1, 33),
    (256, 256, 0, "interleaved", 12, 2, 7), (128, 32, 96, "half", 7, 7, 130), (128, 40, 8, "half", 2, 1, 19),
    (512, 512, 0, "half", 2, 2, 9), (64, 8, 56, "interleaved", 4, 4, 5), (512, 264, 240, "half", 3, 1, 4)])
@pytest.mark.parametrize("norm,din,dout", [("both", F32, BF16), ("q", BF16, F32), ("none", F32, F32),
                                           ("both", BF16, BF16)])
def test_norm_rope(ctx, dim, rot, start, layout, heads, kv, tokens, norm, din, dout):
    say(f"norm_rope dim={dim} rot={rot}@{start} {layout} heads={heads}/{kv} tokens={tokens} {norm} {din} {dout}")
    g = gen(dim + rot + tokens)
    q, k = rand(g, tokens, heads, dim, dtype=din) * 3, rand(g, tokens, kv, dim, dtype=din)
    qw = rand(g, dim) if norm != "none" else None
    kw = rand(g, dim) if norm == "both" else None
    table = table64(4096, rot).float()
    pos = torch.randint(0, 4096, (tokens,), generator=g, dtype=I32)
    rope = A.Rope(table.cuda(), layout, start)
    qo, ko = (torch.empty(x.shape, dtype=dout, device="cuda") for x in (q, k))
    w = [x.cuda() if x is not None else None for x in (qw, kw)]
    A.qk_norm_rope(ctx, q.cuda(), k.cuda(), qo, ko, q_weight=w[0], k_weight=w[1], eps=1e-5, rope=rope,
                   positions=pos.cuda())
    torch.cuda.synchronize()
    for x, weight, got in ((q, qw, qo), (k, kw, ko)):
        y, mag = norm_rope64(x, weight, 1e-5, table, pos, layout, start)
        tol = (dim + 16) * 2.0 ** -24 * mag + (2.0 ** -8 * y.abs() if dout == BF16 else 0) + 1e-30
        assert float(((got.cpu().double() - y).abs() / tol).max()) <= 1.0
    ctx.launch_status()


def test_norm_rope_strides_in_place_and_one_side(ctx):
    say("norm_rope on slices of one projection, in place, q alone, no tokens")
    g = gen(5)
    fused = rand(g, 50, 12 * 128 + 16).cuda()  # q, k, v heads and padding of each token's row
    q, k = fused[:, :8 * 128].view(50, 8, 128), fused[:, 8 * 128:10 * 128].view(50, 2, 128)
    before, qh, kh = fused.cpu(), q.cpu(), k.cpu()
    table = table64(64, 128).float()
    rope, pos = A.Rope(table.cuda()), torch.arange(50, dtype=I32)
    w = rand(g, 128)
    A.qk_norm_rope(ctx, q, k, q, k, q_weight=w.cuda(), k_weight=w.cuda(), rope=rope, positions=pos.cuda())
    torch.cuda.synchronize()
    for x, got in ((qh, q), (kh, k)):
        y, mag = norm_rope64(x, w, 1e-6, table, pos, "half", 0)
        assert bool(((got.cpu().double() - y).abs() <= (128 + 16) * 2.0 ** -24 * mag + 1e-30).all())
    assert torch.equal(fused.cpu()[:, 10 * 128:], before[:, 10 * 128:])
    out = torch.empty(50, 8, 128, device="cuda", dtype=BF16)
    A.qk_norm_rope(ctx, q, None, out, None)  # a plain conversion
    assert torch.equal(out, q.to(BF16))
    A.qk_norm_rope(ctx, q[:0], None, out[:0], None)
    swapped = rand(g, 4, 50, 128).cuda().transpose(0, 1)  # [tokens, heads, dim], heads outermost
    out = torch.empty(50, 4, 128, device="cuda")
    A.qk_norm_rope(ctx, swapped, None, out, None)
    assert torch.equal(out, swapped)


def test_norm_rope_special_values(ctx):
    say("norm_rope: a NaN row, an infinite row and positions outside the table stay in their rows")
    g = gen(6)
    q = rand(g, 6, 2, 128)
    q[1, 0, 5], q[2, 1, 7] = math.nan, math.inf
    rope = A.Rope(table64(16, 128).float().cuda())
    out = torch.empty(6, 2, 128, device="cuda")
    A.qk_norm_rope(ctx, q.cuda(), None, out, None, q_weight=torch.ones(128, device="cuda"), rope=rope,
                   positions=ints([0, 1, 2, 16, -1, 15]))
    bad = out.isnan().any(-1).cpu()
    assert bad.tolist() == [[False, False], [True, False], [False, True], [True, True], [True, True], [False, False]]
    assert bool(out[3:5].isnan().all())
    with pytest.raises(s14.S14Error, match="rotation table"):
        ctx.launch_status()
    ctx.launch_status()


@pytest.mark.parametrize("scaling", [None, A.RopeScaling(8.0), A.RopeScaling(32.0, 4096.0, amplitude=1.2),
                                     A.RopeScaling(4.0, 65536.0, 32.0, 1.0)])
@pytest.mark.parametrize("rot,theta", [(64, 10000.0), (128, 1e6), (8, 500.0)])
def test_rope_table(ctx, rot, theta, scaling):
    say(f"rope_table rot={rot} theta={theta} {scaling}")
    n = 70001
    t = torch.empty(n, rot, device="cuda")
    A.rope_table(ctx, t, theta, scaling)
    inv = np.float64(theta) ** (-np.arange(0, rot, 2, dtype=np.float64) / rot)
    amp = 1.0
    if scaling is not None:
        amp = scaling.amplitude
        part = np.ones(rot // 2)
        if scaling.original:
            def at(turns):  # the frequency index that turns so often in the trained length
                return rot * math.log(scaling.original / (turns * 2 * math.pi)) / (2 * math.log(theta))
            lo, hi = max(math.floor(at(scaling.beta_fast)), 0), min(math.ceil(at(scaling.beta_slow)), rot - 1)
            hi = hi if hi > lo else lo + 0.001
            part = np.clip((np.arange(rot // 2) - lo) / (hi - lo), 0, 1)
        inv = inv / scaling.factor * part + inv * (1 - part)
    a = np.arange(n, dtype=np.float64)[:, None] * inv
    want = np.concatenate([np.cos(a), np.sin(a)], 1) * amp
    # f32 rounding, and the angle's own 64-bit rounding at 70,000 turns
    assert np.max(np.abs(t.cpu().numpy() - want)) <= amp * (2.0 ** -24 + 70001 * 2.0 ** -50)


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------


def scale_code(amax):
    r = np.float32(max(np.float32(amax), np.float32(1e-4))) / np.float32(448)
    m, e = math.frexp(float(r))
    return 127 + (e - 1 if m == 0.5 else e)


def rescaled(codes, shift):
    """e4m3 codes times 2^shift, to nearest even."""
    return (codes.view(E4M3).float() * 2.0 ** shift).to(E4M3).view(U8)


APPEND = [  # lengths before, new counts, kv heads, dim, page
    ([0], [1], 1, 64, 16), ([0, 5, 64, 63], [1, 1, 1, 1], 8, 128, 64), ([299], [8], 1, 512, 64),
    ([7, 0, 31, 16], [40, 0, 1, 17], 2, 128, 16), ([100, 3], [300, 129], 1, 256, 128), ([130], [200], 3, 64, 32),
    ([10, 120], [128, 9], 1, 512, 128)]


@pytest.mark.parametrize("past,new,kv,dim,page", APPEND)
@pytest.mark.parametrize("dtype,norm,rot,layout", [(F32, True, 64, "half"), (BF16, False, 0, "half"),
                                                   (F32, False, 32, "interleaved")])
def test_append(ctx, past, new, kv, dim, page, dtype, norm, rot, layout):
    say(f"append past={past} new={new} kv={kv} dim={dim} page={page} {dtype} norm={norm} rot={rot} {layout}")
    g = gen(sum(past) + 7 * sum(new) + dim)
    p = Paged(dim + page, [a + b for a, b in zip(past, new)], kv, dim, page, lo=118, hi=124)
    tokens = sum(new)
    k, v = (rand(g, tokens, kv, dim, dtype=dtype) * torch.exp(rand(g, tokens, 1, 1)).to(dtype) for _ in range(2))
    w = rand(g, dim).abs() + 0.5 if norm else None
    table = table64(1024, rot).float() if rot else None
    start = dim - rot
    rope = A.Rope(table.cuda(), layout, start) if rot else None
    before = [x.clone() for x in (p.k, p.ks, p.v, p.vs)]
    A.kv_append(ctx, p.cache, k.cuda(), v.cuda(), p.dev_table, cumulative(new), ints(past), k_weight=w.cuda() if norm else None,
                rope=rope, max_new=max(new))
    torch.cuda.synchronize()
    ctx.launch_status()
    pos = torch.cat([torch.arange(a, a + b) for a, b in zip(past, new)])
    k64, kmag = norm_rope64(k, w, 1e-6, table, pos, layout, start)
    v64 = v.double()
    c = p.cache
    got = [x.cpu() for x in (c.k_pages, c.k_scales, c.v_pages, c.v_scales)]
    want_other = [x.clone() for x in before]
    at = 0
    for i, (a, b) in enumerate(zip(past, new)):
        for pg in range(a // page, -(-(a + b) // page) if b else 0):
            lo, hi = max(a, pg * page), min(a + b, pg * page + page)
            if lo >= hi:
                continue
            pid, kept = int(p.table[i, pg]), lo - pg * page
            rows = slice(at + lo - a, at + hi - a)
            for side, (x, mag) in enumerate(((k64, kmag), (v64, v64.abs()))):
                codes, scales, was, was_s = got[2 * side], got[2 * side + 1], before[2 * side], before[2 * side + 1]
                if side:
                    codes, was = codes.transpose(2, 3), was.transpose(2, 3)
                for h in range(kv):
                    y, err = x[rows, h], ((dim + 16) * 2.0 ** -24 * mag[rows, h] if side == 0 else 0 * mag[rows, h])
                    code = int(scales[pid, h])
                    amax, slack = float(y.abs().max()), float(err.max())
                    allowed = {max(scale_code(amax + d), int(was_s[pid, h]) if kept else 0) for d in (-slack, 0, slack)}
                    assert code in allowed, (i, pg, side, h)
                    s = 2.0 ** (code - 127)
                    val = codes[pid, h, kept:kept + hi - lo].contiguous().view(E4M3).double() * s
                    tol = torch.maximum(y.abs() * 2.0 ** -4, torch.full_like(y, s * 2.0 ** -10)) * (1 + 2.0 ** -20) + err
                    assert bool(((val - y).abs() <= tol).all()), (i, pg, side, h)
                    old = rescaled(was[pid, h, :kept].contiguous(), int(was_s[pid, h]) - code)
                    assert torch.equal(codes[pid, h, :kept], old), (i, pg, side, h)
                    assert torch.equal(codes[pid, h, kept + hi - lo:], was[pid, h, kept + hi - lo:])
                    # what this page holds now, for the comparison of the whole cache
                    want_other[2 * side + 1][pid, h] = code
                    tgt = want_other[2 * side][pid, h]
                    (tgt.transpose(0, 1) if side else tgt)[:kept + hi - lo] = codes[pid, h, :kept + hi - lo]
        at += b
    for x, y in zip(got, want_other):
        assert torch.equal(x, y)  # no other page or slot changed


def test_append_grows_a_scale_and_keeps_it(ctx):
    say("append one by one: a page's scale grows with a larger token, and never shrinks")
    cache = A.KvCache.empty(1, 1, 16, 64)
    for t in (cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales):
        t.fill_(0xFF)  # whatever was there
    table, sizes = ints([[0]]), [1.0, 0.01, 100.0, 1e-6, 3000.0, 1.0]
    g = gen(3)
    rows = torch.stack([torch.sign(rand(g, 64)) * s for s in sizes])[:, None]
    for i in range(len(sizes)):
        x = rows[i:i + 1].cuda()
        A.kv_append(ctx, cache, x, x, table, ints([0, 1]), ints([i]))
        code = scale_code(max(sizes[:i + 1]))
        assert int(cache.k_scales[0, 0]) == code and int(cache.v_scales[0, 0]) == code
    s = 2.0 ** (scale_code(3000.0) - 127)
    k = cache.k_pages.cpu().view(E4M3).double()[0, 0] * s
    v = cache.v_pages.cpu().view(E4M3).double()[0, 0].T * s
    for i, size in enumerate(sizes):
        # one rounding to e4m3 and one, below 2^-6 of the scale, when it grew
        tol = size * 2.0 ** -4 + 2 * s * 2.0 ** -10
        assert bool(((k[i] - rows[i, 0].double()).abs() <= tol).all()) and torch.equal(k[i], v[i])
    assert bool((cache.k_pages[0, 0, len(sizes):] == 0xFF).all())
    # a verify block is taken back and written again from the same position
    x = rows[1:2].cuda()
    A.kv_append(ctx, cache, x, x, table, ints([0, 1]), ints([2]))
    assert int(cache.k_scales[0, 0]) == scale_code(3000.0)
    A.kv_append(ctx, cache, x, x, table, ints([0, 1]), ints([0]))  # a page begun again forgets its scale
    assert int(cache.k_scales[0, 0]) == scale_code(0.01)


def test_append_special_values(ctx):
    say("append: NaN, infinity, zeros, bad pages and positions")
    cache = A.KvCache.empty(3, 1, 16, 64)
    for t in (cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales):
        t.zero_()
    x = torch.ones(3, 1, 64)
    x[0, 0, 3], x[1], x[2, 0, 9] = math.nan, 0.0, -math.inf
    A.kv_append(ctx, cache, x[:2].cuda(), x[:2].cuda(), ints([[1]]), ints([0, 2]), ints([0]))
    k, v = cache.k_pages.cpu(), cache.v_pages.cpu()
    assert (int(k[1, 0, 0, 3]) & 0x7F) == 0x7F and (int(v[1, 0, 3, 0]) & 0x7F) == 0x7F
    assert int(cache.k_scales[1, 0]) == scale_code(1.0) and not k[1, 0, 1].any()
    A.kv_append(ctx, cache, x[2:].cuda(), x[2:].cuda(), ints([[2]]), ints([0, 1]), ints([0]))
    assert int(cache.k_scales[2, 0]) == 254 and int(cache.k_pages[2, 0, 0, 9]) == 0xFE
    ctx.launch_status()
    before = [t.clone() for t in (cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales)]
    y = torch.ones(4, 1, 64, device="cuda")
    # a page outside the cache, a negative one, a position past the table, a negative position
    A.kv_append(ctx, cache, y, y, ints([[3], [-1], [0], [0]]), ints([0, 1, 2, 3, 4]), ints([0, 0, 16, -4]))
    with pytest.raises(s14.S14Error, match="cache page"):
        ctx.launch_status()
    for t, b in zip((cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales), before):
        assert torch.equal(t, b)
    # counts that leave the rows or run backwards touch nothing else
    A.kv_append(ctx, cache, y, y, ints([[0], [1]]), ints([3, 2, -7]), ints([0, 0]))
    A.kv_append(ctx, cache, y, y, ints([[0]]), ints([2, 1000]), ints([0]))
    assert int((cache.k_pages[0, 0] != 0).any(-1).sum()) == 2
    ctx.launch_status()


@pytest.mark.parametrize("dim,kv,page", [(64, 2, 16), (128, 1, 64), (512, 1, 128)])
@pytest.mark.parametrize("past,counts,most", [([5, 0], [40, 3], 3), ([0, 15], [2, 1], 1), ([100, 7], [130, 200], 129),
                                              ([3] * 9, [20, 1, 0, 1, 1, 1, 1, 1, 1], 17)])
def test_append_more_rows_than_planned(ctx, dim, kv, page, past, counts, most):
    """Rows past max_new of a sequence are not stored: the cache is that of the
    first max_new, and the status says so."""
    say(f"append: {counts} rows, planned for {most}, dim={dim} page={page}")
    g = gen(5)
    lengths = [a + b for a, b in zip(past, counts)]
    p, w = Paged(4, lengths, kv, dim, page), Paged(4, lengths, kv, dim, page)
    k, v = (rand(g, sum(counts), kv, dim).cuda() for _ in range(2))
    k[::3] *= 50
    A.kv_append(ctx, p.cache, k, v, p.dev_table, cumulative(counts), ints(past), max_new=most)
    with pytest.raises(s14.S14Error, match="max_new"):
        ctx.launch_status()
    start = np.cumsum([0, *counts])
    rows = torch.cat([torch.arange(a, a + min(n, most)) for a, n in zip(start, counts)]).cuda()
    kept = [min(n, most) for n in counts]
    A.kv_append(ctx, w.cache, k[rows], v[rows], w.dev_table, cumulative(kept), ints(past), max_new=most)
    ctx.launch_status()
    for x in ("k_pages", "v_pages", "k_scales", "v_scales"):
        assert torch.equal(getattr(p.cache, x), getattr(w.cache, x)), x


def test_append_before_the_first_position(ctx):
    """A past below 0 stores nothing of its sequence, and the status says so."""
    say("append: a past below 0")
    x = rand(gen(5), 5, 1, 64).cuda()
    for counts, past in (([1, 4], [-4, 0]), ([4, 1], [-1, 0]), ([5, 0], [-(1 << 31), 0]), ([0, 5], [-3, 2])):
        p, w = Paged(4, [20, 20], 1, 64, 16), Paged(4, [20, 20], 1, 64, 16)
        A.kv_append(ctx, p.cache, x, x, p.dev_table, cumulative(counts), ints(past))
        if counts[0]:
            with pytest.raises(s14.S14Error, match="past"):
                ctx.launch_status()
        ctx.launch_status()  # (of a sequence without new tokens it is not asked for)
        y = x[counts[0]:]
        A.kv_append(ctx, w.cache, y, y, w.dev_table, cumulative([0, counts[1]]), ints([0, past[1]]))
        for t in ("k_pages", "v_pages", "k_scales", "v_scales"):
            assert torch.equal(getattr(p.cache, t), getattr(w.cache, t)), t


# ---------------------------------------------------------------------------
# attention over the cache
# ---------------------------------------------------------------------------

PAGED = [  # lengths, new counts, heads, kv, dim, page
    ([1], [1], 32, 8, 128, 64), ([300], [1], 8, 2, 128, 64), ([1000, 17, 64, 1], [1, 1, 1, 1], 32, 8, 128, 64),
    ([700], [8], 32, 8, 128, 64), ([500, 90], [20, 5], 12, 2, 256, 32), ([333], [4], 64, 1, 512, 64),
    ([257, 1500], [3, 1], 16, 16, 64, 16), ([400], [33], 7, 1, 64, 128), ([129, 64, 65], [1, 2, 3], 5, 5, 128, 128),
    ([200, 0, 31], [9, 0, 31], 24, 8, 128, 16), ([77], [77], 20, 4, 128, 32), ([640], [2], 128, 1, 512, 16),
    ([50, 3000], [1, 1], 6, 2, 256, 64)]


@pytest.mark.parametrize("lengths,new,heads,kv,dim,page", PAGED)
@pytest.mark.parametrize("window,dtype", [(0, BF16), (50, F32), (1, BF16)])
def test_paged(ctx, lengths, new, heads, kv, dim, page, window, dtype):
    say(f"paged lens={lengths} new={new} heads={heads}/{kv} dim={dim} page={page} window={window} {dtype}")
    p = Paged(sum(lengths) + dim, lengths, kv, dim, page)
    q = rand(gen(3), sum(new), heads, dim, dtype=BF16).cuda()
    out, lse = run_paged(ctx, p, q, new, heads, dim, window, dtype)
    check_attention(out, lse, paged_want(p, q, new, window), "paged")
    ctx.launch_status()


@pytest.mark.parametrize("heads,kv,dim,new", [(32, 8, 128, 1), (4, 1, 64, 8), (64, 1, 512, 2), (8, 4, 256, 6)])
def test_paged_split_axis(ctx, heads, kv, dim, new):
    """A long sequence is cut; the result does not depend on what max_len
    promises (too short a promise means larger pieces), to the tolerance."""
    say(f"paged split heads={heads}/{kv} dim={dim} new={new}")
    p = Paged(9, [9001, 130], kv, dim, 64)
    q = rand(gen(4), 2 * new, heads, dim, dtype=BF16).cuda()
    want = paged_want(p, q, [new, new])
    for max_len in (9001, 64, 1, 1 << 20):
        out, lse = run_paged(ctx, p, q, [new, new], heads, dim, max_len=max_len)
        check_attention(out, lse, want, f"max_len {max_len}")
        again, _ = run_paged(ctx, p, q, [new, new], heads, dim, max_len=max_len)
        assert torch.equal(out, again)


def test_paged_rows_that_see_nothing(ctx):
    say("paged: more rows than cached tokens, empty sequences, lengths past the table")
    p = Paged(2, [3, 0, 40], 2, 128, 16)
    new = [5, 4, 2]
    q = rand(gen(4), 11, 4, 128, dtype=BF16).cuda()
    out, lse = run_paged(ctx, p, q, new, 4, 128)
    want = paged_want(p, q, new)
    check_attention(out, lse, want, "paged empty rows")
    assert not out[:2].any() and not out[5:9].any() and bool((lse[:2] == -math.inf).all())
    p.lens = ints([3, -5, 1 << 30])  # held inside the table's 3 pages of 16
    out, lse = run_paged(ctx, p, q[9:], [0, 0, 2], 4, 128)
    assert bool(out.isnan().all()) or bool(out.isfinite().all())
    p.table[2, :] = p.table[2, 0]
    p.upload()
    p.lens = ints([3, -5, 1 << 30])
    out, _ = run_paged(ctx, p, q[9:], [0, 0, 2], 4, 128)
    assert bool(out.isfinite().all())
    ctx_status(ctx)


@pytest.mark.parametrize("heads,kv,dim,new", [(4, 1, 128, 1), (32, 8, 128, 8), (8, 1, 64, 5), (8, 2, 128, 40), (16, 1, 512, 1),
                                              (64, 1, 512, 3), (12, 2, 256, 9)])
@pytest.mark.parametrize("window", [0, 70])
def test_paged_without_cached_tokens(ctx, heads, kv, dim, new, window):
    """max_len 0, the longest of empty sequences."""
    say(f"paged: nothing cached, max_len 0, heads={heads}/{kv} dim={dim} new={new} window={window}")
    p = Paged(2, [0, 0], kv, dim, 16)
    q = rand(gen(4), 2 * new, heads, dim, dtype=BF16).cuda()
    out, lse = run_paged(ctx, p, q, [new, new], heads, dim, window=window, max_len=0)
    assert not out.any() and bool((lse == -math.inf).all())
    ctx.launch_status()
    # beside one that the promise left out
    p = Paged(2, [0, 90], kv, dim, 16)
    out, lse = run_paged(ctx, p, q, [new, new], heads, dim, window=window, max_len=0)
    check_attention(out, lse, paged_want(p, q, [new, new], window), "more than promised")
    ctx.launch_status()


@pytest.mark.parametrize("seqs,new,heads,kv,dim", [(40, 33, 32, 8, 128), (96, 8, 32, 8, 64), (2, 1, 32, 8, 128), (40, 4, 64, 1, 512),
                                                   (200, 8, 12, 2, 256)])
def test_paged_longest_promise(ctx, seqs, new, heads, kv, dim):
    """max_len up to the largest that is accepted: planned by the page table's reach."""
    say(f"paged: max_len 2^31 - 1, {seqs} x {new} heads={heads}/{kv} dim={dim}")
    p = Paged(3, [70 + i % 5 for i in range(seqs)], kv, dim, 16)
    q = rand(gen(4), seqs * new, heads, dim, dtype=BF16).cuda()
    out, lse = run_paged(ctx, p, q, [new] * seqs, heads, dim)
    k, v = p.rows(seqs - 1)
    check_attention(out[-new:], lse[-new:], attention64(q[-new:].cpu(), k, v, dim ** -0.5, 0), "the last sequence")
    for most in ((1 << 31) - 1, (1 << 31) - 255, 1 << 20):
        again, lse2 = run_paged(ctx, p, q, [new] * seqs, heads, dim, max_len=most)
        assert torch.equal(again, out) and torch.equal(lse2, lse)


@pytest.mark.parametrize("heads,kv,dim,new", [(4, 2, 128, 1), (8, 2, 128, 8), (8, 1, 64, 6), (4, 1, 128, 40), (16, 1, 512, 1),
                                              (32, 1, 512, 3), (12, 2, 256, 2), (6, 1, 256, 9)])
@pytest.mark.parametrize("page", [16, 32])
def test_paged_pages_behind_the_window_may_be_gone(ctx, heads, kv, dim, new, page):
    """Pages that lie wholly before the window of a sequence's first row are not
    looked up, wherever in 64 tokens the window starts."""
    say(f"paged: pages before the window given back, heads={heads}/{kv} dim={dim} new={new} page={page}")
    window, lengths = 40, [300 + 16 * i + i % 3 for i in range(5)]
    p = Paged(6, lengths, kv, dim, page)
    q = rand(gen(4), new * len(lengths), heads, dim, dtype=BF16).cuda()
    want = paged_want(p, q, [new] * len(lengths), window)
    gone = 0
    for i, n in enumerate(lengths):
        first = (n - new - window + 1) // page  # the first page that a row sees
        p.table[i, :first] = -1 if i % 2 else 0x7FFFFFFF
        gone = max(gone, first * page - ((n - new - window + 1) & ~63))
    assert gone >= page  # some page is gone that lies behind a multiple of 64
    p.upload()
    out, lse = run_paged(ctx, p, q, [new] * len(lengths), heads, dim, window=window)
    check_attention(out, lse, want, "windowed")
    ctx.launch_status()


def test_paged_lengths_outside_the_page_table(ctx):
    """A length past the table is that of the table's reach, one below 0 is 0;
    the outputs are those, and the status says so."""
    say("paged: lengths past the page table and below 0")
    for new, dim, heads, kv in ((2, 128, 4, 2), (9, 64, 8, 1), (3, 512, 16, 1)):
        p = Paged(2, [48, 48, 20], kv, dim, 16)
        q = rand(gen(4), 3 * new, heads, dim, dtype=BF16).cuda()
        want = paged_want(p, q, [new] * 3)
        p.lens = ints([1 << 30, 48, 20])
        out, lse = run_paged(ctx, p, q, [new] * 3, heads, dim)
        check_attention(out, lse, want, "held to 48 positions")
        with pytest.raises(s14.S14Error, match="length"):
            ctx.launch_status()
        p.lens = ints([48, -5, 20])
        out, lse = run_paged(ctx, p, q, [new] * 3, heads, dim)
        assert not out[new:2 * new].any() and bool((lse[new:2 * new] == -math.inf).all())
        check_attention(out[:new], lse[:new], [x[:new] for x in want], "the sequence before")
        with pytest.raises(s14.S14Error, match="length"):
            ctx.launch_status()
        # a sequence without new tokens: its length is not asked for
        p.lens = ints([48, -5, 20])
        cu = cumulative([new, 0, new])
        out = torch.full((2 * new, heads, dim), 7.0, device="cuda")
        A.paged_attention(ctx, torch.cat([q[:new], q[2 * new:]]), p.cache, p.dev_table, cu, p.lens, out, max_new=new, max_len=48)
        check_attention(out, None, [torch.cat([x[:new], x[2 * new:]]) for x in want], "the others")
        ctx.launch_status()


@pytest.mark.parametrize("heads,kv,dim,counts,most", [(4, 2, 128, [3, 1], 1), (8, 1, 64, [2, 9], 8), (4, 1, 128, [50, 3], 40),
                                                      (16, 1, 512, [1, 4], 2)])
def test_paged_more_rows_than_planned(ctx, heads, kv, dim, counts, most):
    """Rows past max_new of a sequence stay as they were, and the status says so."""
    say(f"paged: {counts} rows, planned for {most}")
    p = Paged(2, [100, 70], kv, dim, 16)
    q = rand(gen(4), sum(counts), heads, dim, dtype=BF16).cuda()
    want = paged_want(p, q, counts)
    out = torch.full((sum(counts), heads, dim), 7.0, device="cuda")
    A.paged_attention(ctx, q, p.cache, p.dev_table, cumulative(counts), p.lens, out, max_new=most, max_len=100)
    at = 0
    for n in counts:
        s = slice(at, at + min(n, most))
        check_attention(out[s], None, [x[s] for x in want], "the first rows")
        assert bool((out[s.stop:at + n] == 7).all())
        at += n
    with pytest.raises(s14.S14Error, match="max_new"):
        ctx.launch_status()


def test_status_names_every_cause(ctx):
    say("one launch status for a page, a position and a length that are wrong")
    p = Paged(2, [100, 100], 2, 128, 16)
    p.table[0, 3] = -1
    p.upload()
    p.lens = ints([100, 1 << 20])
    q = rand(gen(4), 2, 4, 128, dtype=BF16).cuda()
    run_paged(ctx, p, q, [1, 1], 4, 128)
    x = torch.zeros(1, 1, 128, device="cuda")
    rope = A.Rope(torch.zeros(4, 128, device="cuda"))
    A.qk_norm_rope(ctx, x, None, x.clone(), None, rope=rope, positions=ints([4]))
    with pytest.raises(s14.S14Error) as e:
        ctx.launch_status()
    assert e.value.code == N.S14_ERR_INVALID
    for cause in ("cache page", "rotation table", "length"):
        assert cause in str(e.value)
    ctx.launch_status()


# query heads, key heads, head size, new tokens: rows of one wavefront, of one
# workgroup through LDS in each tile size, and wide heads
EVERY_TILE = [(4, 1, 128, 1), (4, 1, 128, 4), (8, 1, 64, 2), (4, 1, 256, 3), (4, 1, 128, 7), (4, 1, 64, 6), (4, 1, 64, 12),
              (4, 1, 128, 12), (4, 1, 128, 30), (2, 1, 256, 11), (8, 1, 64, 40), (16, 1, 512, 1), (16, 1, 512, 3)]


@pytest.mark.parametrize("heads,kv,dim,new", EVERY_TILE)
@pytest.mark.parametrize("seqs", [1, 2])
def test_paged_stored_infinities(ctx, heads, kv, dim, new, seqs):
    """A value past f32's range, which is how an infinity is stored, is infinite
    in its dimension of the rows that see it, and nowhere else."""
    say(f"paged: infinities among the values, heads={heads}/{kv} dim={dim} new={new} seqs={seqs}")
    length, page = 90, 16
    for window in (0, 50):
        first = length - new
        # the first row's own; the last row's; of a whole tile of every row; one before some rows' windows
        for pos, sign in ((first, 1), (length - 1, -1), (10, 1), (first - 45, -1)):
            p = Paged(7, [length] * seqs, kv, dim, page)
            q = (rand(gen(4), new * seqs, heads, dim) * 0.01).to(BF16).cuda()  # about equal weights
            pid, slot = int(p.table[0, pos // page]), pos % page
            p.vs[pid, 0] = 254
            p.v[pid, 0] = 0
            p.v[pid, 0, 7, slot] = 0x7E if sign > 0 else 0xFE
            p.v[pid, 0, 9] = 0x01  # 2^118: a value of the same page within the range
            p.upload()
            out, lse = run_paged(ctx, p, q, [new] * seqs, heads, dim, window=window, dtype=F32)
            o, l, mass, big = paged_want(p, q, [new] * seqs, window)
            over = o.abs() > torch.finfo(F32).max
            got = out.cpu().double()
            assert torch.equal(got.isinf(), over) and not bool(got.isnan().any()), (window, pos)
            assert bool((got[over] == sign * math.inf).all())
            hidden = [i for i in range(new) if pos > first + i or (window and pos <= first + i - window)]
            assert not bool(over[hidden].any()) and bool(over[:new, :, 7].any()) == (len(hidden) < new)
            o[over] = got[over] = 0.0
            assert bool(((got - o).abs() <= 2.0 ** -8 * 17 / 16 * mass + 1e-30)[~over].all())
            ctx.launch_status()


@pytest.mark.parametrize("heads,kv,dim,new", EVERY_TILE)
def test_paged_append_of_infinities(ctx, heads, kv, dim, new):
    """The same through kv_append, the last token's value infinite."""
    say(f"append of an infinite value, then attention: heads={heads}/{kv} dim={dim} new={new}")
    g = gen(8)
    length, page = 70 + new, 32
    k, v = rand(g, length, kv, dim), rand(g, length, kv, dim)
    v[length - 1, 0, 3] = math.inf
    q = (rand(g, new, heads, dim) * 0.1).to(BF16).cuda()
    p = Paged(7, [length], kv, dim, page)
    A.kv_append(ctx, p.cache, k.cuda(), v.cuda(), p.dev_table, ints([0, length]), ints([0]))
    pid, slot = int(p.table[0, (length - 1) // page]), (length - 1) % page
    assert int(p.cache.v_pages[pid, 0, 3, slot]) == 0x7E and int(p.cache.v_scales[pid, 0]) == 254
    out = run_paged(ctx, p, q, [new], heads, dim, dtype=F32)[0].cpu()
    assert bool((out[-1, :, 3] == math.inf).all())
    out[-1, :, 3] = 0.0
    assert bool(out.isfinite().all())


@pytest.mark.parametrize("heads,kv,dim,new", EVERY_TILE)
def test_paged_stored_infinities_under_rising_scores(ctx, heads, kv, dim, new):
    """Weights above 1, which later, larger scores have, beside a page of the
    largest scale: the infinity stays in its dimension."""
    say(f"paged: an infinity at a weight of 2^4, heads={heads}/{kv} dim={dim} new={new}")
    length, page = 330, 16
    p = Paged(7, [length], kv, dim, page)
    p.ks.fill_(127)
    p.k.zero_()
    for pos in range(256, length):
        p.k[int(p.table[0, pos // page]), :, pos % page, 0] = 0x38
    pid = int(p.table[0, 260 // page])
    p.vs[pid, 0] = 254
    p.v[pid, 0] = 0
    p.v[pid, 0, 7, 260 % page] = 0xFE
    p.upload()
    q = torch.zeros(new, heads, dim)
    q[:, :, 0] = 4 * math.log(2) * dim ** 0.5  # 2^4 times the first tokens' weights
    q = q.to(BF16).cuda()
    for max_len in (length, 1):  # cut, and in one piece
        out, _ = run_paged(ctx, p, q, [new], heads, dim, dtype=F32, max_len=max_len)
        o, _, mass, _ = paged_want(p, q, [new])
        got = out.cpu().double()
        assert bool((got[:, :, 7] == -math.inf).all())
        o[:, :, 7] = got[:, :, 7] = mass[:, :, 7] = 0.0
        assert bool(((got - o).abs() <= 2.0 ** -8 * 17 / 16 * mass + 1e-30).all())


@pytest.mark.parametrize("heads,kv,dim,new", [(4, 1, 128, 1), (4, 1, 128, 4), (8, 1, 64, 2), (4, 1, 256, 3), (4, 1, 128, 7),
                                              (4, 1, 64, 12), (4, 1, 128, 30), (2, 1, 256, 11), (16, 1, 512, 1), (16, 1, 512, 3)])
@pytest.mark.parametrize("seqs", [1, 2])
def test_paged_infinite_scores(ctx, heads, kv, dim, new, seqs):
    """A key past f32's range: a row that sees it is NaN where their product is
    positive, as if it were not there where it is negative; a row that does not
    see it has what it has without it."""
    say(f"paged: infinities among the keys, heads={heads}/{kv} dim={dim} new={new} seqs={seqs}")
    length, page = 90, 16
    first = length - new
    for pos in (length - 1, 10, first):
        p = Paged(7, [length] * seqs, kv, dim, page)
        q = rand(gen(4), new * seqs, heads, dim)
        q[:, ::2, 7], q[:, 1::2, 7] = 1.0, -1.0
        q = q.to(BF16).cuda()
        pid, slot = int(p.table[0, pos // page]), pos % page
        p.ks[pid, 0] = 254
        p.k[pid, 0] = 0
        p.k[pid, 0, slot, 7] = 0x7E
        p.upload()
        out, lse = run_paged(ctx, p, q, [new] * seqs, heads, dim, dtype=F32)
        o, l, mass, _ = paged_want(p, q, [new] * seqs)
        sees = torch.zeros(new * seqs, heads, dtype=torch.bool)
        sees[[i for i in range(new) if pos <= first + i], ::2] = True
        got = out.cpu().double()
        assert torch.equal(got.isnan().all(-1), sees) and torch.equal(got.isnan().any(-1), sees), pos
        assert torch.equal(lse.cpu().isnan(), sees)
        assert bool(((got - o).abs() <= 2.0 ** -8 * 17 / 16 * mass + 1e-30)[~sees].all())


@pytest.mark.parametrize("heads,kv,dim,n", [(4, 1, 64, 70), (2, 2, 128, 300), (4, 2, 256, 90)])
def test_scores_near_and_past_the_range(ctx, heads, kv, dim, n):
    """Scores of 2^27 pick their key; past the range, here by the scale alone, the
    rows that see them are NaN: in the prompt and through the cache."""
    say(f"scores of 2^27 and 2^128: heads={heads}/{kv} dim={dim}")
    g = gen(12)
    q, k, v = (rand(g, n, h, dim, dtype=BF16).cuda() for h in (heads, kv, kv))
    late = (torch.arange(n) >= 40)[:, None].expand(n, heads)
    for q0, k0, scale in ((2.0 ** 13, 2.0 ** 14, 1.0), (2.0 ** 60, 2.0 ** 60, 256.0), (-(2.0 ** 13), 2.0 ** 14, 1.0)):
        q[:, :, 0], k[:, :, 0] = q0, 0.0
        k[40, :, 0] = k0
        out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device="cuda")
        A.prompt_attention(ctx, q, k, v, ints([0, n]), out, lse=lse, scale=scale)
        p = Paged(7, [n], kv, dim, 32)
        A.kv_append(ctx, p.cache, k, v, p.dev_table, ints([0, n]), ints([0]))
        p.k, p.v, p.ks, p.vs = (x.cpu() for x in (p.cache.k_pages, p.cache.v_pages, p.cache.k_scales, p.cache.v_scales))
        cut = []
        for new in (1, 20):
            o, l = torch.empty_like(q[:new]), torch.empty(new, heads, device="cuda")
            A.paged_attention(ctx, q[n - new:], p.cache, p.dev_table, ints([0, new]), p.lens, o, lse=l, scale=scale)
            cut.append((new, o, l))
        if scale > 1.0:
            assert torch.equal(out.isnan().all(-1).cpu(), late) and torch.equal(out.isnan().any(-1).cpu(), late)
            assert torch.equal(lse.isnan().cpu(), late)
            assert all(bool(o.isnan().all()) and bool(l.isnan().all()) for _, o, l in cut)
            continue
        o, _, mass, _ = attention64(q.cpu(), k.cpu(), v.cpu(), scale, 0)
        # the other scores' f32 sums: 2^27 takes no part in them
        tol = 2.0 ** -8 * 17 / 16 * mass + 2.0 ** -8 * o.abs() + 1e-30
        assert bool(((out.cpu().double() - o).abs() <= tol).all())
        kk, vv = p.rows(0)
        for new, o, l in cut:
            want = attention64(q[n - new:].cpu(), kk, vv, scale, 0)
            assert bool(((o.cpu().double() - want[0]).abs() <= 2.0 ** -8 * 17 / 16 * want[2] + 2.0 ** -8 * want[0].abs() + 1e-30).all())


CUT = [  # lengths, new counts, heads, kv, dim, page, window: chunks that start behind the first token
    ([5000, 1200], [1, 1], 8, 2, 128, 16, 1500), ([4000], [8], 8, 2, 128, 64, 1900), ([6000, 300], [4, 4], 4, 1, 64, 32, 1000),
    ([5000, 2000], [9, 3], 8, 2, 128, 16, 700), ([4000, 900], [30, 12], 4, 1, 128, 64, 1200), ([3000], [60], 8, 2, 64, 32, 800),
    ([4000, 77], [2, 1], 12, 2, 256, 64, 1500), ([3500], [20], 6, 2, 256, 16, 900), ([5000, 640], [1, 1], 16, 1, 512, 16, 1100),
    ([3000], [4], 32, 1, 512, 64, 1300), ([3000, 2000], [60, 60], 4, 1, 128, 64, 0), ([3000, 2000], [60, 41], 4, 1, 128, 16, 900),
    ([2500], [70], 8, 2, 64, 64, 0), ([2500, 1000], [70, 66], 8, 2, 64, 16, 700)]


@pytest.mark.parametrize("lengths,new,heads,kv,dim,page,window", CUT)
def test_paged_cut_windows_and_large_tiles(ctx, lengths, new, heads, kv, dim, page, window):
    """Chunks that start at a window, some before some rows' own; chunks of tiles of 128 rows."""
    say(f"paged cut: lens={lengths} new={new} heads={heads}/{kv} dim={dim} page={page} window={window}")
    p = Paged(sum(lengths), lengths, kv, dim, page)
    q = rand(gen(14), sum(new), heads, dim, dtype=BF16).cuda()
    want = paged_want(p, q, new, window)
    for max_len in (max(lengths), 64, 1 << 24):
        out, lse = run_paged(ctx, p, q, new, heads, dim, window, F32, max_len=max_len)
        check_attention(out, lse, want, f"max_len {max_len}")
    ctx.launch_status()


@pytest.mark.parametrize("heads,new", [(16, 1), (16, 3)])
def test_wide_heads_keep_large_scores(ctx, heads, new):
    """At heads of 512 scores are scaled before their maximum is taken: any finite one picks its key."""
    say(f"paged: scores of 2^60 at heads of 512, {heads} x {new}")
    g = gen(12)
    n = 200
    k, v = rand(g, n, 1, 512).cuda(), rand(g, n, 1, 512).cuda()
    k[:, :, 0] = 0.0
    k[40, :, 0] = 2.0 ** 30
    q = rand(g, new, heads, 512, dtype=BF16)
    q[:, :, 0] = 2.0 ** 30
    p = Paged(7, [n], 1, 512, 32)
    A.kv_append(ctx, p.cache, k, v, p.dev_table, ints([0, n]), ints([0]))
    p.v, p.vs = p.cache.v_pages.cpu(), p.cache.v_scales.cpu()
    out, lse = run_paged(ctx, p, q.cuda(), [new], heads, 512, dtype=F32)
    _, vv = p.rows(0)
    assert torch.equal(out.cpu().double(), vv[40].expand(new, heads, 512)) and bool((lse > 2.0 ** 55).all())


def ctx_status(ctx):
    try:
        ctx.launch_status()
    except s14.S14Error:
        pass


def test_paged_bad_pages(ctx):
    say("paged: a page outside the cache makes its sequence NaN and no other")
    for bad in (-1, 10_000):
        p = Paged(2, [100, 100], 2, 128, 16)
        p.table[0, 3] = bad
        p.upload()
        q = rand(gen(4), 2, 4, 128, dtype=BF16).cuda()
        out, lse = run_paged(ctx, p, q, [1, 1], 4, 128)
        assert bool(out[0].isnan().all()) and bool(lse[0].isnan().all())
        k, v = p.rows(1)
        want = attention64(q[1:].cpu(), k, v, 128 ** -0.5, 0)
        check_attention(out[1:], lse[1:], want, "the other sequence")
        with pytest.raises(s14.S14Error, match="cache page"):
            ctx.launch_status()
        # outside the window it is not read
        out, lse = run_paged(ctx, p, q, [1, 1], 4, 128, window=20)
        assert bool(out.isfinite().all())
        ctx.launch_status()


@pytest.mark.parametrize("page", [16, 64, 128])
def test_paged_special_values_in_hidden_places(ctx, page):
    say(f"paged: NaN codes behind a sequence, after a row's position and before its window, page {page}")
    new, length, window = 8, 150, 40
    p = Paged(3, [length], 2, 128, page)
    lo = length - new
    for side in (p.k, p.v.transpose(2, 3)):
        for pos in (lo + 5, 104, length - 1):  # seen by some rows; before some rows' window; seen by the last
            side[p.table[0, pos // page].long(), 0, pos % page, 7] = 0x7F
        for pos in range(length, -(-length // page) * page):  # slots never written
            side[p.table[0, pos // page].long(), :, pos % page] = 0xFF
    p.upload()
    q = rand(gen(4), new, 4, 128, dtype=BF16).cuda()
    for w in (0, window):
        out, lse = run_paged(ctx, p, q, [new], 4, 128, window=w, lse=False)
        k, v = p.rows(0)
        want = attention64(q.cpu(), k, v, 128 ** -0.5, w)
        got = out.isnan().cpu()
        # a NaN key makes the rows that see it NaN; a NaN value its dimension
        assert torch.equal(got, want[0].isnan())
        assert bool(got[:, :2].any()) and not got[:, 2:].any() and (w == 0 or not bool(got[0].all()))
        ok = ~got
        tol = 2.0 ** -8 * 17 / 16 * want[2] + 2.0 ** -8 * want[0].abs()
        assert bool(((out.cpu().double() - want[0]).abs() <= tol)[ok].all())
    p.k[p.table[0, (lo + 5) // page].long(), 0, (lo + 5) % page, 7] = 0x10  # the values alone
    p.k[p.table[0, 104 // page].long(), 0, 104 % page, 7] = 0x10
    p.k[p.table[0, (length - 1) // page].long(), 0, (length - 1) % page, 7] = 0x10
    p.upload()
    for w in (0, window):
        out, _ = run_paged(ctx, p, q, [new], 4, 128, window=w)
        k, v = p.rows(0)
        want = attention64(q.cpu(), k, v, 128 ** -0.5, w)[0]
        assert torch.equal(out.isnan().cpu(), want.isnan()) and not bool(want[:, 0].isnan().all())


ROWS = [  # lengths, new counts, heads, kv, dim, page: rows (token, query head of the key head) of each count a workgroup takes
    ([300, 65, 1], [3, 2, 1], 8, 1, 64, 16), ([200, 130], [5, 5], 8, 1, 64, 64), ([500, 70], [40, 33], 16, 2, 64, 32),
    ([330], [17], 48, 3, 64, 128), ([100, 700, 64], [8, 8, 7], 8, 2, 128, 64), ([129, 40], [2, 1], 24, 1, 128, 16),
    ([900], [12], 4, 1, 128, 128), ([260, 31], [16, 16], 8, 2, 128, 32), ([300, 64, 5], [33, 64, 2], 4, 2, 128, 64),
    ([400, 90], [90, 3], 6, 2, 128, 16), ([257], [3], 6, 1, 256, 64), ([70, 600], [20, 9], 8, 2, 256, 16),
    ([333, 12, 64], [70, 12, 1], 2, 1, 256, 128)]


@pytest.mark.parametrize("lengths,new,heads,kv,dim,page", ROWS)
@pytest.mark.parametrize("window,dtype", [(0, F32), (90, BF16), (1, BF16)])
def test_paged_rows(ctx, lengths, new, heads, kv, dim, page, window, dtype):
    say(f"paged rows lens={lengths} new={new} heads={heads}/{kv} dim={dim} page={page} window={window} {dtype}")
    p = Paged(sum(lengths) + 3 * dim, lengths, kv, dim, page, lo=112, hi=124)
    q = rand(gen(13), sum(new), heads, dim, dtype=BF16).cuda()
    out, lse = run_paged(ctx, p, q, new, heads, dim, window, dtype)
    want = paged_want(p, q, new, window)
    check_attention(out, lse, want, "paged rows")
    ctx.launch_status()
    # planned for shorter ones: larger pieces of the same sequences
    out, lse = run_paged(ctx, p, q, new, heads, dim, window, dtype, max_len=1)
    check_attention(out, lse, want, "paged rows, uncut")


@pytest.mark.parametrize("heads,dim,new", [(4, 64, 6), (4, 64, 80), (4, 128, 7), (4, 128, 12), (4, 128, 60), (2, 256, 11)])
def test_paged_rows_special_values_and_bad_pages(ctx, heads, dim, new):
    say(f"paged rows: NaN codes that some rows see, rubbish behind the sequences, a bad page; {heads} heads of {dim}, {new} new")
    lengths, page = [150, 90], 32
    p = Paged(7, lengths, 1, dim, page)
    seen = (lengths[0] - new + 3, 20, lengths[0] - 1)  # by some rows; before some windows; by the last row
    for side, codes in ((0, p.k), (1, p.v.transpose(2, 3))):
        for pos in seen:
            codes[p.table[0, pos // page].long(), 0, pos % page, 7] = 0x7F if side else 0xFF
        for i, n in enumerate(lengths):
            for pos in range(n, -(-n // page) * page):
                codes[p.table[i, pos // page].long(), :, pos % page] = 0xFF
    p.upload()
    q = rand(gen(4), 2 * new, heads, dim, dtype=BF16).cuda()
    for keys in (True, False):
        if not keys:  # the values alone
            for pos in seen:
                p.k[p.table[0, pos // page].long(), 0, pos % page, 7] = 0x10
            p.upload()
        for w in (0, 50):
            out, _ = run_paged(ctx, p, q, [new, new], heads, dim, window=w)
            want = paged_want(p, q, [new, new], w)
            assert torch.equal(out.isnan().cpu(), want[0].isnan())
            assert bool(want[0].isnan().any()) and not bool(out[new:].isnan().any())
            tol = 2.0 ** -8 * 17 / 16 * want[2] + 2.0 ** -8 * want[0].abs()
            ok = ~want[0].isnan()
            assert bool(((out.cpu().double() - want[0]).abs() <= tol)[ok].all())
    ctx.launch_status()
    p.table[0, 1] = 10_000
    p.upload()
    out, lse = run_paged(ctx, p, q, [new, new], heads, dim)
    assert bool(out[:new].isnan().all()) and bool(lse[:new].isnan().all()) and bool(out[new:].isfinite().all())
    with pytest.raises(s14.S14Error, match="cache page"):
        ctx.launch_status()


@pytest.mark.parametrize("heads,kv,dim,new", [(8, 2, 128, 1), (8, 1, 128, 3), (8, 1, 64, 7), (4, 1, 256, 9), (16, 1, 512, 2)])
@pytest.mark.parametrize("lo", [40, 200])
def test_paged_far_scales(ctx, heads, kv, dim, new, lo):
    """Page scales far from 1 on the values' side, and on the keys' with queries
    that undo them."""
    say(f"paged: scales near 2^{lo - 127}, heads={heads}/{kv} dim={dim} new={new}")
    p = Paged(5, [200, 70], kv, dim, 32, lo=lo, hi=lo + 6)
    q = (rand(gen(4), 2 * new, heads, dim) * 2.0 ** (120 - lo)).to(BF16).cuda()
    out, _ = run_paged(ctx, p, q, [new, new], heads, dim, dtype=F32, lse=False)
    o, _, mass, _ = paged_want(p, q, [new, new])
    # Below 2^-126 a bf16 weight or an f32 product may count as zero.  A weight
    # stands beside a code (448 at most), a product beside none, and the weights'
    # sum is at least 1: 200 tokens lose at most 200 * 448 * 2^-126.
    tol = 2.0 ** -8 * 17 / 16 * mass + 200 * 448 * 2.0 ** -126
    assert bool(((out.cpu().double() - o).abs() <= tol).all())


def test_paged_strides_scale_and_extreme_scores(ctx):
    say("paged: a slice of a projection as q, output in a wider row, large scores")
    p = Paged(3, [70, 200], 2, 128, 32, lo=124, hi=127)
    new = [2, 1]
    wide = (rand(gen(4), 3, 3 * 4 * 128, dtype=BF16) * 20).cuda()
    q = wide[:, 512:1024].view(3, 4, 128)
    buf = torch.zeros(3, 10, 128, dtype=F32, device="cuda")
    out = buf[:, 3:7]
    A.paged_attention(ctx, q, p.cache, p.dev_table, cumulative(new), p.lens, out, scale=0.5, max_new=2, max_len=200)
    torch.cuda.synchronize()
    check_attention(out, None, paged_want(p, q, new, scale=0.5), "strided, scores of thousands")
    assert not buf[:, :3].any() and not buf[:, 7:].any()


def test_paged_offsets_past_32_bits(ctx):
    say("paged and append: a cache of more than 2^32 bytes a side")
    pages = 36_000  # of 1 * 128 * 1 heads: 128 tokens, 8 heads of 128: 131,072 bytes a page
    cache = A.KvCache.empty(pages, 8, 128, 128)
    assert cache.k_pages.nbytes > 1 << 32
    ids = [pages - 1, 3, pages - 2]
    p = Paged(5, [300], 8, 128, 128)
    for new_id, old in zip(ids, p.table[0, :3].tolist()):
        cache.k_pages[new_id], cache.v_pages[new_id] = p.cache.k_pages[old], p.cache.v_pages[old]
        cache.k_scales[new_id], cache.v_scales[new_id] = p.cache.k_scales[old], p.cache.v_scales[old]
    want_cache, p.cache, p.dev_table = p.cache, cache, ints([ids])
    q = rand(gen(4), 1, 32, 128, dtype=BF16).cuda()
    out, lse = run_paged(ctx, p, q, [1], 32, 128)
    check_attention(out, lse, paged_want(p, q, [1]), "far pages")
    x = rand(gen(6), 1, 8, 128).cuda()
    A.kv_append(ctx, cache, x, x, p.dev_table, ints([0, 1]), ints([300]))
    A.kv_append(ctx, want_cache, x, x, p.table.cuda(), ints([0, 1]), ints([300]))
    last = int(p.table[0, 2])
    assert torch.equal(cache.k_pages[ids[2]], want_cache.k_pages[last])
    assert torch.equal(cache.v_pages[ids[2]], want_cache.v_pages[last])


# ---------------------------------------------------------------------------
# prompts
# ---------------------------------------------------------------------------


def prompt_want(q, k, v, lengths, window=0):
    at, parts = 0, []
    for n in lengths:
        s = slice(at, at + n)
        parts.append(attention64(q[s].cpu(), k[s].cpu(), v[s].cpu(), q.shape[-1] ** -0.5, window))
        at += n
    return [torch.cat(x) for x in zip(*parts)]


def run_prompt(ctx, q, k, v, lengths, window=0, dtype=BF16):
    out = torch.full(q.shape, 7.0, dtype=dtype, device="cuda")
    lse = torch.full(q.shape[:2], 7.0, device="cuda")
    A.prompt_attention(ctx, q, k, v, cumulative(lengths), out, lse=lse, window=window)
    torch.cuda.synchronize()
    return out, lse


PROMPT = [([1], 4, 1, 128), ([130], 8, 2, 128), ([5, 0, 64, 1, 33], 4, 4, 64), ([257, 3], 6, 1, 64),
          ([200], 12, 2, 256), ([33, 65, 31], 3, 3, 256), ([63, 129, 64, 1], 32, 8, 128), ([300], 7, 7, 128),
          ([2] * 70 + [140], 4, 2, 64)]


@pytest.mark.parametrize("lengths,heads,kv,dim", PROMPT)
@pytest.mark.parametrize("window,dtype", [(0, BF16), (40, F32), (1, BF16)])
def test_prompt(ctx, lengths, heads, kv, dim, window, dtype):
    say(f"prompt lens={lengths[:6]} heads={heads}/{kv} dim={dim} window={window} {dtype}")
    g, t = gen(sum(lengths) + dim), sum(lengths)
    q, k, v = (rand(g, t, h, dim, dtype=BF16).cuda() for h in (heads, kv, kv))
    out, lse = run_prompt(ctx, q, k, v, lengths, window, dtype)
    check_attention(out, lse, prompt_want(q, k, v, lengths, window), "prompt")


def test_prompt_strides_and_rows_behind(ctx):
    say("prompt: q, k, v slices of one projection; rows behind the last sequence stay; counts that lie")
    g = gen(8)
    fused = rand(g, 90, 12 * 128, dtype=BF16).cuda()
    q, k, v = (fused[:, a * 128:b * 128].view(90, -1, 128) for a, b in ((0, 8), (8, 10), (10, 12)))
    lengths = [40, 30]  # of 90 rows
    out, lse = run_prompt(ctx, q, k, v, lengths)
    check_attention(out[:70], lse[:70], prompt_want(q[:70], k[:70], v[:70], lengths), "strided")
    assert bool((out[70:] == 7).all()) and bool((lse[70:] == 7).all())
    heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)
    again, _ = run_prompt(ctx, heads_first, k, v, lengths)
    assert torch.equal(again, out)
    o2 = torch.full_like(out, 7.0)
    A.prompt_attention(ctx, q, k, v, ints([-3, 40, 20, 1 << 30]), o2)  # held inside the rows; the second is empty
    assert torch.equal(o2[:20], out[:20]) and bool(o2.isfinite().all())


def test_prompt_special_values_in_hidden_places(ctx):
    say("prompt: infinities and NaN reach the rows that see them and no others")
    g = gen(9)
    q, k, v = (rand(g, 100, h, 128, dtype=BF16) for h in (4, 2, 2))
    v[70, 0, 3], v[71, 0, 4], v[72, 0, 4], v[40, 0, 5], v[95, 1, 9] = math.inf, -math.inf, math.inf, math.nan, math.inf
    k[80, 1, 0] = math.nan
    q[10, 0, 0] = math.nan
    lengths = [90, 10]
    for window in (0, 16):
        out, lse = run_prompt(ctx, q.cuda(), k.cuda(), v.cuda(), lengths, window)
        want = prompt_want(q, k, v, lengths, window)
        check_attention(out, None, want, f"special values, window {window}")


@pytest.mark.parametrize("heads,dim", [(2, 128), (3, 64), (2, 256)])
@pytest.mark.parametrize("window", [0, 90])
def test_prompt_special_values_one_head_a_key(ctx, heads, dim, window):
    """One query head a key head: a workgroup's rows are 128 tokens, and its
    wavefronts see different tiles whole.  An odd value before, in and behind
    each of them."""
    say(f"prompt: odd values, heads={heads} dim={dim} window={window}")
    g = gen(19)
    q, k, v = (rand(g, 300, heads, dim, dtype=BF16) for _ in range(3))
    for i, (pos, val) in enumerate([(5, math.inf), (64, math.nan), (70, -math.inf), (127, math.inf), (128, -math.inf),
                                    (190, math.nan), (191, math.inf), (255, -math.inf), (299, math.inf)]):
        v[pos, 0, 2 * i + 1] = val
    out, lse = run_prompt(ctx, q.cuda(), k.cuda(), v.cuda(), [300], window)
    check_attention(out, lse, prompt_want(q, k, v, [300], window), "odd values")


@pytest.mark.parametrize("lengths", [[130, 0, 70, 1, 200, 90], [300, 2], [1, 129, 64] * 21 + [257], [64] * 64, [70, 60] * 40])
@pytest.mark.parametrize("heads,kv,dim,dtype", [(64, 1, 64, BF16), (64, 2, 128, F32), (40, 1, 256, BF16)])
def test_prompt_blocks_of_several_sequences(ctx, lengths, heads, kv, dim, dtype):
    """Whatever order the sequences' blocks are taken in, each sequence has the
    bits that it has alone."""
    say(f"prompt: {len(lengths)} sequences {lengths[:4]} heads={heads}/{kv} dim={dim} {dtype}")
    g, t = gen(len(lengths)), sum(lengths)
    q, k, v = (rand(g, t, h, dim, dtype=BF16).cuda() for h in (heads, kv, kv))
    out, lse = run_prompt(ctx, q, k, v, lengths, dtype=dtype)
    at = 0
    for n in lengths:
        if n:
            s = slice(at, at + n)
            alone, alone_lse = run_prompt(ctx, q[s], k[s], v[s], [n], dtype=dtype)
            assert torch.equal(out[s], alone) and torch.equal(lse[s], alone_lse)
        at += n
    s = slice(0, lengths[0])
    check_attention(out[s], lse[s], attention64(q[s].cpu(), k[s].cpu(), v[s].cpu(), dim ** -0.5, 0), "the first sequence")


@pytest.mark.parametrize("heads,kv,dim", [(4, 1, 128), (2, 2, 64), (2, 1, 256)])
def test_prompt_long(ctx, heads, kv, dim):
    say(f"prompt of 2,900 tokens heads={heads}/{kv} dim={dim}: late rows against 64 bits, all against the cut form")
    g = gen(10)
    q, k, v = (rand(g, 2900, h, dim, dtype=BF16).cuda() for h in (heads, kv, kv))
    q *= 3  # a few keys carry the weight
    out, lse = run_prompt(ctx, q, k, v, [2900])
    want = attention64(q[-3:].cpu(), k.cpu(), v.cpu(), dim ** -0.5, 0)
    check_attention(out[-3:], lse[-3:], want, "last rows")


def test_prompt_counts_that_lie(ctx):
    """Bounds are held inside the rows: one that runs backwards is an empty
    sequence, one past the rows ends there."""
    say("prompt: counts outside the rows, each sequence against its own run")
    g = gen(8)
    q, k, v = (rand(g, 90, h, 128, dtype=BF16).cuda() for h in (8, 2, 2))
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
    A.prompt_attention(ctx, q, k, v, ints([-3, 40, 20, 1 << 30]), out, lse=lse)
    first = run_prompt(ctx, q[:40], k[:40], v[:40], [40])
    last = run_prompt(ctx, q[20:], k[20:], v[20:], [70])
    # rows 20 to 39 stand in both: either's
    assert torch.equal(out[:20], first[0][:20]) and torch.equal(lse[:20], first[1][:20])
    assert torch.equal(out[40:], last[0][20:]) and torch.equal(lse[40:], last[1][20:])
    both = (out[20:40] == first[0][20:]) | (out[20:40] == last[0][:20])
    assert bool(both.all())


@pytest.mark.parametrize("heads,kv,dim,lengths,window", [(4, 1, 128, [2900], 0), (2, 2, 64, [1500, 700], 0), (2, 1, 256, [1300], 0),
                                                         (4, 4, 128, [1100, 64, 900], 700), (3, 1, 64, [1700], 1000)])
def test_prompt_every_row_of_long_ones(ctx, heads, kv, dim, lengths, window):
    """Every row of prompts whose tiles are mostly walked without a mask."""
    say(f"prompt {lengths} heads={heads}/{kv} dim={dim} window={window}: every row")
    g, t = gen(31), sum(lengths)
    q, k, v = (rand(g, t, h, dim, dtype=BF16).cuda() for h in (heads, kv, kv))
    q *= 2
    out, lse = run_prompt(ctx, q, k, v, lengths, window, F32)
    at = 0
    for n in lengths:
        i = torch.arange(n)
        hidden = i[None] > i[:, None]
        if window:
            hidden |= i[None] <= i[:, None] - window
        for h in range(heads):
            qd, kd, vd = (x[at:at + n, j].cpu().double() for x, j in ((q, h), (k, h // (heads // kv)), (v, h // (heads // kv))))
            s = (qd @ kd.T * dim ** -0.5).masked_fill(hidden, -math.inf)
            l = s.logsumexp(-1)
            w = (s - l[:, None]).exp()
            big = (qd.abs() @ kd.abs().T * dim ** -0.5).masked_fill(hidden, 0.0).amax(-1)
            o, mass = w @ vd, w @ vd.abs()
            assert bool(((out[at:at + n, h].cpu().double() - o).abs() <= 2.0 ** -8 * 17 / 16 * mass + 1e-30).all()), (at, h)
            tol = (dim + 8) * 2.0 ** -24 * big + 2.0 ** -20 * (1 + l.abs())
            assert bool(((lse[at:at + n, h].cpu().double() - l).abs() <= tol).all()), (at, h)
        at += n


# ---------------------------------------------------------------------------
# together, streams, graphs
# ---------------------------------------------------------------------------


def test_prompt_and_cache_agree(ctx):
    """The same prompt through prompt_attention, and through the cache with
    values that e4m3 holds exactly: both within the tolerance of one result."""
    say("prompt attention against append + paged attention")
    g = gen(11)
    n, heads, kv, dim = 140, 8, 2, 128
    q = rand(g, n, heads, dim, dtype=BF16).cuda()
    k, v = (rand(g, n, kv, dim).to(E4M3).float().to(BF16).cuda() for _ in range(2))
    k[::16, :, 0] = 448.0  # every page's scale is 1: the values are their codes
    v[::16, :, 0] = 448.0
    cache = A.KvCache.empty(9, kv, 16, dim)
    table = ints([[8, 0, 7, 1, 6, 2, 5, 3, 4]])
    A.kv_append(ctx, cache, k, v, table, ints([0, n]), ints([0]))
    assert bool((cache.k_scales == 127).all())
    out, lse = run_prompt(ctx, q, k, v, [n])
    out2, lse2 = torch.empty_like(out), torch.empty_like(lse)
    A.paged_attention(ctx, q, cache, table, ints([0, n]), ints([n]), out2, lse=lse2)
    want = prompt_want(q, k, v, [n])
    check_attention(out, lse, want, "prompt")
    check_attention(out2, lse2, want, "cache")


class Layer:
    """The attention half of a layer: FP8 projections, norms and rotation, the
    cache, attention and the output projection, in preallocated buffers."""

    hidden, heads, kv, dim = 1024, 8, 2, 128

    def __init__(self, ctx, tokens, seed=0):
        g = gen(seed)
        self.ctx, self.n = ctx, tokens
        rows = {"q": self.heads * self.dim, "k": self.kv * self.dim, "v": self.kv * self.dim}
        mat = lambda n, k: (rand(g, n, k).clamp(-4, 4) * 16).to(E4M3).view(U8).cuda()  # noqa: E731
        tile = lambda n, k: torch.full((-(-n // 128), k // 128), 118, dtype=U8, device="cuda")  # noqa: E731
        self.w = {x: (mat(n, self.hidden), tile(n, self.hidden)) for x, n in rows.items()}
        self.wo = mat(self.hidden, rows["q"]), tile(self.hidden, rows["q"])
        f32 = lambda *s: torch.empty(s, device="cuda")  # noqa: E731
        self.rows = {x: f32(tokens, n) for x, n in rows.items()}
        self.xq, self.xs = (torch.empty(tokens, s, dtype=U8, device="cuda") for s in (self.hidden, self.hidden // 128))
        self.oq, self.os = (torch.empty(tokens, s, dtype=U8, device="cuda") for s in (rows["q"], rows["q"] // 128))
        self.q16 = torch.empty(tokens, self.heads, self.dim, dtype=BF16, device="cuda")
        self.out, self.y = f32(tokens, self.heads, self.dim), f32(tokens, self.hidden)
        self.norm = [(1 + 0.1 * rand(g, self.dim)).cuda() for _ in range(2)]
        self.table = f32(512, self.dim)
        A.rope_table(ctx, self.table)
        self.rope = A.Rope(self.table)
        self.cache = A.KvCache.empty(12, self.kv, 64, self.dim)
        self.pages = ints([[3, 5, 1, 0], [2, 4, 7, 6]])

    def project(self, x, stream=None):
        s14.act_quant_e4m3(self.ctx, x, self.xq, self.xs, stream=stream)
        for name, (w, ws) in self.w.items():
            s14.fp8_linear(self.ctx, self.xq, self.xs, w, ws, self.rows[name], round_bf16=True, stream=stream)

    def step(self, x, cu, past, lens, pos, most, stream=None):
        self.project(x, stream)
        q, k, v = (self.rows[n].view(self.n, -1, self.dim) for n in ("q", "k", "v"))
        A.qk_norm_rope(self.ctx, q, None, self.q16, None, q_weight=self.norm[0], rope=self.rope, positions=pos, stream=stream)
        A.kv_append(self.ctx, self.cache, k, v, self.pages, cu, past, k_weight=self.norm[1], rope=self.rope,
                    max_new=most, stream=stream)
        A.paged_attention(self.ctx, self.q16, self.cache, self.pages, cu, lens, self.out, max_new=most, max_len=200,
                          stream=stream)
        s14.act_quant_e4m3(self.ctx, self.out.view(self.n, -1), self.oq, self.os, stream=stream)
        s14.fp8_linear(self.ctx, self.oq, self.os, *self.wo, self.y, stream=stream)


def test_layer_prefill_then_decode(ctx):
    """A prompt of two sequences, then verify blocks and single tokens, through
    the projections as a program runs them; every stage against 64 bits from
    the stage's own inputs."""
    say("projections -> norm, rotation -> cache -> attention -> projection")
    g = gen(21)
    first = [70, 9]
    t = sum(first)
    L = Layer(ctx, t)
    L.project(rand(g, t, L.hidden).cuda())
    q, k, v = (L.rows[n].view(t, -1, L.dim) for n in ("q", "k", "v"))
    pos = torch.cat([torch.arange(n) for n in first]).int()
    k16, v16 = torch.empty(t, L.kv, L.dim, dtype=BF16, device="cuda"), v.to(BF16)
    A.qk_norm_rope(ctx, q, k, L.q16, k16, q_weight=L.norm[0], k_weight=L.norm[1], rope=L.rope, positions=pos.cuda())
    cu = cumulative(first)
    out, lse = run_prompt(ctx, L.q16, k16, v16, first)
    for x, w, got in ((q, L.norm[0], L.q16), (k, L.norm[1], k16)):
        y, mag = norm_rope64(x.cpu(), w.cpu(), 1e-6, L.table.cpu(), pos, "half", 0)
        assert bool(((got.cpu().double() - y).abs() <= 144 * 2.0 ** -24 * mag + 2.0 ** -8 * y.abs()).all())
    check_attention(out, lse, prompt_want(L.q16, k16, v16, first), "prompt of the layer")
    A.kv_append(ctx, L.cache, k16, v16, L.pages, cu, ints([0, 0]), max_new=max(first))
    past = list(first)
    for new in ([8, 1], [1, 1], [1, 8], [1, 1]):
        n = sum(new)
        D = Layer(ctx, n)
        D.cache = L.cache
        pos = ints([p + j for p, c in zip(past, new) for j in range(c)])
        lens = [p + c for p, c in zip(past, new)]
        D.step(rand(g, n, D.hidden).cuda(), cumulative(new), ints(past), ints(lens), pos, max(new))
        torch.cuda.synchronize()
        view = Paged.__new__(Paged)
        view.table, view.page, view.lengths = L.pages.cpu(), 64, lens
        view.k, view.v, view.ks, view.vs = (x.cpu() for x in (L.cache.k_pages, L.cache.v_pages, L.cache.k_scales,
                                                             L.cache.v_scales))
        check_attention(D.out, None, paged_want(view, D.q16, new), f"step {new}")
        assert bool(D.y.isfinite().all())
        past = lens
    ctx.launch_status()


def test_layer_captured_and_replayed(ctx):
    """A decode step captured into a graph, replayed with new inputs in its
    buffers between eager steps of the same context: each replay equals an
    eager run of the same step bit for bit."""
    say("graph capture of a layer's step")
    g = gen(22)
    L, E = Layer(ctx, 2), Layer(ctx, 2)
    x, cu, past, lens, pos = torch.empty(2, L.hidden, device="cuda"), cumulative([1, 1]), ints([0, 0]), ints([1, 1]), ints([0, 0])
    for c in (L.cache, E.cache):
        for t in (c.k_pages, c.v_pages, c.k_scales, c.v_scales):
            t.zero_()
    x.copy_(rand(g, 2, L.hidden))
    L.step(x, cu, past, lens, pos, 1)  # warm
    torch.cuda.synchronize()
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
        for a, b in ((L.out, E.out), (L.y, E.y), (L.cache.k_pages, E.cache.k_pages), (L.cache.v_scales, E.cache.v_scales)):
            assert torch.equal(a, b), step


def test_first_split_call_may_be_captured():
    say("the workspace of a split attention is made under capture")
    c = s14.Context(0)
    p = Paged(9, [5000], 2, 128, 64)
    q = rand(gen(4), 1, 4, 128, dtype=BF16).cuda()
    cu, out = cumulative([1]), torch.zeros(1, 4, 128, dtype=BF16, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        A.paged_attention(c, q, p.cache, p.dev_table, cu, p.lens, out, max_new=1, max_len=5000)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        check_attention(out, None, paged_want(p, q, [1]), "captured")
    del graph
    c.destroy()


def test_another_stream(ctx):
    say("the current torch stream, and one given by handle")
    p = Paged(9, [3000], 2, 128, 64)
    q = rand(gen(4), 1, 4, 128, dtype=BF16).cuda()
    want = paged_want(p, q, [1])
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        out = torch.empty(1, 4, 128, dtype=BF16, device="cuda")
        A.paged_attention(ctx, q, p.cache, p.dev_table, cumulative([1]), p.lens, out, max_new=1, max_len=3000)
    s.synchronize()
    check_attention(out, None, want, "current stream")
    out, _ = run_paged(ctx, p, q, [1], 4, 128, stream=s.cuda_stream)
    check_attention(out, None, want, "given stream")


def test_calls_without_tokens(ctx):
    say("no tokens: every call returns, a rotation's positions and the tables as empty as the rows")
    x, none = torch.empty(0, 4, 64, device="cuda"), torch.empty(0, dtype=I32, device="cuda")
    rope = A.Rope(torch.empty(8, 64, device="cuda"))
    A.qk_norm_rope(ctx, x, x, x, x, rope=rope, positions=none)
    cache = A.KvCache.empty(2, 4, 16, 64)
    table = torch.empty(0, 1, dtype=I32, device="cuda")
    A.kv_append(ctx, cache, x, x, table, ints([0]), none, rope=rope)
    y = x.to(BF16)
    A.paged_attention(ctx, y, cache, table, ints([0]), none, y)
    A.prompt_attention(ctx, y, y, y, ints([0]), y)
    torch.cuda.synchronize()


def test_outputs_in_their_inputs_place(ctx):
    say("outputs in the place of their inputs: q and k interleaved, prompts, every tile of the cache's attention")
    g = gen(17)
    rope, pos, w = A.Rope(table64(64, 128).float().cuda()), torch.arange(40, dtype=I32).cuda(), rand(g, 128).cuda()
    fused = rand(g, 40, 4, 3, 128).cuda()  # q, k and v of a head side by side
    q, k = fused[:, :, 0], fused[:, :, 1]
    before = fused.clone()
    want = [torch.empty(40, 4, 128, device="cuda") for _ in range(2)]
    A.qk_norm_rope(ctx, q, k, *want, q_weight=w, k_weight=w, rope=rope, positions=pos)
    A.qk_norm_rope(ctx, q, k, q, k, q_weight=w, k_weight=w, rope=rope, positions=pos)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(fused[:, :, 2], before[:, :, 2])
    with pytest.raises(s14.S14Error, match="shares memory"):
        A.qk_norm_rope(ctx, q, k, k, q)
    packed = rand(g, 300, 12 * 128, dtype=BF16).cuda()
    q, k, v = (packed[:, a * 128:b * 128].view(300, -1, 128) for a, b in ((0, 8), (8, 10), (10, 12)))
    for window in (0, 70):
        mine = packed.clone()
        mq, mk, mv = (mine[:, a * 128:b * 128].view(300, -1, 128) for a, b in ((0, 8), (8, 10), (10, 12)))
        out, _ = run_prompt(ctx, q, k, v, [170, 130], window)
        A.prompt_attention(ctx, mq, mk, mv, cumulative([170, 130]), mq, window=window)
        assert torch.equal(mq, out) and torch.equal(mine[:, 1024:], packed[:, 1024:])
    with pytest.raises(s14.S14Error, match="shares memory"):
        A.prompt_attention(ctx, q[:, :2], k, v, cumulative([170, 130]), v)
    for heads, kv, dim, new in EVERY_TILE:
        p = Paged(7, [700, 150], kv, dim, 32)
        q = rand(gen(4), 2 * new, heads, dim, dtype=BF16).cuda()
        out, _ = run_paged(ctx, p, q, [new, new], heads, dim)
        A.paged_attention(ctx, q, p.cache, p.dev_table, cumulative([new, new]), p.lens, q, max_new=new, max_len=700)
        assert torch.equal(q, out), (heads, kv, dim, new)


def test_operands_of_different_types(ctx):
    say("q f32 to bf16 beside k bf16 to f32; f32 keys with bf16 values")
    g = gen(41)
    q, k = rand(g, 33, 6, 128), rand(g, 33, 2, 128, dtype=BF16)
    w, table, pos = rand(g, 128), table64(64, 64).float(), torch.arange(33, dtype=I32)
    outs = torch.empty(33, 6, 128, dtype=BF16, device="cuda"), torch.empty(33, 2, 128, device="cuda")
    A.qk_norm_rope(ctx, q.cuda(), k.cuda(), *outs, k_weight=w.cuda(), rope=A.Rope(table.cuda()), positions=pos.cuda())
    for x, weight, got in ((q, None, outs[0]), (k, w, outs[1])):
        y, mag = norm_rope64(x, weight, 1e-6, table, pos, "half", 0)
        tol = 144 * 2.0 ** -24 * mag + (2.0 ** -8 * y.abs() if got.dtype == BF16 else 0) + 1e-30
        assert bool(((got.cpu().double() - y).abs() <= tol).all())
    k, v = rand(g, 50, 2, 64), rand(g, 50, 2, 64, dtype=BF16)
    a, b = (Paged(4, [50], 2, 64, 16) for _ in range(2))
    A.kv_append(ctx, a.cache, k.cuda(), v.cuda(), a.dev_table, ints([0, 50]), ints([0]))
    A.kv_append(ctx, b.cache, k.cuda(), v.float().cuda(), b.dev_table, ints([0, 50]), ints([0]))
    for t in ("k_pages", "v_pages", "k_scales", "v_scales"):
        assert torch.equal(getattr(a.cache, t), getattr(b.cache, t)), t


def test_two_contexts_at_once(ctx):
    """Each context has its own partial results and counters: their launches may overlap."""
    say("paged: two contexts on two streams, cut sequences, joined in the launch and after it")
    other = s14.Context(0)
    p = Paged(9, [9000, 4000], 8, 128, 64)
    for new in (1, 8):
        q = [rand(gen(s), 2 * new, 32, 128, dtype=BF16).cuda() for s in (4, 5)]
        want = [run_paged(ctx, p, x, [new, new], 32, 128)[0] for x in q]
        cu, streams = cumulative([new, new]), [torch.cuda.Stream() for _ in q]
        outs = [[torch.empty_like(x) for _ in range(20)] for x in q]
        torch.cuda.synchronize()
        for i in range(20):
            for c, s, x, o in zip((ctx, other), streams, q, outs):
                A.paged_attention(c, x, p.cache, p.dev_table, cu, p.lens, o[i], max_new=new, max_len=9000, stream=s.cuda_stream)
        torch.cuda.synchronize()
        for w, o in zip(want, outs):
            assert all(torch.equal(x, w) for x in o)
    other.destroy()


def test_most_sequences_of_a_call(ctx):
    """65,535 sequences, the last ones among them."""
    say("65,535 sequences: append, attention, prompts")
    n, kv, dim = 65535, 1, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v, q = (torch.randn(n, kv, dim, generator=g, device="cuda") for _ in range(3))
    cache = A.KvCache.empty(n, kv, 16, dim)
    table, cu = torch.randperm(n, generator=g, device="cuda").int()[:, None], torch.arange(n + 1, dtype=I32, device="cuda")
    zero, one = torch.zeros(n, dtype=I32, device="cuda"), torch.ones(n, dtype=I32, device="cuda")
    A.kv_append(ctx, cache, k, v, table.contiguous(), cu, zero, max_new=1)
    out = torch.full((n, kv, dim), 7.0, device="cuda")
    A.paged_attention(ctx, q.to(BF16), cache, table.contiguous(), cu, one, out, max_new=1, max_len=1)
    stored = cache.v_pages[table[:, 0].long(), :, :, 0].view(E4M3).double() * (cache.v_scales[table[:, 0].long()].double() - 127).exp2()[..., None]
    # One visible token: its own value.  Its weight is 2^r, r the rounding of its
    # score: below 2^-24 * 64 where |q| |k| / 8 * log2(e) is below 64.  As bf16 that is 1,
    # the sum of weights is 2^r itself, and two roundings of 2^-24 follow: 2^-17 in all.
    assert float((q.norm(dim=-1) * k.norm(dim=-1)).max()) / 8 * 1.4427 * 1.1 < 64
    assert bool(((out.double() - stored).abs() <= 2.0 ** -17 * stored.abs()).all())
    assert bool(((stored - v.double()).abs() <= v.abs().amax(-1, keepdim=True) * 2.0 ** -4).all())
    ctx.launch_status()
    vb = v.to(BF16)
    A.prompt_attention(ctx, q.to(BF16), k.to(BF16), vb, cu, out)
    assert bool(((out - vb.float()).abs() <= 2.0 ** -17 * vb.float().abs()).all())
    with pytest.raises(s14.S14Error, match="sequences"):
        A.prompt_attention(ctx, q.to(BF16), k.to(BF16), vb, torch.zeros(n + 2, dtype=I32, device="cuda"), out)


def test_refusals_of_tensors(ctx):
    say("tensors that the Python layer refuses")
    x = torch.empty(4, 2, 128, device="cuda")
    bad = [dict(q=x.cpu()), dict(q=x.half()), dict(q=x[:, :, ::2]), dict(q=x[0]), dict(q_out=x[:3]),
           dict(k=torch.empty(3, 2, 128, device="cuda"), k_out=torch.empty(3, 2, 128, device="cuda")),
           dict(q=torch.empty(4, 2, 96, device="cuda"), q_out=torch.empty(4, 2, 96, device="cuda")),
           dict(q_out=x[:, :1].expand(4, 2, 128)), dict(q_weight=torch.empty(127, device="cuda")),
           dict(q_weight=torch.empty(128, device="cuda", dtype=BF16)), dict(q_weight=torch.empty(128))]
    for kw in bad:
        with pytest.raises(s14.S14Error):
            args = dict(q=x, k=None, q_out=x, k_out=None, **{}) | kw
            A.qk_norm_rope(ctx, **args)
    rope = A.Rope(torch.empty(8, 128, device="cuda"))
    with pytest.raises(s14.S14Error):
        A.qk_norm_rope(ctx, x, None, x, None, rope=rope)  # no positions
    with pytest.raises(s14.S14Error):
        A.qk_norm_rope(ctx, x, None, x, None, rope=rope, positions=torch.empty(3, dtype=I32, device="cuda"))
    with pytest.raises(s14.S14Error):
        A.qk_norm_rope(ctx, x, None, x, None, rope=rope, positions=torch.empty(4, dtype=torch.int64, device="cuda"))
    p = Paged(9, [30], 2, 128, 64)
    q = torch.empty(1, 4, 128, dtype=BF16, device="cuda")
    cu, out = cumulative([1]), torch.empty_like(q)
    with pytest.raises(s14.S14Error):
        A.paged_attention(ctx, q.float(), p.cache, p.dev_table, cu, p.lens, out)
    with pytest.raises(s14.S14Error):
        A.paged_attention(ctx, q[:, :3], p.cache, p.dev_table, cu, p.lens, out[:, :3])
    with pytest.raises(s14.S14Error):
        A.paged_attention(ctx, q, p.cache, p.dev_table, cu[:1], p.lens, out)
    with pytest.raises(s14.S14Error):
        A.paged_attention(ctx, q, p.cache, p.dev_table, cu, p.lens, out, scale=math.nan)
    with pytest.raises(s14.S14Error):
        A.prompt_attention(ctx, q, q[:, :3], q[:, :3], cu, out)

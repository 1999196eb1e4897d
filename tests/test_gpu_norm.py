"""add_rms_norm against a plain 64-bit implementation.

Tolerances (f32: 2^-24, bf16: 2^-8): h = x + residual is one rounding.  Of y: the
sum of k squares of rounded values, in partial sums of at most 64 per thread and
then a tree, is off by (64 + 16 + 2) 2^-24 of itself at most, the root by half of
it, and the root's own approximation and three products by 2^-21; h's rounding
adds 2^-24 of the larger of |x| and |residual|.  A bf16 output adds its rounding.
The codes are those of s14_act_quant_e4m3 of the f32 y, bit for bit.
"""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

import test_gpu_attention as T  # noqa: E402
from test_gpu_attention import BF16, F32, U8, gen, rand, say  # noqa: E402

from colormlm_amd import attention as A  # noqa: E402
from colormlm_amd import s14  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    c = s14.Context(0)
    yield c
    torch.cuda.synchronize()
    c.destroy()


def norm64(x, residual, weight, eps):
    """h, y and the errors that each may have before an output's own rounding."""
    h = x.double() + (0 if residual is None else residual.double())
    r = (h.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    y = h * r * weight.double()
    size = torch.maximum(x.double().abs(), 0 * h if residual is None else residual.double().abs()) + h.abs()
    h_err = 0 * h if residual is None else 2.0 ** -24 * h.abs()
    return h, y, h_err, 2.0 ** -24 * (y.abs() * (41 + 8) + size * r * weight.double().abs())


def near(got, want, err, what):
    tol = err * (1 + 2.0 ** -10) + (2.0 ** -8 * want.abs() if got.dtype == BF16 else 2.0 ** -24 * want.abs()) + 1e-37
    bad = (got.cpu().double() - want).abs() > tol
    assert not bad.any(), (what, int(bad.sum()))


def codes_of(ctx, y, group):
    q, s = torch.empty(y.shape, dtype=U8, device="cuda"), torch.empty(y.shape[0], y.shape[1] // group, dtype=U8, device="cuda")
    s14.act_quant_e4m3(ctx, y.contiguous(), q, s, group=group)
    return q, s


SIZES = [(1, 4096, 128), (8, 4096, 32), (333, 1024, 128), (3, 7168, 64), (70, 64, 32), (5, 128, 128), (9, 1536, 64),
         (2, 20480, 128), (4, 8, 0), (3, 72, 0), (1, 65536, 128), (2, 33024, 32), (131, 2048, 128), (6, 8320, 64),
         (1, 16384, 128), (2, 4104, 0), (700, 1000, 0), (1500, 512, 128)]


@pytest.mark.parametrize("rows,k,group", SIZES)
@pytest.mark.parametrize("xt,rt,yt", [(F32, F32, F32), (BF16, F32, BF16), (F32, BF16, None), (BF16, None, F32), (F32, None, None),
                                      (BF16, BF16, BF16)])
def test_add_rms_norm(ctx, rows, k, group, xt, rt, yt):
    if not group and yt is None:
        yt = F32
    say(f"add_rms_norm rows={rows} k={k} group={group} x={xt} residual={rt} y={yt}")
    g = gen(rows + k)
    x = rand(g, rows, k, dtype=xt)
    residual = (5 * rand(g, rows, k) * (1 + 30 * (torch.rand(k, generator=g) < 0.02))).to(rt) if rt else None
    weight = rand(g, k)
    h, y, h_err, y_err = norm64(x, residual, weight, 1e-5)
    outs = {"y": torch.empty(rows, k, dtype=yt, device="cuda") if yt else None}
    if rt:
        outs["residual_out"] = torch.empty(rows, k, dtype=rt, device="cuda")
    if group:
        outs["q"] = torch.empty(rows, k, dtype=U8, device="cuda")
        outs["scales"] = torch.empty(rows, k // group, dtype=U8, device="cuda")
    dev = [t if t is None else t.cuda() for t in (x, residual)]
    A.add_rms_norm(ctx, dev[0], weight.cuda(), residual=dev[1], eps=1e-5, **outs)
    torch.cuda.synchronize()
    if yt:
        near(outs["y"], y, y_err, "y")
    if rt:
        near(outs["residual_out"], h, h_err, "h")
    if group:
        full = torch.empty(rows, k, device="cuda")
        A.add_rms_norm(ctx, dev[0], weight.cuda(), residual=dev[1], eps=1e-5, y=full)
        near(full, y, y_err, "f32 y")
        q, s = codes_of(ctx, full, group)
        assert torch.equal(outs["q"], q) and torch.equal(outs["scales"], s)
    ctx.launch_status()


def test_strides_places_and_rows_behind(ctx):
    say("add_rms_norm on slices, in its inputs' places, bytes around left alone")
    g = gen(3)
    for k, t in ((512, F32), (512, BF16), (4096, F32), (12288, BF16)):
        wide, res = rand(g, 11, k + 24, dtype=t).cuda(), rand(g, 11, k + 8, dtype=t).cuda()
        w = rand(g, k)
        x, r = wide[:9, 8:k + 8], res[1:10, :k]
        h, y, h_err, y_err = norm64(x.cpu(), r.cpu(), w, 1e-6)
        before, before_r = wide.clone(), res.clone()
        A.add_rms_norm(ctx, x, w.cuda(), residual=r, residual_out=r, y=x)
        torch.cuda.synchronize()
        near(x, y, y_err, "y in x's place")
        near(r, h, h_err, "h in the residual's")
        before[:9, 8:k + 8], before_r[1:10, :k] = x, r
        assert torch.equal(wide, before) and torch.equal(res, before_r)
        x.copy_(rand(g, 9, k))
        h, y, h_err, y_err = norm64(x.cpu(), None, w, 1e-6)
        out = torch.full((9, 2 * k), 7.0, device="cuda")
        A.add_rms_norm(ctx, x, w.cuda(), residual_out=out[:, k:], y=out[:, :k])
        near(out[:, :k], y, y_err, "y, no residual")
        assert torch.equal(out[:, k:], x.float())
    A.add_rms_norm(ctx, x[:0], w.cuda(), y=out[:0, :k])
    q = torch.full((5, 256), 9, dtype=U8, device="cuda")
    s = torch.full((5, 2), 9, dtype=U8, device="cuda")
    A.add_rms_norm(ctx, rand(g, 3, 256).cuda(), torch.ones(256, device="cuda"), q=q[1:4], scales=s[1:4])
    torch.cuda.synchronize()
    for t in (q, s):
        assert bool((t[0] == 9).all()) and bool((t[4] == 9).all()) and not bool((t[1:4] == 9).all())


def test_special_values(ctx):
    say("add_rms_norm: NaN and infinite values stay in their rows, zero rows are zero, eps 0")
    x = rand(gen(1), 6, 1024)
    x[1, 700], x[2, 3] = math.nan, math.inf
    x[3] = 0.0
    x[4] = 1e-30 * x[4]
    w = torch.ones(1024)
    y, q, s = torch.empty(6, 1024, device="cuda"), torch.empty(6, 1024, dtype=U8, device="cuda"), torch.empty(6, 8, dtype=U8, device="cuda")
    A.add_rms_norm(ctx, x.cuda(), w.cuda(), y=y, q=q, scales=s)
    assert y[1].isnan().all() and not y[3].any() and y[0].isfinite().all() and y[4:].isfinite().all()
    assert bool(y[2, 3].isnan()) and not torch.cat([y[2, :3], y[2, 4:]]).any()  # inf * 0, and finite values * 0
    want = codes_of(ctx, y, 128)
    assert torch.equal(q, want[0]) and torch.equal(s, want[1])
    _, ref, _, err = norm64(x[[0, 4, 5]], None, w, 1e-6)
    near(y[[0, 4, 5]], ref, err, "rows beside")
    A.add_rms_norm(ctx, x[:1].cuda(), w.cuda(), eps=0.0, y=y[:1])
    _, ref, _, err = norm64(x[:1], None, w, 0.0)
    near(y[:1], ref, err, "eps 0")


def test_streams_capture_and_repeats(ctx):
    say("add_rms_norm on another stream and replayed from a graph, between eager calls")
    g = gen(9)
    x, r, w = rand(g, 40, 4096).cuda(), rand(g, 40, 4096).cuda(), rand(g, 4096).cuda()
    q, s = torch.empty(40, 4096, dtype=U8, device="cuda"), torch.empty(40, 32, dtype=U8, device="cuda")
    ro, y = torch.empty_like(x), torch.empty(40, 4096, dtype=BF16, device="cuda")
    run = lambda **kw: A.add_rms_norm(ctx, x, w, residual=r, residual_out=ro, y=y, q=q, scales=s, **kw)  # noqa: E731
    run()
    torch.cuda.synchronize()
    first = [t.clone() for t in (q, s, ro, y)]
    side = torch.cuda.Stream()
    for t in (q, s, ro, y):
        t.zero_()
    torch.cuda.synchronize()
    run(stream=side.cuda_stream)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, (q, s, ro, y)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        run()
    for _ in range(4):
        x.copy_(rand(g, 40, 4096))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (q, s, ro, y)]
        run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (q, s, ro, y)))


def test_the_codes_feed_the_projection(ctx):
    """fp8_linear of the codes against 64 bits of the codes' own values."""
    g = gen(4)
    m, k, n = 5, 1024, 256
    x, w = rand(g, m, k).cuda(), rand(g, k).cuda()
    q, s = torch.empty(m, k, dtype=U8, device="cuda"), torch.empty(m, k // 128, dtype=U8, device="cuda")
    A.add_rms_norm(ctx, x, w, q=q, scales=s)
    weight = T.quantized(g, n, k).cuda()
    ws = torch.randint(115, 120, (n // 128, k // 128), generator=g, dtype=U8).cuda()
    y = torch.empty(m, n, device="cuda")
    s14.fp8_linear(ctx, q, s, weight, ws, y)
    val = lambda c, sc: c.cpu().view(T.E4M3).double() * (sc.cpu().double() - 127).exp2()  # noqa: E731
    a = val(q, s.repeat_interleave(128, 1))
    b = val(weight, ws.repeat_interleave(128, 0).repeat_interleave(128, 1))
    assert bool(((y.cpu().double() - a @ b.T).abs() <= (k + 8) * 2.0 ** -24 * (a.abs() @ b.abs().T)).all())

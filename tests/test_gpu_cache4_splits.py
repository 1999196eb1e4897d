"""Attention over the paged 4-bit cache where the way its work is split could
show: values that are NaN under weights too small for a number, chunks that the
device sets by the sequences' lengths, and captured calls of those.  Against
plain 64-bit implementations, with the tolerances of the cache's other tests."""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

import test_gpu_attention as T  # noqa: E402
from test_attention_balance import BALANCED  # noqa: E402
from test_gpu_attention import BF16, F32, U8, check_attention, gen, rand, run_paged, say  # noqa: E402
from test_gpu_cache4 import Layer, Paged4, ctx  # noqa: E402, F401

from colormlm_amd import attention as A  # noqa: E402

pytestmark = pytest.mark.gpu

# ---------------------------------------------------------------------------
# NaN values
# ---------------------------------------------------------------------------

# heads, key heads, head size, new tokens: every kernel, with one and two 16-row
# tiles a wavefront or workgroup, and rows that share tokens
TILES = [(4, 1, 64, 1), (4, 1, 64, 7), (8, 1, 64, 8), (8, 1, 64, 40), (4, 1, 128, 1), (4, 1, 128, 8), (8, 1, 128, 3),
         (4, 1, 128, 12), (4, 1, 128, 30), (4, 1, 256, 2), (2, 1, 256, 11), (2, 1, 256, 32), (16, 1, 512, 1), (16, 1, 512, 2)]


def loud_token(p, i, j, q):
    """Key of position j of sequence i along q's signs, as far as E2M1 goes: its
    scores pass every other key's by hundreds."""
    page, slot = p.place(i, j)
    codes = torch.where(q < 0, 15, 7).to(U8)
    p.k[page, :, slot] = codes[0::2] | codes[1::2] << 4
    p.set_scale(0, i, j, 127)


@pytest.mark.parametrize("heads,kv,dim,new", TILES)
@pytest.mark.parametrize("loud,nan", [(900, 40), (40, 900), (701, 700), (700, 701), (130, 70), (70, 130), (1990, 0), (2, 1930)])
def test_nan_values_whatever_their_weight(ctx, heads, kv, dim, new, loud, nan):  # noqa: F811
    """A row that sees a NaN block of a value has its dimensions NaN and no
    others, though a key before, behind, in the same step or in another chunk
    leaves it a weight of exp(-100) and less; a row that does not see it has none."""
    say(f"paged4 NaN value at {nan}, loud key at {loud}, heads={heads}/{kv} dim={dim} new={new}")
    g = gen(dim + new)
    q = (rand(g, dim).sign() + 0.05 * rand(g, 2 * new, heads, dim)).to(BF16)
    base = q.float().mean((0, 1))
    p = Paged4(dim + new, [2000, 1000], kv, dim, 64, lo=123, hi=126)
    loud_token(p, 0, loud, base)
    last = (dim // 128 or 1) - 1
    p.set_scale(1, 0, nan, 255, last)
    p.upload()
    scale = 64.0 / dim
    window = 1900 if (loud, nan) == (1990, 0) else 0  # what lies before a window is not seen: no row has the NaN
    k, v = p.rows(0)
    s = (q[:new].double().flatten(0, 1) @ k[:, 0].T) * scale
    assert bool((s[:, loud] - s[:, nan] > 100 + 2 * math.log(2) * 8).all())
    want = [torch.cat(x) for x in zip(*(T.attention64(q[at:at + new], *p.rows(i), scale, window) for i, at in ((0, 0), (1, new))))]
    seen = bool(want[0].isnan().any())
    assert seen == (window == 0)
    if seen:
        assert bool(want[0][:new, :, -min(dim, 128):].isnan().all())
    for max_len in (2000, 1, 1 << 20):
        out, lse = run_paged(ctx, p, q.cuda(), [new, new], heads, dim, window, F32, max_len=max_len, scale=scale)
        check_attention(out, lse, want, f"max_len {max_len}")
    # one sequence: other kernels up to 32 rows
    p.lens, p.dev_table = p.lens[:1], p.dev_table[:1].contiguous()
    for max_len in (2000, 1):
        out, lse = run_paged(ctx, p, q[:new].cuda(), [new], heads, dim, window, F32, max_len=max_len, scale=scale)
        check_attention(out, lse, [x[:new] for x in want], f"alone, max_len {max_len}")
    ctx.launch_status()


@pytest.mark.parametrize("heads,kv,dim,new", TILES)
@pytest.mark.parametrize("loud,nan", [(900, 40), (40, 900), (700, 701)])
def test_nan_keys_whatever_the_other_scores(ctx, heads, kv, dim, new, loud, nan):  # noqa: F811
    say(f"paged4 NaN key at {nan}, loud key at {loud}, heads={heads}/{kv} dim={dim} new={new}")
    g = gen(dim + new)
    q = (rand(g, dim).sign() + 0.05 * rand(g, 2 * new, heads, dim)).to(BF16)
    p = Paged4(dim + new, [2000, 1000], kv, dim, 64, lo=123, hi=126)
    loud_token(p, 0, loud, q.float().mean((0, 1)))
    p.set_scale(0, 0, nan, 255, 0)
    p.upload()
    for max_len in (2000, 1):
        out, lse = run_paged(ctx, p, q.cuda(), [new, new], heads, dim, 0, F32, max_len=max_len, scale=64.0 / dim)
        assert bool(out[:new].isnan().all()) and bool(lse[:new].isnan().all())
        assert bool(out[new:].isfinite().all()) and bool(lse[new:].isfinite().all())
    p.lens, p.dev_table = p.lens[:1], p.dev_table[:1].contiguous()
    out, lse = run_paged(ctx, p, q[:new].cuda(), [new], heads, dim, 0, F32, scale=64.0 / dim)
    assert bool(out.isnan().all()) and bool(lse.isnan().all())
    ctx.launch_status()


# ---------------------------------------------------------------------------
# chunks by the lengths
# ---------------------------------------------------------------------------


def ragged(seed, seqs, new, most):
    """Lengths with one past the promise, empty sequences, and short ones."""
    g = gen(seed)
    lengths = [int(x) for x in torch.randint(new, max(new + 1, most // 4), (seqs,), generator=g)]
    lengths[0], lengths[-1] = most + 700, most
    if seqs > 2:
        lengths[1] = 0
    return lengths


def check_some(p, q, out, lse, counts, window, what):
    """First and last rows of the first, the last and two other sequences, all heads' first and last."""
    at, seqs = [0], len(counts)
    for n in counts:
        at.append(at[-1] + n)
    for i in {0, 1, seqs // 2, seqs - 1}:
        if not counts[i]:
            continue
        k, v = p.rows(i)
        heads = q.shape[1]
        for row in {0, counts[i] - 1}:
            end = len(k) - counts[i] + row + 1
            kv = k.shape[1]
            group = heads // kv
            pick = [0, heads - 1]
            t = at[i] + row
            parts = [T.attention64(q[t:t + 1, h:h + 1].cpu(), k[:max(end, 0), h // group:h // group + 1], v[:max(end, 0), h // group:h // group + 1],
                                   q.shape[-1] ** -0.5, window) for h in pick]
            want = [torch.cat(x, 1) for x in zip(*parts)]
            check_attention(out[t:t + 1, pick], lse[t:t + 1, pick], want, f"{what}, sequence {i} row {row}")


@pytest.mark.parametrize("seqs,heads,kv,dim,new,most", BALANCED)
@pytest.mark.parametrize("window", [0, 900])
def test_balanced_launches(ctx, seqs, heads, kv, dim, new, most, window):  # noqa: F811
    """Chunks by what the sequences hold in all, one sequence longer than promised,
    one without tokens and one without rows; and, one sequence more than the lengths
    are added up of, by the promise."""
    say(f"paged4 balanced: {seqs} sequences heads={heads}/{kv} dim={dim} new={new} window={window}")
    for more in ((0, 1) if seqs == 256 else (0,)):
        lengths = ragged(seqs, seqs + more, new, most)
        counts = [new] * (seqs + more)
        counts[seqs // 2] = 0
        p = Paged4(seqs, lengths, kv, dim, 64)
        q = rand(gen(4), sum(counts), heads, dim, dtype=BF16).cuda()
        out, lse = run_paged(ctx, p, q, counts, heads, dim, window, F32, max_len=most)
        again, _ = run_paged(ctx, p, q, counts, heads, dim, window, F32, max_len=most)
        assert torch.equal(out, again)
        check_some(p, q, out, lse, counts, window, "balanced")
    ctx.launch_status()


@pytest.mark.parametrize("seqs,heads,kv,dim,new,most", BALANCED)
def test_balanced_launches_captured_and_replayed(ctx, seqs, heads, kv, dim, new, most):  # noqa: F811
    """A captured launch, replayed with other lengths: the chunk, which the join takes
    from the workspace, is another one each time.  Eager launches of the same context
    lie between the replays; each replay equals an eager call bit for bit."""
    say(f"paged4 balanced and captured: {seqs} sequences heads={heads}/{kv} dim={dim} new={new}")
    counts = [new] * seqs
    full = [most] * seqs
    p = Paged4(seqs, full, kv, dim, 64)
    q = rand(gen(4), sum(counts), heads, dim, dtype=BF16).cuda()
    out, lse = torch.zeros(q.shape, device="cuda"), torch.zeros(q.shape[:2], device="cuda")
    cu = T.cumulative(counts)
    call = lambda o, l: A.paged_attention(ctx, q, p.cache, p.dev_table, cu, p.lens, o, lse=l, max_new=new, max_len=most)  # noqa: E731
    call(out, lse)
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        call(out, lse)
    rows = p.rows
    for step, lengths in enumerate((full, [new] * seqs, ragged(3, seqs, new, most - 700), [max(new, most // 8)] * seqs, full)):
        p.lens.copy_(torch.tensor(lengths, dtype=torch.int32))
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        eager, eager_lse = torch.zeros_like(out), torch.zeros_like(lse)
        call(eager, eager_lse)
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(lse, eager_lse), step
        p.rows = lambda i: rows(i, lengths[i])  # noqa: B023
        check_some(p, q, out, lse, counts, 0, f"replay {step}")
    ctx.launch_status()


def test_layer_replays_leave_the_same_cache(ctx):  # noqa: F811
    """A captured layer step replayed from step to step against an eager one: every
    byte of the cache, key scales too, as the tokens cross blocks of slots and pages."""
    say("graph capture of a layer's step, all of the cache's bytes")
    g = gen(23)
    L, E = Layer(ctx, 2), Layer(ctx, 2)
    x, cu = torch.empty(2, L.hidden, device="cuda"), T.cumulative([1, 1])
    past, lens, pos = (T.ints([0, 0]) for _ in range(3))
    tensors = lambda c: (c.k_pages, c.v_pages, c.k_scales, c.v_scales)  # noqa: E731
    for a, b in zip(tensors(L.cache), tensors(E.cache)):
        a.copy_(torch.randint(0, 120, a.shape, generator=g, dtype=U8))
        b.copy_(a)
    x.copy_(rand(g, 2, L.hidden))
    L.step(x, cu, past, T.ints([1, 1]), pos, 1)  # warm
    E.step(x, cu, past, T.ints([1, 1]), pos, 1)
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        L.step(x, cu, past, lens, pos, 1)
    for step, at in enumerate(([1, 1], [63, 2], [64, 150], [197, 65], [198, 66])):
        x.copy_(rand(g, 2, L.hidden))
        for t, v in ((past, at), (lens, [n + 1 for n in at]), (pos, at)):
            t.copy_(torch.tensor(v, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        E.step(x, cu, past, lens, pos, 1)
        torch.cuda.synchronize()
        for a, b in zip((L.out, L.y2, L.h, *tensors(L.cache)), (E.out, E.y2, E.h, *tensors(E.cache))):
            assert torch.equal(a, b), step
    ctx.launch_status()

"""Performance cases of the operators around the FP8 projections that keep less
in memory: the residual norm that writes the projections' 8-bit rows, and the
paged key/value cache in 4 bits with the attention that reads it.

Three kinds of call (colormlm_amd.attention):

  add_norm  residual addition, root-mean-square norm and the E4M3 rows with
            E8M0 scales that fp8_linear takes, in one pass over the rows
  append4   keys and values of new tokens into the paged 4-bit cache (E2M1
            codes, E8M0 scales of 32 dimensions of a key and of 128 of a value),
            the keys' norm and rotation on the way
  paged4    attention of the new tokens over that cache: decode, speculative
            verify, a prompt's later chunks

Row lengths: 4,096 (the package's hidden size), 1,024 (its query rank) and
generic ones.  Head layouts: 32 query heads over 8 key heads of 128 and 64 over
8 of 64, the generic ones at hidden size 4,096, and 64 query heads over one key
head of 512, the layout of the package's own projections (wq_b [32768, 1024],
wkv [512, 4096]).  Rows are N(0, 1), cached codes those of N(0, 1) values, pages
lie in the cache in random order, sequence lengths are log-uniform.  Every
input is drawn from the seed.
"""

from __future__ import annotations

import functools
import math
import random

import torch

own = False

EPS = 1e-6
THETA = 10000.0
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # decode of one token: the hidden state before a projection, where the launch is what counts
        {"name": "add_norm_1", "op": "add_norm", "rows": 1, "k": 4096, "x": "f32", "residual": "f32", "y": "", "group": 128},
        # a verify block before the experts: the router and the expert layer take the f32 rows
        {"name": "add_norm_8_experts", "op": "add_norm", "rows": 8, "k": 4096, "x": "f32", "residual": "f32", "y": "f32",
         "group": 0},
        # an odd number of the query rank's rows, which carry no residual
        {"name": "add_norm_333_rank", "op": "add_norm", "rows": 333, "k": 1024, "x": "f32", "residual": "", "y": "",
         "group": 128},
        # a long prompt with its residual stream in 16 bits
        {"name": "add_norm_16384", "op": "add_norm", "rows": 16384, "k": 4096, "x": "f32", "residual": "bf16", "y": "",
         "group": 128},
        # one speculative-verify block of one sequence, one wide key head
        {"name": "append4_verify_8", "op": "append4", "seqs": 1, "new": 8, "ragged": False, "past": 299, "kv": 1,
         "dim": 512, "page": 64, "rot": 64, "layout": "interleaved", "norm": True, "dtype": "f32", "spread": 1},
        # one decode step of a batch of young sequences
        {"name": "append4_decode_96", "op": "append4", "seqs": 96, "new": 1, "ragged": False, "past": 30, "kv": 8,
         "dim": 128, "page": 16, "rot": 128, "layout": "half", "norm": True, "dtype": "f32", "spread": 2},
        # packed prompts whose keys are rotated already
        {"name": "append4_prompts", "op": "append4", "seqs": 21, "new": 4000, "ragged": True, "past": 100, "kv": 8,
         "dim": 128, "page": 64, "rot": 0, "layout": "half", "norm": False, "dtype": "bf16", "spread": 3},
        # decode of one sequence of an odd length: few rows, a long axis
        {"name": "paged4_1_4097", "op": "paged4", "seqs": 1, "new": 1, "ragged": False, "len": 4097, "same": True,
         "heads": 32, "kv": 8, "dim": 128, "page": 64, "window": 0, "lse": False, "spread": 4},
        # a speculative-verify block at a long context
        {"name": "paged4_verify8_40000", "op": "paged4", "seqs": 1, "new": 8, "ragged": False, "len": 40000, "same": True,
         "heads": 32, "kv": 8, "dim": 128, "page": 64, "window": 0, "lse": True, "spread": 5},
        # one decode step of a batch of ragged lengths
        {"name": "paged4_decode_128", "op": "paged4", "seqs": 128, "new": 1, "ragged": False, "len": 8192, "same": False,
         "heads": 32, "kv": 8, "dim": 128, "page": 64, "window": 0, "lse": False, "spread": 6},
        # 64 query heads over one wide key head: matrix work, not bytes
        {"name": "paged4_wide_4x9000", "op": "paged4", "seqs": 4, "new": 4, "ragged": False, "len": 9000, "same": False,
         "heads": 64, "kv": 1, "dim": 512, "page": 64, "window": 0, "lse": False, "spread": 7},
        # the next chunk of several prompts
        {"name": "paged4_chunk_8x64", "op": "paged4", "seqs": 8, "new": 64, "ragged": False, "len": 3000, "same": True,
         "heads": 32, "kv": 8, "dim": 128, "page": 64, "window": 0, "lse": False, "spread": 8},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


LAYOUTS = [(32, 8, 128), (32, 8, 128), (64, 8, 64), (32, 4, 128), (16, 16, 64), (64, 1, 512), (12, 2, 256)]


def draw(rng):
    op = rng.choice(["add_norm", "append4", "paged4", "paged4"])
    if op == "add_norm":
        group = rng.choice([0, 32, 64, 128, 128])
        k = group * _log_int(rng, max(1, 512 // group), 16384 // group) if group else 8 * _log_int(rng, 8, 2048)
        return {"op": op, "rows": min(_log_int(rng, 1, 16384), 64_000_000 // k), "k": k, "x": rng.choice(["f32", "bf16"]),
                "residual": rng.choice(["", "f32", "bf16"]), "y": rng.choice(["", "f32", "bf16"]) if group else "bf16",
                "group": group}
    heads, kv, dim = rng.choice(LAYOUTS)
    spread = rng.randint(10, 1 << 20)
    page = rng.choice([16, 32, 64, 64, 128])
    if op == "append4":
        rot, layout = rng.choice([(dim, "half"), (dim // 2, "half"), (32, "interleaved"), (64, "interleaved")])
        seqs = _log_int(rng, 1, 128)
        new = _log_int(rng, 1, max(8, min(4000, 24000000 // (seqs * kv * dim))))
        return {"op": op, "seqs": seqs, "new": new, "ragged": rng.random() < 0.6, "past": _log_int(rng, 1, 300), "kv": kv,
                "dim": dim, "page": page, "rot": rng.choice([0, rot]), "layout": layout, "norm": rng.random() < 0.7,
                "dtype": rng.choice(["f32", "bf16"]), "spread": spread}
    seqs = _log_int(rng, 1, 100)
    length = _log_int(rng, 20, max(40, min(60000, 300_000_000 // (seqs * kv * dim * 2))))
    new = rng.choice([1, 1, 2, 4, 8, 8, _log_int(rng, 9, 64)]) if heads // kv <= 8 else rng.choice([1, 2, 4])
    return {"op": op, "seqs": seqs, "new": min(new, length), "ragged": rng.random() < 0.3, "len": length,
            "same": rng.random() < 0.3, "heads": heads, "kv": kv, "dim": dim, "page": page,
            "window": rng.choice([0, 0, 0, _log_int(rng, 16, 2048)]), "lse": rng.random() < 0.5, "spread": spread}


# ---------------------------------------------------------------------------
# the sizes of a case
# ---------------------------------------------------------------------------


def _ragged(case, n, top, salt, low=1):
    """n lengths, log-uniform in [low, top], the first one top itself."""
    rng = random.Random(case["spread"] * 31 + salt)
    return [top] + [_log_int(rng, low, top) for _ in range(n - 1)]


def _lengths(case):
    """new, past (append4) or len (paged4) of each sequence."""
    n = case["seqs"]
    new = _ragged(case, n, case["new"], 1) if case["ragged"] else [case["new"]] * n
    if case["op"] == "append4":
        return new, _ragged(case, n, case["past"], 2)
    length = [case["len"]] * n if case["same"] else _ragged(case, n, case["len"], 3, 1 + case["len"] // 16)
    return [min(a, b) for a, b in zip(new, length)], length


def _parts(dim):
    """Value scales of a token and head: one for each 128 dimensions."""
    return max(1, dim // 128)


def _token_bytes(dim):
    """What the cache holds of a token and key head."""
    return dim + dim // 32 + _parts(dim)


def _visible(new, length, window):
    """Pairs (query, key) that a sequence's new tokens at the end of `length` see."""
    first, last = length - new + 1, length
    if not window:
        return (first + last) * new // 2
    return sum(min(window, p) for p in range(first, last + 1))


def work(case):
    size = {"f32": 4, "bf16": 2, "": 0}
    if case["op"] == "add_norm":
        values = case["rows"] * case["k"]
        each = size[case["x"]] + 2 * size[case["residual"]] + size[case["y"]]
        codes = values + values // case["group"] if case["group"] else 0
        return {"bytes": values * each + codes + 4 * case["k"], "flops": 8 * values}
    dim, kv = case["dim"], case["kv"]
    new, length = _lengths(case)
    if case["op"] == "append4":
        values = 2 * sum(new) * kv * dim
        return {"bytes": values * size[case["dtype"]] + sum(new) * kv * _token_bytes(dim) + 4 * sum(new) * case["rot"],
                "flops": 8 * values}
    rows = sum(new) * case["heads"] * dim * 2 * 2
    read = [min(b, case["window"] + a - 1) if case["window"] else b for a, b in zip(new, length)]
    cache = sum(read) * kv * _token_bytes(dim) + sum(-(-b // case["page"]) for b in read) * 4
    pairs = sum(_visible(a, b, case["window"]) for a, b in zip(new, length))
    return {"bytes": rows + cache + (4 * sum(new) * case["heads"] if case["lse"] else 0),
            "flops": 4 * pairs * case["heads"] * dim}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + 17)
    return g


def _randn(g, *shape, dtype="f32"):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(DTYPES[dtype])


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cumulative(lengths):
    total = [0]
    for n in lengths:
        total.append(total[-1] + n)
    return _ints(total)


@functools.lru_cache(maxsize=4)
def _table(positions, rot):
    """cos | sin of each position, f32 from angles in 64 bits."""
    inv = THETA ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.cat([angle.cos(), angle.sin()], 1).float()


E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


@functools.lru_cache(maxsize=1)
def _normal_byte():
    """Two codes of normal values for each number below 2^16."""
    at = (torch.arange(256, dtype=torch.float64, device="cuda") + 0.5) / 256
    x = 1.8 * math.sqrt(2.0) * torch.erfinv(2.0 * at - 1.0)
    edge = torch.tensor([(a + b) / 2 for a, b in zip(E2M1, E2M1[1:])], dtype=torch.float64, device="cuda")
    code = torch.bucketize(x.abs(), edge) + 8 * (x < 0)
    return (code[:, None] * 16 + code).flatten().to(torch.uint8)


def _codes(g, *shape):
    """Bytes of two E2M1 codes of normal values."""
    out = torch.empty(shape, dtype=torch.uint8, device="cuda")
    table = _normal_byte()
    for part in out.view(shape[0], -1).split(max(1, (1 << 27) // max(1, out[0].numel()))):
        part.copy_(table[torch.randint(0, 1 << 16, part.shape, generator=g, device="cuda", dtype=torch.int32)])
    return out


def _cache(g, pages, case):
    kv, page, dim = case["kv"], case["page"], case["dim"]
    scale = lambda n: torch.randint(125, 128, (pages, kv, n, page), generator=g, device="cuda", dtype=torch.uint8)  # noqa: E731
    return {"k_pages": _codes(g, pages, kv, page, dim // 2), "k_scales": scale(dim // 32),
            "v_pages": _codes(g, pages, kv, dim // 32, page // 16, 16, 16), "v_scales": scale(_parts(dim))}


def _page_table(g, lengths, page):
    """Each sequence's pages, in random places of the cache; entries past its
    last page are 0 and not read.  Also the pages in all."""
    need = [-(-n // page) for n in lengths]
    order = torch.randperm(sum(need), generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((len(need), max(need)), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, at


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    s = {"case": case}
    if op == "add_norm":
        rows, k = case["rows"], case["k"]
        s["x"] = _randn(g, rows, k, dtype=case["x"])
        # a residual stream is wider than what is added to it, and some of its dimensions much wider
        wide = 1.0 + 30.0 * (torch.rand(k, generator=g, device="cuda") < 0.01)
        s["residual"] = (3.0 * wide * _randn(g, rows, k)).to(DTYPES[case["residual"]]) if case["residual"] else None
        s["weight"] = 1.0 + 0.1 * _randn(g, k)
        return s
    kv, dim = case["kv"], case["dim"]
    new, length = _lengths(case)
    s["cu"], s["total"], s["most"] = _cumulative(new), sum(new), max(new)
    if op == "append4":
        past, length = length, [a + b for a, b in zip(new, length)]
        s["past"] = _ints(past)
        s["k"] = _randn(g, s["total"], kv, dim, dtype=case["dtype"])
        s["v"] = _randn(g, s["total"], kv, dim, dtype=case["dtype"])
        s["k_weight"] = 1.0 + 0.1 * _randn(g, dim) if case["norm"] else None
        s["table"] = _table(8192, case["rot"]) if case["rot"] else None
    else:
        s["q"] = _randn(g, s["total"], case["heads"], dim, dtype="bf16")
        s["longest"], s["lengths"] = max(length), _ints(length)
    s["pages"], n = _page_table(g, length, case["page"])
    s.update(_cache(g, n, case))
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------


def _power(code):
    """2^(code - 127) in f32, code 1 to 254."""
    return (code.int() << 23).view(torch.float32)


@functools.lru_cache(maxsize=2)
def _pairs(dtype):
    """The two values of each byte of codes, the low half's first."""
    v = torch.tensor(E2M1 + tuple(-x for x in E2M1), device="cuda")
    byte = torch.arange(256, device="cuda")
    return torch.stack([v[byte % 16], v[byte // 16]], 1).to(dtype)


def _plain_add_norm(s):
    case = s["case"]
    rows, k = s["x"].shape
    x = s["x"].float()
    outs = []
    if s["residual"] is not None:
        x = x + s["residual"].float()
        outs.append(x.to(s["residual"].dtype))
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s["weight"]
    if case["y"]:
        outs.append(y.to(DTYPES[case["y"]]))
    if case["group"]:
        part = y.view(rows, k // case["group"], case["group"])
        bits = (part.abs().amax(-1).clamp(min=1e-4) / 448.0).view(torch.int32)
        code = (bits >> 23) + ((bits & 0x7FFFFF) != 0).int()
        q = (part / _power(code)[..., None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
        outs += [q.view(rows, k), code.to(torch.uint8).view(torch.float8_e8m0fnu)]
    return outs


def _rotate(x, c, s, layout, start):
    """x [..., dim] with dimensions start .. start + rot rotated, c and s [tokens, 1, rot / 2]."""
    half = c.shape[-1]
    part = x[..., start:start + 2 * half]
    if layout == "half":
        a, b = part[..., :half], part[..., half:]
        part = torch.cat([a * c - b * s, b * c + a * s], -1)
    else:
        a, b = part[..., 0::2], part[..., 1::2]
        part = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    return torch.cat([x[..., :start], part, x[..., start + 2 * half:]], -1)


def _key_rows(s, positions):
    """The new keys in f32, normed and rotated."""
    case, x = s["case"], s["k"].float()
    if s["k_weight"] is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s["k_weight"]
    if s["table"] is not None:
        c, sn = s["table"][positions][:, None].chunk(2, -1)
        x = _rotate(x, c, sn, case["layout"], case["dim"] - case["rot"])
    return x


def _quantise(x, block):
    """x [tokens, kv, dim]: codes of the same shape, and scales [tokens, kv, dim / block]."""
    part = x.unflatten(-1, (-1, block))
    bits = part.abs().amax(-1).view(torch.int32)
    scale = ((bits >> 23) - 2 + ((bits & 0x7FFFFF) > 0x400000).int()).clamp(27, 227)
    a = part.abs() / _power(scale)[..., None]
    # round to nearest, ties to the even code
    code = (a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    return (code + 8 * (part < 0)).flatten(-2).to(torch.uint8), scale.to(torch.uint8)


def _place(s):
    """Page and slot of each new token, its position and its sequence."""
    case, cu, past = s["case"], s["cu"].long(), s["past"].long()
    row = torch.arange(s["total"], device="cuda")
    seq = torch.searchsorted(cu, row, right=True) - 1
    pos = past[seq] + row - cu[seq]
    return s["pages"].long()[seq, pos // case["page"]], pos % case["page"], pos, seq


def _scale_slot(slot):
    """Where a slot's key scale lies: the 4 x 4 slots of each 16 transposed."""
    return slot // 16 * 16 + slot % 4 * 4 + slot % 16 // 4


def _plain_append(s):
    case = s["case"]
    page, slot, pos, seq = _place(s)
    codes, scale = _quantise(_key_rows(s, pos), 32)
    s["k_pages"][page, :, slot] = codes[..., 0::2] | (codes[..., 1::2] << 4)
    s["k_scales"][page, :, :, _scale_slot(slot)] = scale
    codes, scale = _quantise(s["v"].float(), case["dim"] // _parts(case["dim"]))
    s["v_scales"][page, :, :, slot] = scale
    # a byte holds two slots: the other one's code is a new token's too, or what lies there
    codes = codes.unflatten(-1, (-1, 2, 16)).transpose(-1, -2)
    odd = slot % 2
    other = (torch.arange(s["total"], device="cuda") + 1 - 2 * odd).clamp(0, s["total"] - 1)
    at = (page, slice(None), slice(None), slot // 16, slice(None), slice(None), slot % 16 // 2)
    byte = s["v_pages"].unflatten(-1, (2, 8))
    wide = lambda x: x.view(-1, 1, 1, 1, 1)  # noqa: E731
    new = wide((seq[other] == seq) & (slot[other] // 2 == slot // 2) & (other != torch.arange(s["total"], device="cuda")))
    old = byte[at]
    neighbour = torch.where(new, codes[other], torch.where(wide(odd) == 1, old & 15, old >> 4))
    byte[at] = torch.where(wide(odd) == 1, neighbour | (codes << 4), codes | (neighbour << 4))
    return _cache_out(s)


def _cache_out(s):
    """The cache as the values that its codes and scales stand for."""
    value = lambda x: _pairs(torch.float8_e4m3fn).view(torch.int16)[:, 0].index_select(0, x.view(-1).int()).view(torch.float8_e4m3fn)  # noqa: E731
    return [value(s["k_pages"]), s["k_scales"].view(torch.float8_e8m0fnu), value(s["v_pages"]),
            s["v_scales"].view(torch.float8_e8m0fnu)]


def _key_pages(codes, scales, table, value, power):
    """[n, kv, tokens, dim] of the pages of table [n, width]."""
    x = value(codes[table]).flatten(-2)  # [n, width, kv, page, dim]
    p = power(scales[table]).unflatten(-1, (-1, 4, 4)).transpose(-1, -2).flatten(-3).transpose(-1, -2)
    x = (x.unflatten(-1, (-1, 32)) * p[..., None]).flatten(-2)
    return x.transpose(1, 2).flatten(2, 3)


def _value_pages(codes, scales, table, value, power):
    x = value(codes[table].unflatten(-1, (2, 8)))  # [n, width, kv, dim / 32, page / 16, 16, 2, 8, 2]
    x = x.permute(0, 1, 2, 4, 7, 8, 3, 6, 5).flatten(6).flatten(3, 5)  # [n, width, kv, page, dim]
    p = power(scales[table]).transpose(-1, -2)
    x = (x.unflatten(-1, (p.shape[-1], -1)) * p[..., None]).flatten(-2)
    return x.transpose(1, 2).flatten(2, 3)


def _attend(q, k, v, visible, scale):
    """q [n, h, g * t, d], k and v [n, h, l, d] f32, visible [n, 1, g * t, l]: the outputs and each row's log sum."""
    score = q @ k.transpose(-1, -2).contiguous()
    score.mul_(scale).masked_fill_(~visible, -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p @ v) / torch.where(total == 0, 1.0, total)
    return out, (top + total.log())[..., 0]


def _plain_paged(s):
    case, cu, kv_len = s["case"], s["cu"].long(), s["lengths"].long()
    kv, dim, group, most = case["kv"], case["dim"], case["heads"] // case["kv"], s["most"]
    value = lambda x: _pairs(torch.float32)[x.int()]  # noqa: E731
    table = s["pages"].long()
    k = _key_pages(s["k_pages"], s["k_scales"], table, value, _power).contiguous()
    v = _value_pages(s["v_pages"], s["v_scales"], table, value, _power).contiguous()
    # row of q for each (sequence, new token), whether there is one, and its position
    step, count = torch.arange(most, device="cuda"), cu[1:] - cu[:-1]
    real = step < count[:, None]
    row = (cu[:-1, None] + step).clamp(max=s["total"] - 1)
    pos = kv_len[:, None] - count[:, None] + step
    n = row.shape[0]
    q = s["q"].float()[row].view(n, most, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(n, kv, group * most, dim)
    j = torch.arange(k.shape[2], device="cuda")
    seen = (j <= pos[..., None]) & (j < kv_len[:, None, None]) & real[..., None]
    if case["window"]:
        seen &= j > pos[..., None] - case["window"]
    seen = seen[:, None, None].expand(n, 1, group, most, k.shape[2]).reshape(n, 1, group * most, k.shape[2])
    out, lse = _attend(q, k, v, seen, 1.0 / math.sqrt(dim))
    out = out.view(n, kv, group, most, dim).permute(0, 3, 1, 2, 4).reshape(n, most, case["heads"], dim)
    lse = lse.view(n, kv, group, most).permute(0, 3, 1, 2).reshape(n, most, case["heads"])
    return (out[real].to(torch.bfloat16), lse[real]) if case["lse"] else out[real].to(torch.bfloat16)


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------


@functools.lru_cache(maxsize=1)
def _context():
    from colormlm_amd import s14

    return s14.Context(0)  # a program keeps one


def _kept(s):
    """What a program makes once: its rotation and its cache."""
    if "cache" not in s:
        from colormlm_amd import attention as A

        case, table = s["case"], s.get("table")
        s["rope"] = None if table is None else A.Rope(table, case["layout"], start=case["dim"] - case["rot"])
        s["cache"] = A.KvCache4(s["k_pages"], s["k_scales"], s["v_pages"], s["v_scales"])
    return s["rope"], s["cache"]


def _run_own(s):
    from colormlm_amd import attention as A

    case, ctx = s["case"], _context()
    op = case["op"]
    if op == "add_norm":
        x, residual = s["x"], s["residual"]
        rows, k = x.shape
        outs = {}
        if residual is not None:
            outs["residual_out"] = torch.empty_like(residual)
        if case["y"]:
            outs["y"] = torch.empty(rows, k, dtype=DTYPES[case["y"]], device="cuda")
        if case["group"]:
            outs["q"] = torch.empty(rows, k, dtype=torch.uint8, device="cuda")
            outs["scales"] = torch.empty(rows, k // case["group"], dtype=torch.uint8, device="cuda")
        A.add_rms_norm(ctx, x, s["weight"], residual=residual, eps=EPS, **outs)
        if case["group"]:
            outs["q"] = outs["q"].view(torch.float8_e4m3fn)
            outs["scales"] = outs["scales"].view(torch.float8_e8m0fnu)
        return list(outs.values())
    rope, cache = _kept(s)
    if op == "append4":
        A.kv_append(ctx, cache, s["k"], s["v"], s["pages"], s["cu"], s["past"], k_weight=s["k_weight"], eps=EPS,
                    rope=rope, max_new=s["most"])
        return _cache_out(s)
    out = torch.empty_like(s["q"])
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float32, device="cuda") if case["lse"] else None
    A.paged_attention(ctx, s["q"], cache, s["pages"], s["cu"], s["lengths"], out, lse=lse, window=case["window"],
                      max_new=s["most"], max_len=s["longest"])
    return out if lse is None else (out, lse)


def run(state):
    if own:
        return _run_own(state)
    return {"add_norm": _plain_add_norm, "append4": _plain_append, "paged4": _plain_paged}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------


def _exact_norm(x, weight):
    return x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * weight.double()


def _exact_add_norm(s):
    case = s["case"]
    x = s["x"].double()
    outs = []
    if s["residual"] is not None:
        x = x + s["residual"].double()
        outs.append(x)
    y = _exact_norm(x, s["weight"])
    if case["y"]:
        outs.append(y)
    if case["group"]:
        part = y.unflatten(-1, (-1, case["group"]))
        # the nearest f32 of the quotient: a maximum at a border goes the operator's way
        scale = (part.abs().amax(-1).clamp(min=1e-4) / 448.0).float().double().log2().ceil().exp2()
        outs += [(part / scale[..., None]).flatten(-2), scale]
    return outs


def _exact_keys(s, positions):
    case, y = s["case"], s["k"].double()
    if s["k_weight"] is not None:
        y = _exact_norm(y, s["k_weight"])
    if case["rot"]:
        rot, start = case["rot"], case["dim"] - case["rot"]
        i = torch.arange(rot // 2, device="cuda")
        angle = positions.double()[:, None] / THETA ** (2.0 * i.double() / rot)
        turn = torch.polar(torch.ones_like(angle), angle)[:, None]
        at = (start + i, start + i + rot // 2) if case["layout"] == "half" else (start + 2 * i, start + 2 * i + 1)
        z = torch.complex(y[..., at[0]], y[..., at[1]]) * turn
        y[..., at[0]], y[..., at[1]] = z.real, z.imag
    return y


def _values64(x):
    v = torch.tensor(E2M1 + tuple(-x for x in E2M1), dtype=torch.float64, device="cuda")
    return torch.stack([v[(x & 15).long()], v[(x >> 4).long()]], -1)


def _power64(code):
    return (code.double() - 127.0).exp2()


def _to_e2m1(x):
    """The nearest E2M1 value, ties to the even code, which has steps of 1/2 below 2, 1 below 4 and then 2."""
    step = torch.where(x.abs() < 2.0, 0.5, torch.where(x.abs() < 4.0, 1.0, 2.0))
    return (x / step).round().mul(step).clamp(-6.0, 6.0)


def _exact_append(s):
    case = s["case"]
    page, dim, cu, past = case["page"], case["dim"], s["cu"].tolist(), s["past"].tolist()
    position = torch.cat([torch.arange(p, p + b - a) for p, a, b in zip(past, cu, cu[1:])]).cuda()
    seq = torch.cat([torch.full((b - a,), i) for i, (a, b) in enumerate(zip(cu, cu[1:]))]).cuda()
    at, slot = s["pages"][seq, position // page].long(), position % page
    outs = []
    for name, rows, block in (("k", _exact_keys(s, position), 32), ("v", s["v"].double(), dim // _parts(dim))):
        part = rows.unflatten(-1, (-1, block))
        most = part.abs().amax(-1).float().double()  # a maximum at a border goes the operator's way
        scale = (most / 6.0).log2().ceil().clamp(-100.0, 100.0).exp2()
        value = _to_e2m1(part / scale[..., None]).flatten(-2)
        codes, scales = _values64(s[name + "_pages"]), _power64(s[name + "_scales"])
        if name == "k":
            codes.flatten(-2)[at, :, slot] = value
            scales.unflatten(-1, (-1, 4, 4))[at, :, :, slot // 16, slot % 4, slot % 16 // 4] = scale
        else:
            codes.unflatten(-2, (2, 8))[at, :, :, slot // 16, :, :, slot % 16 // 2, slot % 2] = (
                value.unflatten(-1, (-1, 2, 16)).transpose(-1, -2))
            scales[at, :, :, slot] = scale
        outs += [codes.flatten(), scales]
    return outs


def _exact_sequence(q, k, v, case):
    """q [t, heads, dim] at the end of k, v [kv, l, dim], all in 64 bits."""
    t, length, group = q.shape[0], k.shape[1], case["heads"] // case["kv"]
    at = torch.arange(length - t, length, device="cuda")[:, None]
    j = torch.arange(length, device="cuda")
    hidden = (j > at) | (j <= at - case["window"]) if case["window"] else j > at
    out, lse = torch.empty_like(q), torch.empty(q.shape[:2], dtype=torch.float64, device="cuda")
    for h in range(case["heads"]):
        score = (q[:, h] @ k[h // group].T) / math.sqrt(case["dim"])
        score.masked_fill_(hidden, -math.inf)
        lse[:, h] = score.logsumexp(-1)
        out[:, h] = (score - lse[:, h, None]).exp() @ v[h // group]
    return out, lse


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "add_norm":
        return _exact_add_norm(s)
    if case["op"] == "append4":
        return _exact_append(s)
    outs, cu = [], s["cu"].tolist()
    for i, (a, b) in enumerate(zip(cu, cu[1:])):
        length = int(s["lengths"][i])
        ids = s["pages"][i:i + 1, :-(-length // case["page"])].long()
        k = _key_pages(s["k_pages"], s["k_scales"], ids, _values64, _power64)[0, :, :length]
        v = _value_pages(s["v_pages"], s["v_scales"], ids, _values64, _power64)[0, :, :length]
        outs.append(_exact_sequence(s["q"][a:b].double(), k, v, case))
    out, lse = (torch.cat(x) for x in zip(*outs))
    return (out, lse) if case["lse"] else out

"""The operators of a streamed attention layer over a 4-bit cache, and what their speed is measured on.

Every 4-bit value is OCP MX: a code of four bits (sign, two exponent bits, one
of mantissa: 0, 0.5, 1, 1.5, 2, 3, 4, 6) times one power of two per 32
consecutive values, held as a biased byte (255: the group is NaN).

- ``qk_norm_rope``: RMSNorm of every query and key head, then the rotation of
  the last lanes at the token's own position.
- ``kv4_append`` / ``kv4_read``: keys and values into a paged 4-bit cache and
  back out of it.
- ``kv4_attention``: softmax attention of one or more new tokens per sequence
  over that cache.
- ``linear_fp4``: x W^T + b with 4-bit weights.

A cache is a uint8 tensor [pages, kv_heads, page_size * (head_dim + head_dim / 16)].
One (page, head) holds the key codes [page_size][head_dim / 2], the value codes
[head_dim / 2][page_size], the key scales [page_size][head_dim / 32] and the
value scales [head_dim / 32][page_size]; a byte holds elements 2 j (low four
bits) and 2 j + 1 of a token. ``page_table`` [batch, n] (int32) names a
sequence's pages, ``positions`` [batch, length] (int32) each token's place in
its sequence; a negative position is padding.

``listed()`` names fixed cases, ``draw(rng)`` gives further ones of the same
ranges, ``prepare`` makes what a program holds before the call, ``run`` is the
call, ``exact`` its results in float64 and ``work`` the bytes and operations it
cannot do without. With ``own`` the calls are the package's operators,
otherwise their plain form in tensor operations.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
_DT = {"f32": torch.float32, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "bf16": 2}


def listed():
    return [
        # One new token for each of 16 streams, 8 key heads: a microsecond of traffic, so the launch counts.
        dict(name="qk_16x1", kind="qk", batch=16, length=1, heads=32, kv_heads=8, head_dim=128, rope=128, dtype="bf16"),
        # Two prompts of uneven length in fp32, half of each head rotated (the decoupled slice of the MLA layers).
        dict(name="qk_2x4001_f32", kind="qk", batch=2, length=4001, heads=16, kv_heads=16, head_dim=64, rope=32,
             dtype="f32"),
        # The same 16 streams' token into their caches and back.
        dict(name="cache_16x1", kind="cache", batch=16, length=1, kv_heads=8, head_dim=128, page=64, dtype="bf16"),
        # Prompts written to the cache, padded to the longest, and read back (a prefix handed on).
        dict(name="cache_4x2048_f32", kind="cache", batch=4, length=2048, kv_heads=8, head_dim=128, page=64,
             dtype="f32"),
        # One stream at the MLA geometry of this package (8 heads of 32, a 480-bar window), fp32: latency.
        dict(name="attn_1x480_f32", kind="attn", batch=1, length=1, context=480, heads=8, kv_heads=8, head_dim=32,
             page=32, dtype="f32"),
        # A server's step: 32 streams of uneven length, four query heads to a key head.
        dict(name="attn_32x8000", kind="attn", batch=32, length=1, context=8000, heads=32, kv_heads=8, head_dim=128,
             page=64, dtype="bf16"),
        # One stream with a very long past: the keys have to be split over the chip.
        dict(name="attn_1x131072", kind="attn", batch=1, length=1, context=131072, heads=32, kv_heads=8, head_dim=128,
             page=256, dtype="bf16"),
        # The largest step: 64 long streams, fp32 activations.
        dict(name="attn_64x16384_f32", kind="attn", batch=64, length=1, context=16384, heads=32, kv_heads=8,
             head_dim=128, page=64, dtype="f32"),
        # A chunk of a long prompt against what is cached: bound by products, not by bytes.
        dict(name="attn_chunk_512", kind="attn", batch=2, length=512, context=8192, heads=32, kv_heads=8, head_dim=128,
             page=64, dtype="bf16"),
        # A decode projection of one token, and of a batch in fp32 (an odd number of outputs).
        dict(name="lin_1", kind="linear", rows=1, k=4096, n=12288, bias=False, dtype="bf16"),
        dict(name="lin_16_f32", kind="linear", rows=16, k=4096, n=4100, bias=True, dtype="f32"),
        # A batch of prompts' tokens: as many operations as bytes allow.
        dict(name="lin_256", kind="linear", rows=256, k=8192, n=8192, bias=False, dtype="bf16"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["qk", "cache", "attn", "attn", "linear"])
    dtype = rng.choice(["f32", "bf16"])
    if kind == "linear":
        return dict(kind=kind, rows=_log_int(rng, 1, 256), k=32 * _log_int(rng, 2, 256), n=_log_int(rng, 48, 8192),
                    bias=rng.random() < 0.5, dtype=dtype)
    head_dim = rng.choice([32, 64, 128, 256])
    heads, kv_heads = rng.choice([(8, 8), (4, 4), (32, 8), (16, 2), (12, 4), (8, 1), (24, 1)])
    batch = _log_int(rng, 1, 64)
    if kind == "qk":
        length = rng.choice([1, _log_int(rng, 1, max(1, 8192 // batch))])
        return dict(kind=kind, batch=batch, length=length, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                    rope=rng.choice([head_dim, head_dim // 2]), dtype=dtype)
    page = rng.choice([16, 32, 48, 64, 128, 256])
    if kind == "cache":
        length = rng.choice([1, _log_int(rng, 1, max(1, 8192 // batch))])
        return dict(kind=kind, batch=batch, length=length, kv_heads=kv_heads, head_dim=head_dim, page=page, dtype=dtype)
    most = min(131072, 2 ** 30 // (batch * kv_heads * head_dim))  # no more bytes than the largest listed case
    length = rng.choice([1, 1, 1, rng.randint(2, 8), _log_int(rng, 9, 300)])
    context = _log_int(rng, length, max(length, most // max(1, length // 16)))
    return dict(kind=kind, batch=batch, length=length, context=context, heads=heads, kv_heads=kv_heads,
                head_dim=head_dim, page=page, dtype=dtype)


# --------------------------------------------------------------- what a case holds


def _lengths(case):
    """Tokens of each sequence after this call: uneven, from a quarter of the context up, the first the longest.
    A sequence holds at least the new tokens."""
    most, n = case["context"], case["batch"]
    spread = most - max(case["length"], most // 4)
    return [most - (spread * ((b * 37) % 64)) // 64 if n > 1 else most for b in range(n)]


def _real(case):
    """Tokens of each row of a padded batch: the first is full."""
    n = case["length"]
    return [n - (n * ((b * 29) % 64)) // 160 for b in range(case["batch"])]


def _positions(case):
    length = case["length"]
    if case["kind"] == "attn":
        rows = [[total - length + i for i in range(length)] for total in _lengths(case)]
    else:  # a sequence that has (37 b + 11) % 500 tokens already; padding behind the new ones
        rows = [[(37 * b + 11) % 500 + i if i < real else -1 for i in range(length)]
                for b, real in enumerate(_real(case))]
    return torch.tensor(rows, dtype=torch.int32, device=DEV)


def _pages(case, gen, tokens):
    """A page table over shuffled pages (-1 where a sequence has no page) and the number of pages."""
    page = case["page"]
    counts = [-(-t // page) for t in tokens]
    order = torch.randperm(sum(counts), generator=gen, device=DEV).to(torch.int32)
    table = torch.full((len(counts), max(counts)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = order[at:at + n]
        at += n
    return table, at


def _bank(gen, spread):
    """4096 groups of 32 normal values in four bits, 16 bytes and a scale byte each."""
    x = torch.randn(4096, 32, generator=gen, device=DEV) * torch.exp(0.3 * torch.randn(4096, 1, generator=gen, device=DEV)) * spread
    return _quantise(x)


def _random_cache(case, gen, pages):
    """A filled cache of normal keys and values, groups drawn from a bank."""
    heads, dim, page = case["kv_heads"], case["head_dim"], case["page"]
    groups = dim // 32
    codes, scales = _bank(gen, 1.0)
    cache = torch.empty(pages, heads, page * (dim + dim // 16), dtype=torch.uint8, device=DEV)
    kc, vc, ks, vs = _parts(cache, page, dim)
    step = max(1, (1 << 22) // (heads * page * groups))
    for p in range(0, pages, step):
        for part, scale, minor in ((kc, ks, False), (vc, vs, True)):
            n = min(step, pages - p)
            pick = torch.randint(0, 4096, (n, heads, page, groups), generator=gen, device=DEV, dtype=torch.int32)
            c, s = codes[pick].flatten(3), scales[pick].flatten(3)
            part[p:p + n] = c.transpose(2, 3) if minor else c
            scale[p:p + n] = s.transpose(2, 3) if minor else s
    return cache


def _rope_tables(positions, dim):
    inv = 10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=DEV) / dim)
    angle = torch.arange(positions, dtype=torch.float64, device=DEV)[:, None] * inv
    angle = torch.cat([angle, angle], 1)
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dtype = _DT[case["dtype"]]
    state = {"case": case}

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)

    if case["kind"] == "linear":
        codes, scales = _bank(gen, case["k"] ** -0.5)
        pick = torch.randint(0, 4096, (case["n"], case["k"] // 32), generator=gen, device=DEV)
        state.update(x=normal(case["rows"], case["k"]).to(dtype), codes=codes[pick].flatten(1), scales=scales[pick].flatten(1),
                     bias=normal(case["n"]) if case["bias"] else None)
    else:
        batch, length, dim = case["batch"], case["length"], case["head_dim"]
        state["positions"] = _positions(case)
        if case["kind"] == "attn":
            table, pages = _pages(case, gen, _lengths(case))
            state.update(q=normal(batch, length, case["heads"], dim).to(dtype), page_table=table,
                         cache=_random_cache(case, gen, pages), scale=dim ** -0.5)
        elif case["kind"] == "cache":
            # Keys and values are views of one projection's rows, as a layer has them.
            kv = (normal(batch, length, 2 * case["kv_heads"], dim) * 1.7).to(dtype)
            table, pages = _pages(case, gen, [(37 * b + 11) % 500 + n for b, n in enumerate(_real(case))])
            state.update(k=kv[:, :, :case["kv_heads"]], v=kv[:, :, case["kv_heads"]:], page_table=table,
                         cache=_random_cache(case, gen, pages))
        else:
            heads, kv_heads = case["heads"], case["kv_heads"]
            qkv = (normal(batch, length, heads + 2 * kv_heads, dim) * 1.7).to(dtype)
            cos, sin = _rope_tables(500 + length, case["rope"])
            state.update(q=qkv[:, :, :heads], k=qkv[:, :, heads:heads + kv_heads], q_weight=1 + 0.2 * normal(dim),
                         k_weight=1 + 0.2 * normal(dim), cos=cos, sin=sin)
    if own:
        package = str(Path("montlok.cpp_amd").resolve())  # the working folder is the repository's root
        if package not in sys.path:
            sys.path.insert(0, package)
        from montlok import _C

        state["ops"] = _C
    return state


# --------------------------------------------------------------- the calls


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    ops, case = s["ops"], s["case"]
    if case["kind"] == "linear":
        return ops.linear_fp4(s["x"], s["codes"], s["scales"], s["bias"])
    if case["kind"] == "attn":
        return ops.kv4_attention(s["q"], s["cache"], s["page_table"], s["positions"], s["scale"])
    if case["kind"] == "cache":
        ops.kv4_append(s["k"], s["v"], s["cache"], s["page_table"], s["positions"])
        return ops.kv4_read(s["cache"], s["page_table"], s["positions"], case["head_dim"], _DT[case["dtype"]])
    return ops.qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], 1e-5, s["cos"], s["sin"], s["positions"])


def _parts(cache, page, dim):
    """Views of a cache: key codes [.., page, dim/2], value codes [.., dim/2, page], key scales, value scales."""
    a, b = page * dim // 2, page * dim // 32
    return (cache[..., :a].unflatten(-1, (page, dim // 2)), cache[..., a:2 * a].unflatten(-1, (dim // 2, page)),
            cache[..., 2 * a:2 * a + b].unflatten(-1, (page, dim // 32)),
            cache[..., 2 * a + b:].unflatten(-1, (dim // 32, page)))


def _quantise(x):
    """[..., 32 g] in fp32 -> codes [..., 16 g], scale bytes [..., g]."""
    groups = x.float().unflatten(-1, (-1, 32))
    most = groups.abs().amax(-1, keepdim=True)
    fine = torch.isfinite(groups).all(-1, keepdim=True)
    byte = ((most.view(torch.int32) + 0x3FFFFF) >> 23) - 2  # the smallest power of two whose six-fold reaches `most`
    byte = byte.clamp(3, 252)
    y = torch.where(fine, torch.ldexp(groups, 127 - byte), 0.0)
    a = y.abs()
    code = ((a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = torch.where(torch.signbit(y), code + 8, code)
    packed = code[..., 0::2] + 16 * code[..., 1::2]
    byte = torch.where(fine, byte, 255)
    return packed.to(torch.uint8).flatten(-2), byte.squeeze(-1).to(torch.uint8)


def _values(codes, scales):
    """[..., 16 g] codes and [..., g] scale bytes -> [..., 32 g] in fp32."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=DEV)
    table = torch.cat([table, -table])
    both = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    value = table[both.int()].unflatten(-1, (-1, 32))
    power = torch.ldexp(torch.ones((), device=DEV), scales.int() - 127)
    power = torch.where(scales == 255, torch.nan, power)
    return (value * power[..., None]).flatten(-2)


def _run_plain(s):
    case = s["case"]
    dtype = _DT[case["dtype"]]
    if case["kind"] == "linear":
        y = s["x"].float() @ _values(s["codes"], s["scales"]).t()
        return (y if s["bias"] is None else y + s["bias"]).to(dtype)
    if case["kind"] == "attn":
        return _plain_attention(s, case).to(dtype)
    if case["kind"] == "cache":
        page, dim = case["page"], case["head_dim"]
        parts = _parts(s["cache"], page, dim)
        valid = (s["positions"] >= 0)
        at = s["positions"].clamp(min=0).long()
        where = s["page_table"].long().gather(1, at // page)[valid]
        offset = (at % page)[valid]
        for x, codes, scales, minor in ((s["k"], parts[0], parts[2], False), (s["v"], parts[1], parts[3], True)):
            c, e = _quantise(x[valid])
            if minor:
                codes[where, :, :, offset], scales[where, :, :, offset] = c, e
            else:
                codes[where, :, offset], scales[where, :, offset] = c, e
        out = []
        for codes, scales, minor in ((parts[0], parts[2], False), (parts[1], parts[3], True)):
            read = torch.zeros(s["k"].shape, device=DEV)
            read[valid] = _values(codes[where, :, :, offset], scales[where, :, :, offset]) if minor else \
                _values(codes[where, :, offset], scales[where, :, offset])
            out.append(read.to(dtype))
        return tuple(out)
    out = []
    for x, weight in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
        x = x.double()
        y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5) * weight
        rope = case["rope"]
        valid = (s["positions"] >= 0)[..., None, None]
        at = s["positions"].clamp(min=0).long()
        cos, sin = s["cos"].double()[at][:, :, None], s["sin"].double()[at][:, :, None]
        keep, turn = y[..., :y.shape[-1] - rope], y[..., y.shape[-1] - rope:]
        half = torch.cat([-turn[..., rope // 2:], turn[..., :rope // 2]], -1)
        out.append(torch.where(valid, torch.cat([keep, turn * cos + half * sin], -1), 0.0).to(dtype))
    return tuple(out)


def _plain_attention(s, case):
    page, dim, kv_heads = case["page"], case["head_dim"], case["kv_heads"]
    per = case["heads"] // kv_heads
    parts = _parts(s["cache"], page, dim)
    out = torch.empty(s["q"].shape, device=DEV)
    for b, total in enumerate(_lengths(case)):
        pages = s["page_table"][b, :-(-total // page)].long()
        k = _values(parts[0][pages], parts[2][pages])  # [pages, kv_heads, page, dim]
        v = _values(parts[1][pages].transpose(2, 3), parts[3][pages].transpose(2, 3))
        seen = torch.arange(len(pages) * page, device=DEV) <= s["positions"][b][:, None, None]  # [length, 1, keys]
        for h in range(kv_heads):
            kh, vh = k[:, h].flatten(0, 1), v[:, h].flatten(0, 1)
            q = s["q"][b, :, h * per:(h + 1) * per].float()
            score = (q.flatten(0, 1) @ kh.t() * s["scale"]).unflatten(0, (-1, per))
            score = torch.where(seen, score, -torch.inf)
            weight = torch.exp(score - score.amax(-1, keepdim=True))
            weight = weight / weight.sum(-1, keepdim=True)
            out[b, :, h * per:(h + 1) * per] = (weight.flatten(0, 1) @ vh).unflatten(0, (-1, per))
    return out


# --------------------------------------------------------------- float64, from the definitions


def _number(code):
    """The value of a four-bit code in float64: sign, exponent and mantissa bits taken apart."""
    code = code.long()
    exponent, mantissa = (code >> 1) & 3, (code & 1).double()
    size = torch.where(exponent == 0, 0.5 * mantissa, (1 + 0.5 * mantissa) * 2.0 ** (exponent - 1).double())
    return torch.where(code >= 8, -size, size)


def _mx64(codes, scales):
    """Row-major codes [n, 16 g] and scales [n, g] -> [n, 32 g] in float64."""
    out = torch.empty(codes.shape[0], 2 * codes.shape[1], dtype=torch.float64, device=DEV)
    out[:, 0::2], out[:, 1::2] = _number(codes & 15), _number(codes >> 4)
    out *= (2.0 ** (scales.double() - 127)).repeat_interleave(32, 1)
    return out


def _rounded64(x):
    """Every group of 32 of [n, 32 g] at the nearest value of its 4-bit grid, in float64."""
    y = x.double().unflatten(-1, (-1, 32))
    most = y.abs().amax(-1, keepdim=True)
    power = torch.ceil(torch.log2(torch.where(most > 0, most, 1e-300) / 6))
    power = torch.where(6 * 2.0 ** (power - 1) >= most, power - 1, power)  # the logarithm's rounding put right
    power = torch.where(6 * 2.0 ** power < most, power + 1, power).clamp(-124, 125)
    grid = torch.tensor([0, 1, 2, 3, 4, 6, 8, 12], dtype=torch.float64, device=DEV) / 2
    a = (y / 2.0 ** power).abs()
    low = torch.bucketize(a, grid, right=True) - 1  # grid[low] <= a
    up = (low + 1).clamp(max=7)
    to_up, to_low = grid[up] - a, a - grid[low]
    pick = torch.where((to_up < to_low) | ((to_up == to_low) & (up % 2 == 0)), up, low)
    return (torch.sign(y) * grid[pick] * 2.0 ** power).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "linear":
        y = s["x"].double() @ _mx64(s["codes"], s["scales"]).t()
        return y if s["bias"] is None else y + s["bias"].double()
    if case["kind"] == "cache":
        shown = (s["positions"] >= 0)[..., None, None]
        return tuple(torch.where(shown, _rounded64(x.reshape(-1, x.shape[-1])).view(x.shape), 0.0) for x in (s["k"], s["v"]))
    if case["kind"] == "qk":
        rope, dim = case["rope"], case["head_dim"]
        result = []
        for x, weight in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
            x = x.double()
            y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / dim + 1e-5) * weight.double()
            first, second = y[..., dim - rope:dim - rope // 2].clone(), y[..., dim - rope // 2:].clone()
            at = torch.clamp(s["positions"], min=0).long()
            c, d = s["cos"][at].double()[:, :, None], s["sin"][at].double()[:, :, None]
            y[..., dim - rope:dim - rope // 2] = first * c[..., :rope // 2] - second * d[..., :rope // 2]
            y[..., dim - rope // 2:] = second * c[..., rope // 2:] + first * d[..., rope // 2:]
            y[s["positions"] < 0] = 0
            result.append(y)
        return tuple(result)
    # Attention: a sequence's pages laid end to end for one key head at a time.
    page, dim, per = case["page"], case["head_dim"], case["heads"] // case["kv_heads"]
    codes, scales = page * dim // 2, page * dim // 32
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for b, total in enumerate(_lengths(case)):
        table = s["page_table"][b, :(total + page - 1) // page].long()
        for h in range(case["kv_heads"]):
            held = s["cache"][table, h]
            keys = _mx64(held[:, :codes].reshape(-1, dim // 2),
                         held[:, 2 * codes:2 * codes + scales].reshape(-1, dim // 32))[:total]
            values = _mx64(held[:, codes:2 * codes].reshape(-1, dim // 2, page).transpose(1, 2).reshape(-1, dim // 2),
                           held[:, 2 * codes + scales:].reshape(-1, dim // 32, page).transpose(1, 2).reshape(-1, dim // 32))[:total]
            for j in range(h * per, (h + 1) * per):
                score = s["q"][b, :, j].double() @ keys.t() * s["scale"]
                score.masked_fill_(torch.arange(total, device=DEV) > s["positions"][b][:, None], -math.inf)
                out[b, :, j] = torch.softmax(score, -1) @ values
    return out


# --------------------------------------------------------------- the least work


def work(case):
    size = _SIZE[case["dtype"]]
    if case["kind"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        return {"bytes": n * k // 2 + n * k // 32 + size * m * (k + n) + (4 * n if case["bias"] else 0), "flops": 2.0 * m * n * k}
    dim, length = case["head_dim"], case["length"]
    if case["kind"] == "attn":
        totals = _lengths(case)
        keys = sum(t * length - length * (length - 1) // 2 for t in totals)
        return {"bytes": sum(totals) * case["kv_heads"] * (dim + dim // 16) + 2 * size * len(totals) * length * case["heads"] * dim,
                "flops": 4.0 * dim * case["heads"] * keys}
    tokens = case["batch"] * length
    real = sum(_real(case))
    if case["kind"] == "cache":
        return {"bytes": case["kv_heads"] * (2 * size * dim * (real + tokens) + 2 * real * (dim + dim // 16)),
                "flops": 8.0 * real * case["kv_heads"] * dim}
    heads = case["heads"] + case["kv_heads"]
    return {"bytes": size * heads * dim * (real + tokens) + 8 * real * case["rope"] + 8 * dim,
            "flops": 7.0 * real * heads * dim}

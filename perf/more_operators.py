"""The operators of a streamed latent attention (MLA) layer, and what their speed is measured on.

A layer of this kind keeps one latent vector a token and a short rotated key
part that all heads share; a head's keys and values are products of the latent
with its own weights. A streamed layer multiplies those weights into the query
and into the output instead ("absorbed"), so that every head reads the same
cached rows.

- ``rope``: the rotation of queries and keys at their own positions, neighbours
  or halves paired, a part of the head, frequencies stretched for long contexts.
- ``latent_append`` / ``latent_read``: latents and rotated key parts into a
  paged cache and back out of it, in eight bits or in bfloat16.
- ``latent_attention``: softmax attention of one or more new tokens a sequence,
  or of a tree of drafted ones, over that cache.
- ``head_linear``: every head's own matrix times its part of the activations.

A cache is a uint8 tensor [pages, page_size, row]. A row of the eight-bit cache
is R e4m3 codes, P bfloat16 of the key part and 16 bytes that begin with the
float32 power of two that the codes are multiplied by (NaN: the latent is NaN).
A row of the bfloat16 cache is R + P bfloat16 and 16 unused bytes.
``page_table`` [batch, n] (int32) names a sequence's pages, ``positions``
[batch, length] (int32) each token's place in its sequence; a negative position
is padding. ``ancestors`` [batch, length] (int64) makes the tokens of a call a
tree: token i, at the place p, sees the places below p - i, and p - i + j where
its bit j is set.

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
_FLOPS, _BYTES = 1.6e11, 4.2e8  # what a drawn attention may cost: the largest listed ones


def listed():
    return [
        # One new token of 16 streams, queries of 64 heads and the shared key part: a launch's latency.
        dict(name="rope_16x1", kind="rope", batch=16, length=1, heads=64, kv_heads=1, head_dim=64, rope=64,
             interleaved=True, factor=40.0, far=150000, dtype="bf16"),
        # Two prompts of uneven length in fp32, the last half of each head rotated, at ordinary positions.
        dict(name="rope_2x4001_f32", kind="rope", batch=2, length=4001, heads=16, kv_heads=16, head_dim=64, rope=32,
             interleaved=False, factor=1.0, far=500, dtype="f32"),
        # The 16 streams' token into their caches and back.
        dict(name="cache_16x1", kind="cache", batch=16, length=1, rank=512, rope=64, page=64, store="e4m3", dtype="bf16"),
        # Prompts written to the cache, padded to the longest, and read back (a prefix handed on).
        dict(name="cache_8x4000_f32", kind="cache", batch=8, length=4000, rank=512, rope=64, page=64, store="e4m3",
             dtype="f32"),
        # One stream at the MLA geometry of this package (8 heads of 32, latents of 64, a 480-bar window), fp32: latency.
        dict(name="attn_1x480_f32", kind="attn", batch=1, length=1, context=480, heads=8, rank=64, rope=16, page=32,
             store="bf16", tree=False, dtype="f32"),
        # A server's step: 24 streams of uneven length, 16 heads: bound by the cache's bytes.
        dict(name="attn_24x8000", kind="attn", batch=24, length=1, context=8000, heads=16, rank=512, rope=64, page=64,
             store="e4m3", tree=False, dtype="bf16"),
        # One stream with a very long past: the tokens have to be split over the chip.
        dict(name="attn_1x131072", kind="attn", batch=1, length=1, context=131072, heads=32, rank=512, rope=64, page=256,
             store="e4m3", tree=False, dtype="bf16"),
        # The largest step: 64 long streams of 64 heads, as many products as bytes.
        dict(name="attn_64x16384", kind="attn", batch=64, length=1, context=16384, heads=64, rank=512, rope=64, page=64,
             store="e4m3", tree=False, dtype="bf16"),
        # Trees of 48 drafted tokens to be verified over a bfloat16 cache.
        dict(name="attn_tree_8x48", kind="attn", batch=8, length=48, context=4096, heads=16, rank=256, rope=32, page=48,
             store="bf16", tree=True, dtype="bf16"),
        # A chunk of two long prompts against what is cached: bound by products.
        dict(name="attn_chunk_256", kind="attn", batch=2, length=256, context=8000, heads=24, rank=512, rope=64, page=64,
             store="e4m3", tree=False, dtype="bf16"),
        # A step's queries of 64 heads into the latents' space: the weights' bytes.
        dict(name="head_in_24", kind="head", tokens=24, heads=64, inner=128, rank=512, out=False, dtype="bf16",
             weights="bf16"),
        # A chunk's attended latents back to the heads' values, fp32.
        dict(name="head_out_600_f32", kind="head", tokens=600, heads=24, inner=96, rank=512, out=True, dtype="f32",
             weights="f32"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["rope", "cache", "attn", "attn", "head"])
    dtype = rng.choice(["f32", "bf16"])
    if kind == "head":
        weights = "bf16" if dtype == "bf16" else rng.choice(["f32", "bf16"])
        heads = rng.choice([4, 8, 16, 24, 64, 128])
        return dict(kind=kind, tokens=_log_int(rng, 1, 40000 // heads), heads=heads, inner=rng.choice([16, 32, 64, 96, 128, 192]),
                    rank=rng.choice([64, 128, 256, 512]), out=rng.random() < 0.5, dtype=dtype, weights=weights)
    batch = _log_int(rng, 1, 64)
    if kind == "rope":
        head_dim = rng.choice([16, 32, 64, 96, 128])
        return dict(kind=kind, batch=batch, length=rng.choice([1, _log_int(rng, 1, max(1, 8192 // batch))]),
                    heads=rng.choice([4, 8, 12, 16, 24]), kv_heads=rng.choice([1, 1, 2, 4, 8]), head_dim=head_dim,
                    rope=rng.choice([head_dim, head_dim // 2]), interleaved=rng.random() < 0.5,
                    factor=rng.choice([1.0, 1.0, 4.0, 40.0]), far=_log_int(rng, 500, 1000000), dtype=dtype)
    rank, rope = rng.choice([(64, 16), (64, 32), (128, 32), (256, 32), (256, 64), (512, 32), (512, 64)])
    page, store = rng.choice([16, 32, 48, 64, 128, 256]), rng.choice(["e4m3", "e4m3", "bf16"])
    if kind == "cache":
        length = rng.choice([1, _log_int(rng, 1, max(1, 30000 // batch))])
        return dict(kind=kind, batch=batch, length=length, rank=rank, rope=rope, page=page, store=store, dtype=dtype)
    tree = rng.random() < 0.25
    length = rng.randint(2, 64) if tree else rng.choice([1, 1, 1, rng.randint(2, 8), _log_int(rng, 9, 300)])
    heads = rng.choice([4, 8, 12, 16, 24, 32, 64, 128])
    flops = _FLOPS * (0.3 if dtype == "f32" else 1.0)
    length = min(length, int(math.sqrt(flops / (2.0 * (2 * rank + rope) * heads * batch))))
    per_token = rank + 2 * rope + 4 if store == "e4m3" else 2 * (rank + rope)
    moved = _SIZE[dtype] * batch * heads * (2 * rank + rope)  # queries and outputs of one token a sequence
    length = max(1, min(length, int(_BYTES / 2 / moved)))
    most = min(131072, int((_BYTES - moved * length) / (batch * per_token)), int(flops / (2.0 * (2 * rank + rope) * heads * batch * length)))
    return dict(kind=kind, batch=batch, length=length, context=_log_int(rng, length, max(length, most)), heads=heads, rank=rank,
                rope=rope, page=page, store=store, tree=tree, dtype=dtype)


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


def _had(case, b):
    """Tokens that a sequence holds before a call that only writes or rotates."""
    return (37 * b + 11) * 7919 % case.get("far", 500)


def _positions(case):
    length = case["length"]
    if case["kind"] == "attn":
        rows = [[total - length + i for i in range(length)] for total in _lengths(case)]
    else:
        rows = [[_had(case, b) + i if i < real else -1 for i in range(length)] for b, real in enumerate(_real(case))]
    return torch.tensor(rows, dtype=torch.int32, device=DEV)


def _ancestors(case, seed):
    """A tree for each sequence: every drafted token hangs on one of the eight before it, or on the cached text, and sees
    its ancestors and itself."""
    rows = []
    for b in range(case["batch"]):
        bits = []
        for i in range(case["length"]):
            back = (seed * 31 + b * 17 + i * 7) * 2654435761 % 4294967296 // 65536 % 8 + 1
            bits.append((bits[i - back] if i >= back else 0) | 1 << i)
        rows.append([v - 2 ** 64 if v >= 2 ** 63 else v for v in bits])
    return torch.tensor(rows, dtype=torch.int64, device=DEV)


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


def _row_bytes(case):
    rank, rope = case["rank"], case["rope"]
    return rank + 2 * rope + 16 if case["store"] == "e4m3" else 2 * (rank + rope) + 16


def _random_cache(case, gen, pages):
    """A filled cache of normal latents and key parts, rows drawn from a bank."""
    rank, rope, n = case["rank"], case["rope"], 8192
    latent = torch.randn(n, rank, generator=gen, device=DEV) * torch.exp(0.3 * torch.randn(n, 1, generator=gen, device=DEV))
    bank = torch.zeros(n, _row_bytes(case), dtype=torch.uint8, device=DEV)
    _write(bank, latent, torch.randn(n, rope, generator=gen, device=DEV), case)
    cache = torch.empty(pages * case["page"], bank.shape[1], dtype=torch.uint8, device=DEV)
    step = 1 << 17
    for i in range(0, len(cache), step):
        cache[i:i + step] = bank[torch.randint(0, n, (min(step, len(cache) - i),), generator=gen, device=DEV)]
    return cache.view(pages, case["page"], -1)


def _frequencies(case):
    """Radians a position of each pair, and the rotated part's factor: 10000^(-2 i / rope); stretched by ``factor``, pairs
    that turn less than once over 4096 positions are slowed down by it, those that turn more than 32 times are kept, with a
    straight ramp over the pairs between (the method published as YaRN)."""
    rope, factor, theta, original = case["rope"], case["factor"], 10000.0, 4096
    plain = [theta ** (-2.0 * i / rope) for i in range(rope // 2)]
    if factor == 1.0:
        return plain, 1.0

    def pair(turns):
        return rope * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))

    low, high = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), rope // 2 - 1)
    out = []
    for i, f in enumerate(plain):
        slow = min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
        out.append(f * (1 - slow) + f / factor * slow)
    return out, 0.1 * math.log(factor) + 1.0


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dtype = _DT[case["dtype"]]
    state = {"case": case}

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)

    if case["kind"] == "head":
        tokens, heads, inner, rank = case["tokens"], case["heads"], case["inner"], case["rank"]
        # One projection holds a head's key rows, then its value rows; queries are a part of each head's row.
        weight = (normal(heads, 2 * inner, rank) * rank ** -0.5).to(_DT[case["weights"]])
        if case["out"]:
            state.update(x=normal(tokens, heads, rank).to(dtype), weight=weight[:, inner:])
        else:
            state.update(x=normal(tokens, heads, inner + 32).to(dtype)[..., :inner], weight=weight[:, :inner].transpose(1, 2))
    else:
        batch, length, rope = case["batch"], case["length"], case["rope"]
        state["positions"] = _positions(case)
        if case["kind"] == "rope":
            heads, dim = case["heads"], case["head_dim"]
            # Queries are the last part of wider heads, keys the last columns of another projection, as a layer has them.
            q = normal(batch, length, heads, dim + 32).to(dtype)
            k = normal(batch, length, 64 + case["kv_heads"] * dim).to(dtype)
            frequencies, magnitude = _frequencies(case)
            state.update(q=q[..., 32:], k=k[..., 64:].unflatten(-1, (case["kv_heads"], dim)), magnitude=magnitude,
                         frequencies=torch.tensor(frequencies, dtype=torch.float64, device=DEV))
        elif case["kind"] == "cache":
            both = (normal(batch, length, case["rank"] + rope) * 1.7).to(dtype)
            table, pages = _pages(case, gen, [_had(case, b) + n for b, n in enumerate(_real(case))])
            state.update(latent=both[..., :case["rank"]], k_rope=both[..., case["rank"]:], page_table=table,
                         cache=torch.zeros(pages, case["page"], _row_bytes(case), dtype=torch.uint8, device=DEV))
        else:
            table, pages = _pages(case, gen, _lengths(case))
            state.update(q_latent=normal(batch, length, case["heads"], case["rank"]).to(dtype),
                         q_rope=normal(batch, length, case["heads"], rope).to(dtype), page_table=table,
                         cache=_random_cache(case, gen, pages), scale=(case["rank"] + rope) ** -0.5,
                         ancestors=_ancestors(case, seed) if case["tree"] else None)
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
    if case["kind"] == "head":
        return ops.head_linear(s["x"], s["weight"])
    if case["kind"] == "rope":
        return ops.rope(s["q"], s["k"], s["frequencies"], s["positions"], case["interleaved"], s["magnitude"])
    if case["kind"] == "cache":
        ops.latent_append(s["latent"], s["k_rope"], s["cache"], s["page_table"], s["positions"])
        return ops.latent_read(s["cache"], s["page_table"], s["positions"], case["rank"], case["rope"], _DT[case["dtype"]])
    return ops.latent_attention(s["q_latent"], s["q_rope"], s["cache"], s["page_table"], s["positions"], s["scale"],
                                s["ancestors"])


def _write(rows, latent, k_rope, case):
    """latent [n, R] and k_rope [n, P] into rows [n, bytes]."""
    rank = case["rank"]
    k_rope = k_rope.to(torch.bfloat16).contiguous().view(torch.uint8)
    if case["store"] == "bf16":
        latent = latent.to(torch.bfloat16).contiguous().view(torch.uint8)
        rows[:, :2 * rank], rows[:, 2 * rank:2 * rank + k_rope.shape[1]] = latent, k_rope
        return
    x = latent.float()
    fine = torch.isfinite(x).all(-1, keepdim=True)
    most = torch.where(fine, x, 0.0).abs().amax(-1, keepdim=True)
    power = (((most.view(torch.int32) + 0x1FFFFF) >> 23) - 135).clamp(-117, 119)  # the least with most <= 448 * 2^power
    codes = torch.where(fine, x * (127 - power << 23).view(torch.float32), 0.0).to(torch.float8_e4m3fn)
    scale = torch.where(fine, (127 + power << 23).view(torch.float32), torch.nan)
    rows[:, :rank], rows[:, rank:rank + k_rope.shape[1]] = codes.view(torch.uint8), k_rope
    rows[:, rank + k_rope.shape[1]:rank + k_rope.shape[1] + 4] = scale.view(torch.uint8)


def _read(rows, case):
    """rows [n, bytes] -> latent [n, R], k_rope [n, P] in fp32."""
    rank, rope = case["rank"], case["rope"]
    if case["store"] == "bf16":
        both = rows[:, :2 * (rank + rope)].contiguous().view(torch.bfloat16).float()
        return both[:, :rank], both[:, rank:]
    scale = rows[:, rank + 2 * rope:rank + 2 * rope + 4].contiguous().view(torch.float32)
    latent = rows[:, :rank].contiguous().view(torch.float8_e4m3fn).float() * scale
    return latent, rows[:, rank:rank + 2 * rope].contiguous().view(torch.bfloat16).float()


def _run_plain(s):
    case = s["case"]
    dtype = _DT[case["dtype"]]
    if case["kind"] == "head":
        y = torch.bmm(s["x"].float().transpose(0, 1).contiguous(), s["weight"].float().transpose(1, 2).contiguous())
        return y.transpose(0, 1).to(dtype).contiguous()
    if case["kind"] == "rope":
        return _plain_rope(s, case)
    if case["kind"] == "cache":
        valid = s["positions"] >= 0
        at = s["positions"].clamp(min=0).long()
        place = (s["page_table"].long().gather(1, at // case["page"]) * case["page"] + at % case["page"])[valid]
        flat = s["cache"].view(-1, s["cache"].shape[-1])
        rows = flat[place]
        _write(rows, s["latent"][valid], s["k_rope"][valid], case)
        flat[place] = rows
        out = []
        for x, values in zip((s["latent"], s["k_rope"]), _read(flat[place], case)):
            read = torch.zeros(x.shape, device=DEV)
            read[valid] = values
            out.append(read.to(dtype))
        return tuple(out)
    page, rank = case["page"], case["rank"]
    out = torch.empty(s["q_latent"].shape, device=DEV)
    for b, total in enumerate(_lengths(case)):
        rows = s["cache"][s["page_table"][b, :-(-total // page)].long()].flatten(0, 1)[:total]
        latent, k_rope = _read(rows, case)
        place = torch.arange(total, device=DEV)
        at = s["positions"][b].long()[:, None]
        if s["ancestors"] is None:
            seen = place <= at
        else:
            base = at - torch.arange(case["length"], device=DEV)[:, None]
            bit = (s["ancestors"][b][:, None] >> (place - base).clamp(0, 63)) & 1
            seen = (place < base) | ((place - base < case["length"]) & (bit == 1))
        score = s["q_latent"][b].float().flatten(0, 1) @ latent.t() + s["q_rope"][b].float().flatten(0, 1) @ k_rope.t()
        score = (score * s["scale"]).unflatten(0, (-1, case["heads"]))
        score = torch.where(seen[:, None], score, -torch.inf)
        weight = torch.exp(score - score.amax(-1, keepdim=True))
        weight = weight / weight.sum(-1, keepdim=True)
        out[b] = (weight.flatten(0, 1) @ latent).unflatten(0, (-1, case["heads"]))
    return out.to(dtype)


def _plain_rope(s, case):
    rope, dtype = case["rope"], _DT[case["dtype"]]
    valid = (s["positions"] >= 0)[..., None, None]
    angle = s["positions"].double()[..., None] * s["frequencies"]
    cos, sin = angle.cos()[:, :, None] * s["magnitude"], angle.sin()[:, :, None] * s["magnitude"]
    out = []
    for x in (s["q"], s["k"]):
        x = x.double()
        keep, turn = x[..., :x.shape[-1] - rope], x[..., x.shape[-1] - rope:]
        if case["interleaved"]:
            a, b = turn[..., 0::2], turn[..., 1::2]
            turn = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = turn[..., :rope // 2], turn[..., rope // 2:]
            turn = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        out.append(torch.where(valid, torch.cat([keep, turn], -1), 0.0).to(dtype))
    return tuple(out)


# --------------------------------------------------------------- float64, from the definitions


def _two(power):
    """2^power in float64, from its exponent bits (the device's pow and ldexp are not exact)."""
    return (power.long() + 1023 << 52).view(torch.float64)


def _e4m3_64(codes):
    """Codes (uint8) in float64: sign, four exponent bits (bias 7), three of mantissa."""
    exponent, mantissa = ((codes >> 3) & 15).double(), (codes & 7).double()
    size = torch.where(exponent == 0, mantissa * 2.0 ** -9, (8 + mantissa) * _two(exponent - 10))
    size = torch.where((codes & 127) == 127, torch.nan, size)
    return torch.where(codes >= 128, -size, size)


def _rows64(rows, case):
    """Latents and key parts of cached rows in float64."""
    rank, rope = case["rank"], case["rope"]
    first = rank if case["store"] == "e4m3" else 2 * rank
    words = rows[:, first:first + 2 * rope].contiguous().view(torch.bfloat16).double()
    if case["store"] == "bf16":
        return rows[:, :first].contiguous().view(torch.bfloat16).double(), words
    tail = rows[:, first + 2 * rope:first + 2 * rope + 4].contiguous().view(torch.float32).double()
    return _e4m3_64(rows[:, :rank]) * tail, words


def _nearest64(x, case):
    """Every latent of [n, R] at the nearest value of its row's grid, ties to the even one, in float64."""
    x = x.double()
    if case["store"] == "bf16":
        least, low = torch.full_like(x[:, :1], -133.0), 7  # 2^-133 is the least bfloat16
    else:
        most = x.abs().amax(-1, keepdim=True).clamp(min=1e-300)
        power = torch.ceil(torch.log2(most / 448))
        power = torch.where(448 * _two(power - 1) >= most, power - 1, power)  # the logarithm's rounding put right
        power = torch.where(448 * _two(power) < most, power + 1, power).clamp(-117, 119)
        least, low = power - 9, 3
    _, exponent = torch.frexp(x)
    step = _two(torch.maximum(exponent.double() - 1 - low, least))
    return torch.round(x / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "head":
        out = torch.empty(case["tokens"], case["heads"], s["weight"].shape[1], dtype=torch.float64, device=DEV)
        for h in range(case["heads"]):
            out[:, h] = s["x"][:, h].double() @ s["weight"][h].double().t()
        return out
    if case["kind"] == "cache":
        shown = (s["positions"] >= 0)[..., None]
        latent = _nearest64(s["latent"].reshape(-1, case["rank"]), case).view(s["latent"].shape)
        words = _nearest64(s["k_rope"].reshape(-1, case["rope"]), {**case, "store": "bf16"}).view(s["k_rope"].shape)
        return torch.where(shown, latent, 0.0), torch.where(shown, words, 0.0)
    if case["kind"] == "rope":
        rope, half = case["rope"], case["rope"] // 2
        frequencies, magnitude = _frequencies(case)
        turn = torch.outer(s["positions"].flatten().double(),
                           torch.tensor(frequencies, dtype=torch.float64, device=DEV)).view(*s["positions"].shape, 1, half)
        turn = torch.polar(torch.full_like(turn, magnitude), turn)
        result = []
        for x in (s["q"], s["k"]):
            y = x.double().clone()
            start = y.shape[-1] - rope
            first = slice(start, None, 2) if case["interleaved"] else slice(start, start + half)
            second = slice(start + 1, None, 2) if case["interleaved"] else slice(start + half, None)
            z = torch.complex(y[..., first], y[..., second]) * turn
            y[..., first], y[..., second] = z.real, z.imag
            y[s["positions"] < 0] = 0
            result.append(y)
        return tuple(result)
    # Attention: a sequence's rows laid end to end, one head at a time.
    out = torch.zeros(s["q_latent"].shape, dtype=torch.float64, device=DEV)
    for b, total in enumerate(_lengths(case)):
        table = s["page_table"][b, :(total + case["page"] - 1) // case["page"]].long()
        latent, words = _rows64(s["cache"][table].view(-1, s["cache"].shape[-1])[:total], case)
        hidden = torch.ones(case["length"], total, dtype=torch.bool, device=DEV)
        for i in range(case["length"]):
            at = total - case["length"] + i
            if s["ancestors"] is None:
                hidden[i, :at + 1] = False
            else:
                base, bits = at - i, int(s["ancestors"][b, i]) % 2 ** 64
                hidden[i, :base] = False
                hidden[i, base:] = torch.tensor([bits >> j & 1 == 0 for j in range(case["length"])], device=DEV)
        for h in range(case["heads"]):
            score = s["q_latent"][b, :, h].double() @ latent.t() + s["q_rope"][b, :, h].double() @ words.t()
            out[b, :, h] = torch.softmax((score * s["scale"]).masked_fill_(hidden, -math.inf), -1) @ latent
    return out


# --------------------------------------------------------------- the least work


def work(case):
    size = _SIZE[case["dtype"]]
    if case["kind"] == "head":
        m, h, k = case["tokens"], case["heads"], case["inner"] * case["rank"]
        return {"bytes": h * k * _SIZE[case["weights"]] + size * m * h * (case["inner"] + case["rank"]), "flops": 2.0 * m * h * k}
    length, rope = case["length"], case["rope"]
    if case["kind"] == "attn":
        totals, rank, heads = _lengths(case), case["rank"], case["heads"]
        if case["tree"]:  # an ancestor every four or five tokens back
            keys = sum((t - length) * length for t in totals) + len(totals) * sum(1 + i // 5 for i in range(length))
        else:
            keys = sum(t * length - length * (length - 1) // 2 for t in totals)
        row = rank + 2 * rope + 4 if case["store"] == "e4m3" else 2 * (rank + rope)
        return {"bytes": sum(totals) * row + size * len(totals) * length * heads * (2 * rank + rope),
                "flops": 2.0 * (2 * rank + rope) * heads * keys}
    tokens, real = case["batch"] * length, sum(_real(case))
    if case["kind"] == "cache":
        return {"bytes": size * (case["rank"] + rope) * (real + tokens) + 2 * real * _row_bytes(case),
                "flops": 4.0 * real * case["rank"]}
    heads = case["heads"] + case["kv_heads"]
    return {"bytes": size * heads * case["head_dim"] * (real + tokens) + 4 * tokens, "flops": 3.0 * real * heads * rope}

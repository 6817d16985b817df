"""The 4-bit cache on the GPU: what is written and read back exactly, and attention over it against float64."""

from __future__ import annotations

import pytest
import torch

import kv4_reference as ref

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _c():
    from montlok import _C

    return _C


def _same(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a[~torch.isnan(a)], b[~torch.isnan(b)])


# ------------------------------------------------------------------ append and read


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,L,H,D,page,width", [(1, 1, 1, 32, 16, 1), (3, 5, 2, 64, 48, 3), (2, 130, 3, 128, 64, 4), (5, 1, 8, 128, 256, 2),
                                                (1, 37, 1, 256, 16, 5), (4, 33, 2, 32, 32, 2), (2, 70, 4, 64, 1024, 1)])
def test_append_then_read_is_the_nearest_grid_value(dev, dtype, B, L, H, D, page, width):
    """Bit for bit the definition's values; every other byte of the cache as it was."""
    g = torch.Generator().manual_seed(B * 1000 + L * 10 + D)
    pages = B * width + 2
    cache0 = ref.random_cache(g, pages, H, page, D)
    table = ref.random_table(g, B, width, pages)
    kv = (torch.randn(B, L, 2 * H, D, generator=g) * torch.exp(3 * torch.randn(B, L, 2 * H, 1, generator=g))).to(dtype)
    positions = torch.stack([torch.randperm(width * page, generator=g)[:L] for _ in range(B)]).to(torch.int32)
    positions[torch.rand(B, L, generator=g) < 0.15] = -1
    cache = cache0.to(dev)
    d = kv.to(dev)
    _c().kv4_append(d[:, :, :H], d[:, :, H:], cache, table.to(dev), positions.to(dev))
    k, v = _c().kv4_read(cache, table.to(dev), positions.to(dev), D, dtype)
    shown = (positions >= 0)[..., None, None]
    for got, x in ((k, kv[:, :, :H]), (v, kv[:, :, H:])):
        assert got.dtype == dtype and _same(got, torch.where(shown, ref.nearest(x), 0.0))
    # Where the bytes lie: the layout's own views, and nothing else touched.
    keys, values = ref.contents(cache, page, D)
    keys0, values0 = ref.contents(cache0, page, D)
    for b in range(B):
        for i in range(L):
            at = int(positions[b, i])
            if at >= 0:
                p, o = int(table[b, at // page]), at % page
                assert _same(keys[p, :, o], k[b, i]) and _same(values[p, :, o], v[b, i])
                keys[p, :, o], values[p, :, o] = keys0[p, :, o], values0[p, :, o]
    assert torch.equal(keys, keys0) and torch.equal(values, values0)


def test_rounding_at_every_border(dev):
    """Values on, next to and between the grid's borders, at scales from the smallest to the largest, and both signs."""
    sizes = torch.tensor([0, 0.25, 0.5, 0.75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6])
    near = torch.cat([sizes, torch.nextafter(sizes, torch.tensor(0.0)), torch.nextafter(sizes, torch.tensor(7.0))])
    near = near[near <= 6][:31 * (len(near[near <= 6]) // 31) or None]
    rows = []
    for e in (-126, -125, -124, -60, -1, 0, 1, 60, 124):
        x = near * 2.0 ** e
        for start in range(0, len(x), 31):
            row = torch.zeros(32)
            part = x[start:start + 31]
            row[:len(part)] = part
            row[31] = 6 * 2.0 ** e  # the group's largest
            rows += [row, -row]
    biggest = torch.full((32,), 3.4e38)  # above 6 * 2^125: saturates
    tiny = torch.full((32,), 1e-44)
    x = torch.stack(rows + [biggest, -biggest, tiny, torch.zeros(32), -torch.zeros(32)])[None, :, None]
    n = x.shape[1]
    table = torch.arange(-(-n // 16), dtype=torch.int32)[None].to(dev)
    positions = torch.arange(n, dtype=torch.int32)[None].to(dev)
    cache = _c().kv4_cache(table.shape[1], 1, 16, 32, dev)
    _c().kv4_append(x.to(dev), x.to(dev), cache, table, positions)
    for got in _c().kv4_read(cache, table, positions, 32):
        assert torch.equal(got.double().cpu(), ref.nearest(x))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_non_finite_groups_become_nan_alone(dev, dtype):
    x = torch.randn(1, 4, 2, 128, generator=torch.Generator().manual_seed(1)).to(dtype)
    x[0, 0, 0, 5], x[0, 1, 1, 64], x[0, 2, 0, 127], x[0, 3, 1, 32] = torch.nan, torch.inf, -torch.inf, torch.nan
    table, positions = torch.zeros(1, 1, dtype=torch.int32, device=dev), torch.arange(4, dtype=torch.int32, device=dev)[None]
    cache = _c().kv4_cache(1, 2, 16, 128, dev)
    _c().kv4_append(x.to(dev), x.to(dev), cache, table, positions)
    for got in _c().kv4_read(cache, table, positions, 128, dtype):
        assert _same(got, ref.nearest(x)) and int(torch.isnan(got).sum()) == 4 * 32


def test_tokens_without_a_page_are_dropped_and_read_as_nan(dev):
    """Pages outside the cache, positions past the table: nothing is written for them, NaN is read."""
    g = torch.Generator().manual_seed(3)
    cache0 = ref.random_cache(g, 4, 2, 16, 64)
    table = torch.tensor([[1, -1, 4], [2, 2 ** 31 - 1, -2 ** 31]], dtype=torch.int32)
    positions = torch.tensor([[0, 17, 32, 47, 48, 2 ** 31 - 1], [15, 16, 40, -1, -2 ** 31, 1000]], dtype=torch.int32)
    x = torch.randn(2, 6, 2, 64, generator=g)
    cache = cache0.to(dev)
    _c().kv4_append(x.to(dev), x.to(dev), cache, table.to(dev), positions.to(dev))
    k, v = _c().kv4_read(cache, table.to(dev), positions.to(dev), 64)
    expect = ref.nearest(x)
    expect[0, 1:] = torch.nan
    expect[1, 1:3], expect[1, 3:5], expect[1, 5] = torch.nan, 0, torch.nan
    assert _same(k, expect) and _same(v, expect)
    changed = (cache.cpu() != cache0).flatten(2).any(-1)
    assert not changed[0].any() and not changed[3].any()


# ------------------------------------------------------------------ attention


def _check(dev, g, B, L, H, Hkv, D, page, positions, dtype, scale=None, cache=None, table=None, q=None, spare=3):
    width = max(1, -(-(int(positions.max()) + 1) // page))
    pages = B * width + spare
    cache = ref.random_cache(g, pages, Hkv, page, D) if cache is None else cache
    table = ref.random_table(g, B, width, len(cache)) if table is None else table
    q = torch.randn(B, L, H, D, generator=g).to(dtype) if q is None else q
    scale = D ** -0.5 if scale is None else scale
    got = _c().kv4_attention(q.to(dev), cache.to(dev), table.to(dev), positions.to(dev), scale)
    keys, values = ref.contents(cache, page, D)
    out, size, spread = ref.attention(q, keys, values, table, positions, scale)
    assert got.shape == q.shape and got.dtype == dtype and got.is_contiguous()
    bound = ref.attention_bound(size, spread, out, int(positions.max()) + 1, D, dtype)
    _within(got, out, bound)
    return got


def _within(got, out, bound):
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(out))
    fine = ~torch.isnan(out)
    off = ((got - out).abs() / bound)[fine]
    assert not fine.any() or float(off.max()) <= 1.0, f"{float(off.max()):.3g} of the bound"


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("page", [16, 48, 64, 256])
def test_one_token_at_lengths_around_every_border(dev, dtype, D, page):
    """Sequences of 1 to 130 keys: the ends of runs, tiles and pages, an empty one among them."""
    at = torch.tensor([-1, 0, 1, 14, 15, 16, 31, 47, 48, 62, 63, 64, 65, 127, 128, 129], dtype=torch.int32)[:, None]
    _check(dev, torch.Generator().manual_seed(D + page), len(at), 1, 4, 2, D, page, at, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,Hkv", [(1, 1), (8, 8), (6, 2), (32, 8), (16, 1), (17, 1), (40, 1), (21, 3)])
@pytest.mark.parametrize("L", [1, 3, 40])
def test_heads_and_lengths(dev, dtype, H, Hkv, L):
    """Groups that do and do not divide a tile of rows; several tokens, causal among themselves."""
    g = torch.Generator().manual_seed(H * 100 + L)
    total = torch.tensor([L, 100, 77 + L])
    positions = (total[:, None] - L + torch.arange(L)).to(torch.int32)
    _check(dev, g, 3, L, H, Hkv, 64, 32, positions, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D,page,lengths", [(128, 64, [3000, 1, 700]), (64, 16, [2100, 64, 63]), (32, 32, [5000, 4999, 0]), (256, 256, [1500, 257, 256])])
def test_long_sequences_split_over_the_chip(dev, dtype, D, page, lengths):
    lib = _c().library()
    width = -(-max(lengths) // page)
    assert lib.mlk_kv4_attention_workspace_bytes(3, 1, 8, 2, D, page, width) > 0
    positions = torch.tensor(lengths, dtype=torch.int32)[:, None] - 1
    _check(dev, torch.Generator().manual_seed(D), 3, 1, 8, 2, D, page, positions, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_a_chunk_of_tokens(dev, dtype, D):
    """Many rows a key head: every tile of rows, the causal edge inside tiles of keys, positions in no order, padding."""
    g = torch.Generator().manual_seed(D + 1)
    B, L = 2, 150
    positions = torch.stack([torch.arange(L) + 201, torch.randperm(351, generator=g)[:L]]).to(torch.int32)
    positions[0, 120:] = -1
    positions[1, ::7] = -5
    got = _check(dev, g, B, L, 6, 2, D, 48, positions, dtype)
    assert not got[0, 120:].any() and not got[1, ::7].any()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_that_see_nothing_are_zero(dev, dtype):
    cache = torch.full((2, 2, 16 * 34), 255, dtype=torch.uint8, device=dev)  # NaN everywhere
    q = torch.randn(2, 3, 4, 32, device=dev).to(dtype)
    table, positions = torch.full((2, 1), -1, dtype=torch.int32, device=dev), torch.full((2, 3), -1, dtype=torch.int32, device=dev)
    assert not _c().kv4_attention(q, cache, table, positions, 1.0).any()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D,page", [(32, 16), (64, 48), (128, 64), (256, 128)])
@pytest.mark.parametrize("L", [1, 30])
def test_what_lies_behind_a_position_does_not_reach_it(dev, dtype, D, page, L):
    """NaN codes behind every row's own position, in the same tile as keys it sees: the same bits as without them."""
    g = torch.Generator().manual_seed(D + L)
    total = torch.tensor([L, 71, 64, 333])[:4]
    total = torch.maximum(total, torch.tensor(L))
    positions = (total[:, None] - L + torch.arange(L)).to(torch.int32)
    positions[3, 0] = 20  # a row that sees far less than the others
    width = -(-int(total.max()) // page)
    cache = ref.random_cache(g, 4 * width + 1, 2, page, D)
    table = ref.random_table(g, 4, width, len(cache))
    q = torch.randn(4, L, 6, D, generator=g).to(dtype)
    first = _check(dev, g, 4, L, 6, 2, D, page, positions, dtype, cache=cache, table=table, q=q)
    dirty = cache.clone()
    kc, vc, ks, vs = ref.parts(dirty, page, D)
    used = torch.zeros(len(cache), page, dtype=torch.bool)
    for b in range(4):
        for t in range(int(positions[b].max()) + 1):
            used[table[b, t // page].long(), t % page] = True
    ks.copy_(torch.where(used[:, None, :, None], ks, torch.tensor(255, dtype=torch.uint8)))
    vs.copy_(torch.where(used[:, None, None, :], vs, torch.tensor(255, dtype=torch.uint8)))
    second = _c().kv4_attention(q.to(dev), dirty.to(dev), table.to(dev), positions.to(dev), D ** -0.5)
    assert torch.equal(first, second)
    junk = table.clone()  # pages that no token needs may be anything
    for b in range(4):
        junk[b, int(positions[b].max()) // page + 1:] = torch.tensor([-7, 2 ** 30, len(cache)])[b % 3]
    assert torch.equal(first, _c().kv4_attention(q.to(dev), dirty.to(dev), junk.to(dev), positions.to(dev), D ** -0.5))
    # NaN at a token that some rows see and others do not.
    if L > 1:
        at = int(positions[1, 10])
        ks[table[1, at // page].long(), 0, at % page, 0] = 255
        vs[table[2, int(positions[2, 7]) // page].long(), 1, D // 32 - 1, int(positions[2, 7]) % page] = 255
        got = _c().kv4_attention(q.to(dev), dirty.to(dev), table.to(dev), positions.to(dev), D ** -0.5)
        nan = torch.zeros(got.shape, dtype=torch.bool)
        nan[1, 10:, :3] = True
        nan[2, 7:, 3:, D - 32:] = True
        assert torch.equal(torch.isnan(got).cpu(), nan)
        assert torch.equal(got.cpu()[~nan], first.cpu()[~nan])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_without_their_pages_are_nan_alone(dev, dtype):
    """A page outside the cache, or a position past the page table: NaN for the rows that need it, no other row changes."""
    g = torch.Generator().manual_seed(11)
    page, D, L = 32, 64, 5
    cache = ref.random_cache(g, 20, 2, page, D)
    positions = torch.tensor([[10, 40, 70, 100, 159], [5, 31, 32, 63, 64], [160, 1000, 2 ** 31 - 1, 12, -1]], dtype=torch.int32)
    table = ref.random_table(g, 3, 5, 20)
    table[0, 3], table[1, 1] = -1, 20
    q = torch.randn(3, L, 4, D, generator=g).to(dtype)
    got = _c().kv4_attention(q.to(dev), cache.to(dev), table.to(dev), positions.to(dev), 0.125)
    keys, values = ref.contents(cache, page, D)
    out, size, spread = ref.attention(q, keys, values, table, positions, 0.125)
    assert torch.isnan(out[0, 3:]).all() and torch.isnan(out[1, 2:]).all() and torch.isnan(out[2, :3]).all()
    _within(got, out, ref.attention_bound(size, spread, out, 160, D, dtype))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_sharp_and_flat_softmax(dev, dtype):
    """Scores of hundreds (one key takes all), a scale of 0 (the mean) and a negative one."""
    g = torch.Generator().manual_seed(13)
    positions = torch.tensor([[200], [63], [64]], dtype=torch.int32)
    for scale in (8.0, 0.0, -0.3):
        _check(dev, g, 3, 1, 4, 2, 64, 32, positions, dtype, scale=scale)


def test_strided_queries(dev):
    """q as a view of one projection's rows, rows of odd alignment among them: the same bits as a copy."""
    g = torch.Generator().manual_seed(17)
    cache, table = ref.random_cache(g, 8, 2, 32, 64).to(dev), torch.arange(8, dtype=torch.int32).view(2, 4).to(dev)
    positions = torch.tensor([[99, 100, 101], [3, 4, 5]], dtype=torch.int32, device=dev)
    for dtype in (F32, BF16):
        wide = torch.randn(2, 3, 4, 67, generator=g).to(dtype).to(dev)
        q = wide[..., 1:65]
        assert torch.equal(_c().kv4_attention(q, cache, table, positions, 0.1), _c().kv4_attention(q.contiguous(), cache, table, positions, 0.1))
        turned = q.transpose(0, 1).contiguous().transpose(0, 1)
        assert torch.equal(_c().kv4_attention(turned, cache, table, positions, 0.1), _c().kv4_attention(q.contiguous(), cache, table, positions, 0.1))
        # A table and positions that are views.
        t2 = torch.stack([table, table], -1)[..., 0]
        p2 = positions.t().contiguous().t()
        assert torch.equal(_c().kv4_attention(q, cache, t2, p2, 0.1), _c().kv4_attention(q, cache, table, positions, 0.1))


def test_offsets_past_32_bits(dev):
    """A cache of more than 4 GiB, the sequence on its last pages."""
    page, H, D = 256, 8, 128
    record = H * page * (D + D // 16)
    pages = (1 << 32) // record + 40
    cache = _c().kv4_cache(pages, H, page, D, dev)
    assert cache.numel() > 1 << 32
    table = torch.arange(pages - 1, pages - 5, -1, dtype=torch.int32, device=dev)[None]
    g = torch.Generator().manual_seed(19)
    n = 4 * page
    k, v = torch.randn(1, n, H, D, generator=g), torch.randn(1, n, H, D, generator=g)
    positions = torch.arange(n, dtype=torch.int32, device=dev)[None]
    _c().kv4_append(k.to(dev), v.to(dev), cache, table, positions)
    rk, rv = _c().kv4_read(cache, table, positions, D)
    assert torch.equal(rk.double().cpu(), ref.nearest(k)) and torch.equal(rv.double().cpu(), ref.nearest(v))
    q = torch.randn(1, 1, 16, D, generator=g)
    got = _c().kv4_attention(q.to(dev), cache, table, positions[:, -1:].contiguous(), 0.1)
    keys = ref.nearest(k)[0].transpose(0, 1)[None]
    values = ref.nearest(v)[0].transpose(0, 1)[None]
    out, size, spread = ref.attention(q, keys, values, torch.zeros(1, 1, dtype=torch.int32), torch.tensor([[n - 1]]), 0.1)
    _within(got, out, ref.attention_bound(size, spread, out, n, D, F32))


def test_no_tokens(dev):
    cache, table = _c().kv4_cache(1, 2, 16, 32, dev), torch.zeros(0, 1, dtype=torch.int32, device=dev)
    empty = torch.zeros(0, 1, dtype=torch.int32, device=dev)
    x = torch.zeros(0, 1, 2, 32, device=dev)
    assert _c().kv4_attention(x, cache, table, empty, 1.0).shape == x.shape
    _c().kv4_append(x, x, cache, table, empty)
    assert _c().kv4_read(cache, table, empty, 32)[0].shape == x.shape
    none = torch.zeros(1, 0, dtype=torch.int32, device=dev)
    assert _c().kv4_attention(torch.zeros(1, 0, 4, 32, device=dev), cache, none.new_zeros(1, 1), none, 1.0).shape == (1, 0, 4, 32)


def test_refusals(dev):
    c = _c()
    cache, table, at = c.kv4_cache(2, 2, 16, 32, dev), torch.zeros(1, 1, dtype=torch.int32, device=dev), torch.zeros(1, 1, dtype=torch.int32, device=dev)
    x, q = torch.zeros(1, 1, 2, 32, device=dev), torch.zeros(1, 1, 4, 32, device=dev)
    for call, text in (
            (lambda: c.kv4_append(x.half(), x, cache, table, at), "k must be float32 or bfloat16"),
            (lambda: c.kv4_append(x, x.bfloat16(), cache, table, at), "v must be of k's dtype"),
            (lambda: c.kv4_append(x, x[..., :1], cache, table, at), "k and v must be"),
            (lambda: c.kv4_append(x[0], x[0], cache, table, at), "k must have 4 dimensions"),
            (lambda: c.kv4_append(x.expand(1, 1, 2, 32).transpose(2, 3).contiguous().transpose(2, 3), x, cache, table, at), "dense along"),
            (lambda: c.kv4_append(q, q, cache, table, at), "cache holds 2 key heads, expected 4"),
            (lambda: c.kv4_append(x, x, cache.int(), table, at), "cache must be uint8"),
            (lambda: c.kv4_append(x, x, cache[..., 1:], table, at), "cache must be contiguous"),
            (lambda: c.kv4_append(x, x, cache[:, :, :100].contiguous(), table, at), "cache records must be"),
            (lambda: c.kv4_append(x, x, cache[:, :, :34].contiguous(), table, at), "page_size must be a multiple of 16"),
            (lambda: c.kv4_append(x, x, cache, table.long(), at), "page_table must be int32"),
            (lambda: c.kv4_append(x, x, cache, table, at.long()), "positions must be int32"),
            (lambda: c.kv4_append(x, x, cache, table[0], at), "page_table must have 2 dimensions"),
            (lambda: c.kv4_append(x, x, cache, table.expand(2, 1), at), "page_table must have a row for each sequence"),
            (lambda: c.kv4_append(x, x, cache, table, at.expand(1, 2)), r"positions must be \[batch, length\]"),
            (lambda: c.kv4_append(x, x, cache, table.cpu(), at), "page_table must be on the same GPU"),
            (lambda: c.kv4_attention(x[:, :, :1], cache, table, at, 1.0), "multiple of the cache's"),
            (lambda: c.kv4_attention(q[..., :16], cache, table, at, 1.0), "head_dim must be"),
            (lambda: c.kv4_attention(q, cache, table[:, :0], at, 1.0), "page_table must hold"),
            (lambda: c.kv4_attention(q, cache[:0], table, at, 1.0), "between 1 and"),
            (lambda: c.kv4_read(cache, table, at, 48), "head_dim must be"),
            (lambda: c.kv4_read(cache, table, at, 64), "page_size must be a multiple of 16")):
        with pytest.raises(RuntimeError, match=text):
            call()


# ------------------------------------------------------------------ streams and graphs


def test_other_streams_and_two_at_once(dev):
    """Calls with workspaces on two streams at a time, each against its own result alone."""
    g = torch.Generator().manual_seed(23)
    sets = []
    for seed in (1, 2):
        cache, table = ref.random_cache(g, 64, 2, 64, 128).to(dev), torch.randperm(64, generator=g).view(1, 64).to(torch.int32).to(dev)
        q, at = torch.randn(1, 1, 8, 128, generator=g).to(dev), torch.tensor([[4000 + seed]], dtype=torch.int32, device=dev)
        sets.append((q, cache, table, at, 0.09))
    expect = [_c().kv4_attention(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    results = [[], []]
    for _ in range(20):
        for s, stream, out in zip(sets, streams, results):
            with torch.cuda.stream(stream):
                out.append(_c().kv4_attention(*s))
    torch.cuda.synchronize()
    assert all(torch.equal(r, e) for out, e in zip(results, expect) for r in out)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_decode_step_in_a_graph(dev, dtype):
    """Norm, append and attention of one token captured once and replayed as positions advance, each replay against eager
    calls on a copy; two graphs of different lengths side by side."""
    c = _c()
    g = torch.Generator().manual_seed(29)
    B, H, Hkv, D, page, width = 3, 8, 2, 64, 16, 40
    weight = (1 + 0.1 * torch.randn(D, generator=g)).to(dev)
    angle = torch.arange(page * width)[:, None] * 10000.0 ** (-torch.arange(0, D, 2) / D)
    cos, sin = torch.cat([angle, angle], 1).cos().to(dev), torch.cat([angle, angle], 1).sin().to(dev)
    table = torch.randperm(B * width, generator=g).view(B, width).to(torch.int32).to(dev)

    def step(x, cache, at):
        q, k = c.qk_norm_rope(x[:, :, :H], x[:, :, H:H + Hkv], weight, weight, 1e-5, cos, sin, at)
        c.kv4_append(k, x[:, :, H + Hkv:], cache, table, at)
        return c.kv4_attention(q, cache, table, at, D ** -0.5)

    start = ref.random_cache(g, B * width, Hkv, page, D).to(dev)
    graphs = []
    for first in (250, 7):
        x = torch.randn(B, 1, H + 2 * Hkv, D, generator=g).to(dtype).to(dev)
        at = torch.tensor([[first], [first + 300], [first + 100]], dtype=torch.int32, device=dev)
        cache = start.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(x, start.clone(), at)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(x, cache, at)
        graphs.append((graph, x, at, cache, out, start.clone()))
    for replay in range(5):
        for graph, x, at, cache, out, eager in graphs:
            x.copy_(torch.randn(x.shape, generator=g).to(dtype))
            at += 1
            out.fill_(float("nan"))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            expect = step(x, eager, at)
            assert torch.equal(out, expect) and torch.equal(cache, eager), f"replay {replay}"


def test_a_prompt_then_tokens_equals_the_sequence(dev):
    """A prompt in chunks, then token by token, over padded sequences: as they would be used together, each new row
    against float64 attention over the rounded keys and values of its sequence."""
    c = _c()
    g = torch.Generator().manual_seed(31)
    B, H, Hkv, D, page, total = 3, 4, 2, 32, 16, 90
    lengths = [90, 61, 17]
    table = torch.randperm(B * 6, generator=g).view(B, 6).to(torch.int32)
    cache = c.kv4_cache(B * 6, Hkv, page, D, dev)
    q, k, v = torch.randn(B, total, H, D, generator=g), torch.randn(B, total, Hkv, D, generator=g), torch.randn(B, total, Hkv, D, generator=g)
    got = torch.zeros(B, total, H, D)
    for begin, end in [(0, 40), (40, 80)] + [(i, i + 1) for i in range(80, 90)]:
        at = torch.tensor([[i if i < n else -1 for i in range(begin, end)] for n in lengths], dtype=torch.int32).to(dev)
        c.kv4_append(k[:, begin:end].to(dev), v[:, begin:end].to(dev), cache, table.to(dev), at)
        got[:, begin:end] = c.kv4_attention(q[:, begin:end].to(dev), cache, table.to(dev), at, D ** -0.5).cpu()
    for b, n in enumerate(lengths):
        keys, values = ref.nearest(k[b, :n]).transpose(0, 1)[None], ref.nearest(v[b, :n]).transpose(0, 1)[None]
        out, size, spread = ref.attention(q[b:b + 1, :n], keys, values, torch.zeros(1, 1, dtype=torch.int32), torch.arange(n)[None], D ** -0.5)
        _within(got[b:b + 1, :n], out, ref.attention_bound(size, spread, out, n, D, F32))
        assert not got[b, n:].any()


# ------------------------------------------------------------------ many rows: waves that share the keys


def _wide(table, width):
    """The same table with more room than any sequence needs, as a server allots it."""
    return torch.cat([table, torch.full((len(table), width - table.shape[1]), -1, dtype=torch.int32)], 1)


def _shared_case(g, B, L, H, Hkv, page, room, dtype):
    """A chunk of each of B sequences, causal, among them padding, rows in no order and a row at the start; the page table
    of `room` tokens a sequence, most of it unused."""
    positions = torch.stack([torch.arange(L) + 37 * b + (b % 3) * 130 for b in range(B)]).to(torch.int32)
    positions[0] = positions[0][torch.randperm(L, generator=g)]
    positions[B - 1, L // 2:] = -1
    positions[0, 3] = 0
    width = -(-(int(positions.max()) + 1) // page)
    cache = ref.random_cache(g, B * width + 1, Hkv, page, 128)
    table = ref.random_table(g, B, width, len(cache))
    return torch.randn(B, L, H, 128, generator=g).to(dtype), cache, table, _wide(table, max(width, room // page)), positions


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,L,H,Hkv,page,room", [(2, 150, 6, 2, 48, 48 * 350), (2, 150, 6, 2, 64, 1 << 14), (1, 140, 1, 1, 16, 1 << 17),
                                                 (3, 17, 40, 4, 1024, 1 << 14), (32, 33, 32, 8, 64, 1024), (2, 70, 16, 1, 32, 1 << 15)])
def test_waves_that_share_the_keys(dev, dtype, B, L, H, Hkv, page, room):
    g = torch.Generator().manual_seed(B * L + page)
    q, cache, table, wide, positions = _shared_case(g, B, L, H, Hkv, page, room, dtype)
    rows = L * H // Hkv
    assert rows >= 128 and B * Hkv * -(-rows // 256) * (wide.shape[1] * page // 64) >= 2048  # what takes this form
    got = _c().kv4_attention(q.to(dev), cache.to(dev), wide.to(dev), positions.to(dev), 0.09)
    keys, values = ref.contents(cache, page, 128)
    out, size, spread = ref.attention(q, keys, values, table, positions, 0.09)
    _within(got, out, ref.attention_bound(size, spread, out, int(positions.max()) + 1, 128, dtype))
    assert not got[B - 1, L // 2:].any()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_shared_keys_nan_and_missing_pages(dev, dtype):
    """As for the other form: what lies behind a row's position does not reach it, NaN reaches the rows that see it and the
    elements it belongs to, a missing page the rows that need it."""
    g = torch.Generator().manual_seed(41)
    page, D = 48, 128
    q, cache, table, wide, positions = _shared_case(g, 2, 150, 6, 2, page, 48 * 350, dtype)
    call = lambda c, t: _c().kv4_attention(q.to(dev), c.to(dev), t.to(dev), positions.to(dev), 0.09).cpu()
    first = call(cache, wide)
    dirty = cache.clone()
    kc, vc, ks, vs = ref.parts(dirty, page, D)
    used = torch.zeros(len(cache), page, dtype=torch.bool)
    for b in range(2):
        for t in range(int(positions[b].max()) + 1):
            used[table[b, t // page].long(), t % page] = True
    ks.copy_(torch.where(used[:, None, :, None], ks, torch.tensor(255, dtype=torch.uint8)))
    vs.copy_(torch.where(used[:, None, None, :], vs, torch.tensor(255, dtype=torch.uint8)))
    junk = wide.clone()
    junk[:, table.shape[1]:] = torch.tensor([-3, 2 ** 30], dtype=torch.int32)[:, None]
    assert torch.equal(call(dirty, junk), first)
    place = lambda b, t: (table[b, t // page].long(), t % page)
    p, o = place(0, 70)
    ks[p, 0, o, 3] = 255
    p, o = place(1, 180)
    vs[p, 1, 1, o] = 255
    got = call(dirty, wide)
    nan = torch.zeros(got.shape, dtype=torch.bool)
    nan[0, :, :3] = (positions[0] >= 70)[:, None, None]
    nan[1, :, 3:, 32:64] = (positions[1] >= 180)[:, None, None]
    assert torch.equal(torch.isnan(got), nan) and torch.equal(got[~nan], first[~nan])
    gone = wide.clone()
    gone[0, 2], gone[1, 3] = -1, len(cache)
    got = call(cache, gone)
    nan = torch.zeros(got.shape, dtype=torch.bool)
    nan[0] = (positions[0] >= 2 * page)[:, None, None]
    nan[1] = (positions[1] >= 3 * page)[:, None, None]
    assert torch.equal(torch.isnan(got), nan) and torch.equal(got[~nan], first[~nan])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("scale", [3.0, 0.0, -0.2])
def test_shared_keys_at_other_scales(dev, dtype, scale):
    g = torch.Generator().manual_seed(43)
    q, cache, table, wide, positions = _shared_case(g, 1, 140, 2, 1, 64, 1 << 16, dtype)
    strided = torch.empty(1, 140, 2, 131, dtype=dtype)[..., 1:129].copy_(q)
    got = _c().kv4_attention(strided.to(dev), cache.to(dev), wide.to(dev), positions.to(dev), scale)
    keys, values = ref.contents(cache, 64, 128)
    out, size, spread = ref.attention(q, keys, values, table, positions, scale)
    _within(got, out, ref.attention_bound(size, spread, out, int(positions.max()) + 1, 128, dtype))


# ------------------------------------------------------------------ scale bytes whose values leave bf16


def _junk(g, cache, page, D, used):
    """The cache with any bytes at the places [pages, page] that no token needs: every scale byte, half of them 253 and 254,
    whose larger codes stand for 2^128 and more."""
    dirty = cache.clone()
    any_byte = lambda t: torch.randint(0, 256, t.shape, generator=g, dtype=torch.uint8)
    kc, vc, ks, vs = ref.parts(dirty, page, D)
    for codes, scales, place in ((kc, ks, used[:, None, :, None]), (vc, vs, used[:, None, None, :])):
        codes.copy_(torch.where(place, codes, any_byte(codes)))
        huge = torch.randint(253, 255, scales.shape, generator=g, dtype=torch.uint8)
        scales.copy_(torch.where(place, scales, torch.where(torch.rand(scales.shape, generator=g) < 0.5, huge, any_byte(scales))))
    return dirty


def _places(table, positions, pages, page):
    used = torch.zeros(pages, page, dtype=torch.bool)
    for b in range(len(table)):
        for t in range(int(positions[b].max()) + 1):
            used[table[b, t // page].long(), t % page] = True
    return used


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D,page", [(32, 16), (32, 64), (64, 48), (64, 128), (128, 32), (128, 64), (256, 128)])
@pytest.mark.parametrize("L", [1, 30])
def test_any_bytes_behind_a_position_do_not_reach_it(dev, dtype, D, page, L):
    g = torch.Generator().manual_seed(3 * D + L)
    total = torch.tensor([max(L, 1), 71, 64, 333, 130])
    positions = (total[:, None] - L + torch.arange(L)).to(torch.int32)
    positions[3, 0] = 20
    width = -(-int(total.max()) // page)
    cache = ref.random_cache(g, 5 * width + 1, 2, page, D)
    table = ref.random_table(g, 5, width, len(cache))
    q = torch.randn(5, L, 6, D, generator=g).to(dtype)
    first = _check(dev, g, 5, L, 6, 2, D, page, positions, dtype, cache=cache, table=table, q=q)
    dirty = _junk(g, cache, page, D, _places(table, positions, len(cache), page))
    assert torch.equal(first, _c().kv4_attention(q.to(dev), dirty.to(dev), table.to(dev), positions.to(dev), D ** -0.5))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("page,room", [(48, 48 * 350), (64, 1 << 14)])
def test_shared_keys_any_bytes_behind_a_position(dev, dtype, page, room):
    """The same for the waves that share the keys."""
    g = torch.Generator().manual_seed(page)
    q, cache, table, wide, positions = _shared_case(g, 2, 150, 6, 2, page, room, dtype)
    dirty = _junk(g, cache, page, 128, _places(table, positions, len(cache), page))
    call = lambda c: _c().kv4_attention(q.to(dev), c.to(dev), wide.to(dev), positions.to(dev), 0.09)
    first = call(cache)
    assert torch.isfinite(first).all() and torch.equal(first, call(dirty))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,L,D,page,room", [(1, 1, 64, 16, 0), (1, 3, 128, 32, 0), (1, 70, 128, 48, 48 * 1500), (1, 70, 32, 16, 0)])
def test_a_missing_page_reaches_only_the_rows_that_need_it(dev, dtype, B, L, D, page, room):
    """Whatever the cache's first page holds: in a tile of keys of which one page is missing, the rows before it keep their
    bits, beside rows that need it."""
    g = torch.Generator().manual_seed(L + D)
    width = 4
    cache = ref.random_cache(g, 9, 2, page, D)
    table = torch.tensor([[5, 3, 7, 2]], dtype=torch.int32)
    positions = torch.arange(page // 2, page // 2 + L, dtype=torch.int32)[None]  # the first page, the second of long chunks
    q = torch.randn(B, L, 8, D, generator=g).to(dtype)
    wide = _wide(table, max(width, room // page))
    call = lambda c, t: _c().kv4_attention(q.to(dev), c.to(dev), t.to(dev), positions.to(dev), D ** -0.5).cpu()
    first = call(cache, wide)
    dirty = cache.clone()
    kc, vc, ks, vs = ref.parts(dirty, page, D)
    kc[0], vc[0], ks[0], vs[0] = 0x77, 0x77, 254, 254
    gone = wide.clone()
    gone[0, 1:4] = torch.tensor([-1, 9, 2 ** 30], dtype=torch.int32)
    got = call(dirty, gone)
    nan = torch.zeros(got.shape, dtype=torch.bool)
    nan[0] = (positions[0] >= page)[:, None, None]
    assert torch.equal(torch.isnan(got), nan) and torch.equal(got[~nan], first[~nan])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("room", [0, 1 << 17])
def test_huge_values_reach_only_the_rows_that_see_them(dev, dtype, room):
    """A value under byte 254 in a tile that some rows do not see whole: the rows before it and the other groups of 32 keep
    their bits, in both forms."""
    g = torch.Generator().manual_seed(53)
    page, D, L = 64, 128, 70
    cache = ref.random_cache(g, 4, 1, page, D)
    table = torch.tensor([[2, 0, 3]], dtype=torch.int32)
    positions = torch.arange(60, 60 + L, dtype=torch.int32)[None]
    q = torch.randn(1, L, 4, D, generator=g).to(dtype)
    wide = _wide(table, max(3, room // page))
    call = lambda c: _c().kv4_attention(q.to(dev), c.to(dev), wide.to(dev), positions.to(dev), 0.09).cpu()
    first = call(cache)
    kc, vc, ks, vs = ref.parts(cache, page, D)
    vs[0, 0, 1, 70 - page], vc[0, 0, 16:32, 70 - page] = 254, 0x77
    got = call(cache)
    sees = torch.zeros(got.shape, dtype=torch.bool)
    sees[0, :, :, 32:64] = (positions[0] >= 70)[:, None, None]
    assert torch.equal(got[~sees], first[~sees]) and not torch.isfinite(got[sees]).any()


# ------------------------------------------------------------------ the forms and splits that a call's sizes choose


def _splits(lib, B, L, H, Hkv, D, page, width):
    """Parts of a row, from the workspace's size."""
    return lib.mlk_kv4_attention_workspace_bytes(B, L, H, Hkv, D, page, width) // (4 * (D + 2) * B * L * H)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("page,L,H,Hkv", [(64, 7, 6, 2), (128, 1, 17, 1), (192, 2, 6, 2), (64, 1, 3, 1), (128, 1, 2, 1), (64, 40, 1, 1)])
def test_rows_on_pages_of_whole_tiles(dev, dtype, D, page, L, H, Hkv):
    g = torch.Generator().manual_seed(D + page + L)
    total = torch.tensor([L, 77, 64, 301, 129 + L]).clamp(min=L)
    positions = (total[:, None] - L + torch.arange(L)).to(torch.int32)
    positions[4, L // 2] = -1
    _check(dev, g, 5, L, H, Hkv, D, page, positions, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D,page,L,H,Hkv,length,splits", [(32, 64, 1, 4, 1, 9700, 19), (64, 48, 1, 8, 2, 9300, 19), (128, 64, 1, 4, 1, 10240, 20),
                                                          (256, 32, 1, 3, 1, 9001, 18), (32, 16, 5, 4, 1, 8711, 18), (64, 128, 3, 7, 1, 16001, 32),
                                                          (256, 256, 2, 6, 1, 16384, 32), (128, 16, 6, 6, 2, 20011, 20)])
def test_many_parts_that_all_hold_keys(dev, dtype, D, page, L, H, Hkv, length, splits):
    """More than 16 parts of every row, joined by groups of lanes; among the rows short ones, whose parts are mostly empty."""
    width = -(-length // page)
    assert _splits(_c().library(), 2, L, H, Hkv, D, page, width) == splits
    g = torch.Generator().manual_seed(length)
    positions = torch.stack([torch.arange(L) + length - L, torch.arange(L) * 613 % length]).to(torch.int32)
    _check(dev, g, 2, L, H, Hkv, D, page, positions, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_shared_keys_many_parts_that_all_hold_keys(dev, dtype):
    g = torch.Generator().manual_seed(59)
    page, D, L, H, Hkv, length, width = 64, 128, 16, 64, 8, 6000, 256
    assert _splits(_c().library(), 1, L, H, Hkv, D, page, width) == 32  # by strides of 32 tiles, 94 of them in use
    positions = (torch.arange(L) * 400).to(torch.int32)[None]
    positions[0, L - 1] = length - 1
    used = -(-length // page)
    cache, table = ref.random_cache(g, used, Hkv, page, D), ref.random_table(g, 1, used, used)
    q = torch.randn(1, L, H, D, generator=g).to(dtype)
    got = _c().kv4_attention(q.to(dev), cache.to(dev), _wide(table, width).to(dev), positions.to(dev), D ** -0.5)
    keys, values = ref.contents(cache, page, D)
    out, size, spread = ref.attention(q, keys, values, table, positions, D ** -0.5)
    _within(got, out, ref.attention_bound(size, spread, out, length, D, dtype))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_every_scale_byte_and_code_is_read_as_its_value(dev, dtype):
    """All 256 bytes under all 16 codes: exactly the value, an infinity from 2^128 on (bytes 253 and 254), NaN for 255."""
    page, D = 256, 32
    cache = torch.zeros(1, 1, page * (D + D // 16), dtype=torch.uint8)
    kc, vc, ks, vs = ref.parts(cache, page, D)
    kc[0, 0] = torch.arange(16, dtype=torch.uint8) * 16 + torch.arange(16, dtype=torch.uint8).flip(0)
    vc[0, 0] = kc[0, 0].t()
    ks[0, 0, :, 0] = vs[0, 0, 0] = torch.arange(256, dtype=torch.int32).to(torch.uint8)
    positions = torch.arange(page, dtype=torch.int32, device=dev)[None]
    keys, values = ref.contents(cache, page, D)
    assert torch.equal(keys.nan_to_num(nan=0.5), values.nan_to_num(nan=0.5))
    expect = torch.where(keys.abs() >= 2.0 ** 128, torch.sign(keys) * torch.inf, keys)[0, 0][None, :, None]
    assert int(torch.isinf(expect).sum()) == 8 + 16  # of 32 elements each: codes 6 and 7 under 253, 4 to 7 under 254
    for got in _c().kv4_read(cache.to(dev), torch.zeros(1, 1, dtype=torch.int32, device=dev), positions, D, dtype):
        assert _same(got, expect)

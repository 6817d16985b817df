"""latent_attention on the GPU against float64: formats, sizes, masks, trees, missing pages, bytes that no token sees."""

from __future__ import annotations

import pytest
import torch

import latent_reference as ref

pytestmark = pytest.mark.gpu

F32, BF16, E4M3 = torch.float32, torch.bfloat16, torch.float8_e4m3fn


def _c():
    from montlok import _C

    return _C


def _queries(g, B, L, H, rank, rope, dtype):
    return torch.randn(B, L, H, rank, generator=g).to(dtype), torch.randn(B, L, H, rope, generator=g).to(dtype)


def _within(got, out, bound):
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(out))
    fine = ~torch.isnan(out)
    off = ((got - out).abs() / bound)[fine]
    assert not fine.any() or float(off.max()) <= 1.0, f"{float(off.max()):.3g} of the bound"


def _check(dev, q, qr, cache, table, positions, store, scale=None, ancestors=None):
    rank, rope = q.shape[3], qr.shape[3]
    scale = (rank + rope) ** -0.5 if scale is None else scale
    got = _c().latent_attention(q.to(dev), qr.to(dev), cache.to(dev), table.to(dev), positions.to(dev), scale,
                                None if ancestors is None else ancestors.to(dev))
    out, size, spread = ref.attention(q, qr, cache, table, positions, scale, store, ancestors)
    assert got.shape == q.shape and got.dtype == q.dtype and got.is_contiguous()
    _within(got, out, ref.attention_bound(size, spread, out, max(1, int(positions.max()) + 1), rank + rope, q.dtype))
    return got


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("store", [E4M3, BF16])
@pytest.mark.parametrize("rank", [64, 128, 256, 512])
@pytest.mark.parametrize("rope", [16, 32, 64])
@pytest.mark.parametrize("H", [3, 24, 70])
def test_every_form(dev, dtype, store, rank, rope, H):
    """One token of two sequences over a short past, and five with a row of padding: every built form once."""
    g = torch.Generator().manual_seed(rank + rope + H)
    for L, lengths, page, width in ((1, (1, 200), 64, 4), (5, (67, 130), 24, 40)):
        table = ref.random_table(g, 2, width, 2 * width + 1)
        cache = ref.random_cache(g, 2 * width + 1, page, rank, rope, store)
        positions = torch.tensor([[n - L + i for i in range(L)] for n in lengths], dtype=torch.int32)
        if L > 1:
            positions[1, 3] = -1
        q, qr = _queries(g, 2, L, H, rank, rope, dtype)
        _check(dev, q, qr, cache, table, positions, store)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("store", [E4M3, BF16])
@pytest.mark.parametrize("B,L,H,rank,rope,page,lengths", [
    (1, 1, 1, 64, 16, 1, [1]), (1, 1, 16, 512, 64, 64, [63]), (1, 1, 16, 512, 64, 64, [64]), (1, 1, 17, 512, 64, 64, [65]),
    (3, 1, 8, 64, 16, 32, [480, 1, 129]), (2, 7, 12, 128, 32, 48, [7, 300]), (1, 1, 128, 512, 64, 256, [1000]),
    (1, 64, 5, 256, 64, 16, [64]), (2, 33, 16, 64, 32, 100, [33, 150]), (5, 1, 33, 256, 32, 7, [1, 2, 63, 128, 129]),
    (1, 100, 4, 64, 64, 1000, [613]), (1, 1, 4, 64, 16, 16, [5000])])
def test_sizes(dev, dtype, store, B, L, H, rank, rope, page, lengths):
    g = torch.Generator().manual_seed(sum(lengths) + H)
    width = -(-max(lengths) // page)
    table = ref.random_table(g, B, width, B * width + 2)
    cache = ref.random_cache(g, B * width + 2, page, rank, rope, store)
    positions = torch.tensor([[n - L + i for i in range(L)] for n in lengths], dtype=torch.int32)
    q, qr = _queries(g, B, L, H, rank, rope, dtype)
    _check(dev, q, qr, cache, table, positions, store)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("store", [E4M3, BF16])
@pytest.mark.parametrize("L,H,rank", [(1, 8, 64), (7, 16, 128), (48, 5, 256), (64, 3, 64), (63, 2, 512)])
def test_trees(dev, dtype, store, L, H, rank):
    """Random ancestors, words with bits of no token, a tree over no cached text, a padded token and one that sees nothing."""
    g = torch.Generator().manual_seed(L)
    B, page, width = 4, 20, 12
    table = ref.random_table(g, B, width, B * width)
    cache = ref.random_cache(g, B * width, page, rank, 16, store)
    base = [0, 1, 100, width * page - L]
    positions = torch.tensor([[n + i for i in range(L)] for n in base], dtype=torch.int32)
    ancestors = torch.randint(-2 ** 63, 2 ** 63 - 1, (B, L), generator=g)
    ancestors[0, 0] = 0
    ancestors[1] = -1
    if L > 2:
        positions[2, 1] = -1
    q, qr = _queries(g, B, L, H, rank, 16, dtype)
    got = _check(dev, q, qr, cache, table, positions, store, ancestors=ancestors)
    assert (got[0, 0] == 0).all()
    # A chain is the plain call.
    chain = torch.tensor([[min(2 ** (i + 1) - 1, 2 ** 63 - 1) if i < 63 else -1 for i in range(L)]] * B)
    scale = (rank + 16) ** -0.5
    args = (q.to(dev), qr.to(dev), cache.to(dev), table.to(dev), positions.to(dev), scale)
    assert torch.equal(_c().latent_attention(*args, chain.to(dev)), _c().latent_attention(*args))


@pytest.mark.parametrize("store", [E4M3, BF16])
def test_a_tree_at_places_before_the_sequence(dev, store):
    """Token i at a place below i: the tree would begin before the sequence, and what lies there is not seen."""
    g = torch.Generator().manual_seed(9)
    table, cache = ref.random_table(g, 1, 2, 2), ref.random_cache(g, 2, 16, 64, 16, store)
    positions = torch.tensor([[0, 0, 1, 5]], dtype=torch.int32)
    ancestors = torch.tensor([[1, 3, 7, 15]])
    q, qr = _queries(g, 1, 4, 2, 64, 16, F32)
    _check(dev, q, qr, cache, table, positions, store, ancestors=ancestors)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("store", [E4M3, BF16])
@pytest.mark.parametrize("rank,H", [(64, 4), (512, 16), (512, 64), (128, 40)])
def test_what_no_token_sees_does_not_reach_it(dev, dtype, store, rank, H):
    """Any bytes behind each token's position, in the same tile and page, and pages that only later tokens name."""
    g = torch.Generator().manual_seed(rank + H)
    page, width, L = 48, 5, 3
    table = ref.random_table(g, 2, width, 2 * width)
    cache = ref.random_cache(g, 2 * width, page, rank, 32, store)
    positions = torch.tensor([[30, 70, 71], [5, -1, 100]], dtype=torch.int32)
    q, qr = _queries(g, 2, L, H, rank, 32, dtype)
    clean = _check(dev, q, qr, cache, table, positions, store)
    for b, last in ((0, 71), (1, 100)):
        flat = cache[table[b].long()].flatten(0, 1)
        flat[last + 1:] = 255  # NaN in every format
        flat[last + 1::3] = torch.randint(0, 256, flat[last + 1::3].shape, generator=g, dtype=torch.uint8)
        cache[table[b].long()] = flat.view(width, page, -1)
    table[0, 2:], table[1, 3:] = -1, 2 ** 31 - 1
    assert torch.equal(_check(dev, q, qr, cache, table, positions, store), clean)
    # A row of no numbers between tokens of one call: those before it keep their results, those after it get NaN.
    row = cache[table[0, 1].item(), 50 - page]
    row[:] = 255
    got = _c().latent_attention(q.to(dev), qr.to(dev), cache.to(dev), table.to(dev), positions.to(dev), (rank + 32) ** -0.5)
    assert torch.equal(got[0, 0], clean[0, 0]) and torch.isnan(got[0, 1:]).all() and torch.equal(got[1], clean[1])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_an_infinite_latent_of_another_token(dev, dtype):
    """Bytes of infinities in a bf16 cache, seen by the later token only."""
    g = torch.Generator().manual_seed(3)
    cache, table = ref.random_cache(g, 1, 64, 64, 16, BF16), torch.zeros(1, 1, dtype=torch.int32)
    positions = torch.tensor([[9, 20]], dtype=torch.int32)
    q, qr = _queries(g, 1, 2, 4, 64, 16, dtype)
    clean = _check(dev, q, qr, cache, table, positions, BF16)
    cache[0, 15].view(BF16)[3] = torch.inf
    got = _c().latent_attention(q.to(dev), qr.to(dev), cache.to(dev), table.to(dev), positions.to(dev), 80 ** -0.5)
    assert torch.equal(got[0, 0], clean[0, 0])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_missing_pages_and_places_past_the_table(dev, dtype):
    g = torch.Generator().manual_seed(6)
    cache = ref.random_cache(g, 4, 16, 64, 16, E4M3)
    table = torch.tensor([[1, -1, 4, 0], [2, 3, 2 ** 31 - 1, -2 ** 31], [0, 1, 2, 3]], dtype=torch.int32)
    positions = torch.tensor([[15, 16, 40, 63, 64], [31, 32, -1, 2 ** 31 - 1, 0], [63, 10 ** 6, -2 ** 31, 62, 64]], dtype=torch.int32)
    q, qr = _queries(g, 3, 5, 6, 64, 16, dtype)
    got = _check(dev, q, qr, cache, table, positions, E4M3)
    assert torch.isnan(got).all(-1).all(-1).tolist() == [[False, True, True, True, True], [False, True, False, True, False],
                                                        [False, True, False, False, True]]


@pytest.mark.parametrize("store", [E4M3, BF16])
def test_rows_of_nan_and_of_extreme_scales(dev, store):
    """A token that append made NaN; latents near the largest and the smallest numbers."""
    c = _c()
    x = torch.randn(1, 40, 64, generator=torch.Generator().manual_seed(8))
    x[0, 10] *= 1e30
    x[0, 20] *= 1e-30
    words = torch.randn(1, 40, 16, generator=torch.Generator().manual_seed(9))
    table = torch.tensor([[1, 0, 2]], dtype=torch.int32)
    cache = c.latent_cache(3, 16, 64, 16, store, dev)
    at = torch.arange(40, dtype=torch.int32)[None]
    c.latent_append(x.to(dev), words.to(dev), cache, table.to(dev), at.to(dev))
    q, qr = _queries(torch.Generator().manual_seed(7), 1, 40, 4, 64, 16, F32)
    q[:, :, 1] = 0
    _check(dev, q * 1e-3, qr, cache.cpu(), table, at, store, scale=1e-4)
    x[0, 30, 5] = torch.nan
    c.latent_append(x.to(dev), words.to(dev), cache, table.to(dev), at.to(dev))
    got = c.latent_attention(q.to(dev), qr.to(dev), cache, table.to(dev), at.to(dev), 1e-4)
    assert not torch.isnan(got[0, :30]).any() and torch.isnan(got[0, 30:]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,rank", [(5, 64), (16, 512), (40, 512)])
def test_long_and_uneven_sequences_in_parts(dev, dtype, H, rank):
    """Keys in parts over the chip, a sequence so short that most parts are empty, a table with room to spare."""
    g = torch.Generator().manual_seed(H)
    page, width = 64, 320
    lengths = [9000, 3, 4096, 1]
    pages = sum(-(-n // page) for n in lengths)
    cache = ref.random_cache(g, pages, page, rank, 32, E4M3)
    table, at = torch.full((4, width), -1, dtype=torch.int32), 0
    for b, n in enumerate(lengths):
        need = -(-n // page)
        table[b, :need] = torch.arange(at, at + need)
        at += need
    positions = torch.tensor([[n - 1] for n in lengths], dtype=torch.int32)
    q, qr = _queries(g, 4, 1, H, rank, 32, dtype)
    q *= 3  # a few tokens carry the weight
    _check(dev, q, qr, cache, table, positions, E4M3)
    # Scores that rise towards the end: the maximum moves in every tile.
    cache = cache.clone()
    flat = cache.view(-1, cache.shape[-1])
    flat[:141 * 64, rank:rank + 2] = (torch.arange(141 * 64)[:, None] / 100).to(BF16).view(torch.uint8)
    qr[..., 0] = rank ** 0.5 * 3
    _check(dev, q, qr, cache, table, positions, E4M3)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_views_at_any_alignment_and_order(dev, dtype):
    """Queries as parts of wider heads at odd elements, heads before tokens, and a table and positions that are views."""
    g = torch.Generator().manual_seed(4)
    wide = torch.randn(2, 6, 5, 64 + 16 + 3, generator=g).to(dtype)  # [B, H, L, ..]
    cache, table = ref.random_cache(g, 8, 16, 64, 16, E4M3), ref.random_table(g, 2, 4, 8)
    positions = torch.tensor([[50, 51, 52, 53, 54], [3, 4, 5, 6, 7]], dtype=torch.int32)
    q, qr = wide[..., 1:65].transpose(1, 2), wide[..., 66:82].transpose(1, 2)
    expect = _check(dev, q.contiguous(), qr.contiguous(), cache, table, positions, E4M3)
    d = wide.to(dev)
    got = _c().latent_attention(d[..., 1:65].transpose(1, 2), d[..., 66:82].transpose(1, 2), cache.to(dev),
                                table.t().contiguous().to(dev).t(), positions.t().contiguous().to(dev).t(), 80 ** -0.5)
    assert torch.equal(got, expect)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("tree", [False, True])
def test_in_a_graph_and_on_streams(dev, dtype, tree):
    """A captured call, replayed at further positions with other queries, and eager calls between the replays; two streams at
    once. Each result equals the eager call's, bit for bit."""
    c, g = _c(), torch.Generator().manual_seed(11)
    B, L, H, rank, page, width = 3, 4, 16, 512, 64, 40
    cache, table = ref.random_cache(g, B * width, page, rank, 64, E4M3).to(dev), ref.random_table(g, B, width, B * width).to(dev)
    q, qr = (t.to(dev) for t in _queries(g, B, L, H, rank, 64, dtype))
    at = torch.tensor([[100 + 50 * b + i for i in range(L)] for b in range(B)], dtype=torch.int32, device=dev)
    words = torch.randint(0, 16, (B, L), generator=g).to(dev) if tree else None
    call = lambda: c.latent_attention(q, qr, cache, table, at, 0.04, words)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for replay in range(4):
        q.copy_(torch.randn(q.shape, generator=g).to(dtype))
        at += 311
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call()), f"replay {replay}"
    expect = call()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        one = [call() for _ in range(5)]
    two = [call() for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(t, expect) for t in one + two)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("store", [E4M3, BF16])
@pytest.mark.parametrize("H,rank", [(5, 64), (70, 128), (16, 512)])
@pytest.mark.parametrize("scale", [0.0, -0.05])
def test_scales_that_are_not_positive(dev, dtype, store, H, rank, scale):
    """A scale of 0 weighs every token alike, a negative one the other way round; in parts and trees too."""
    g = torch.Generator().manual_seed(H)
    cache, table = ref.random_cache(g, 16, 48, rank, 16, store), ref.random_table(g, 2, 8, 16)
    positions = torch.tensor([[200, 201, 202], [5, 6, 7]], dtype=torch.int32)
    q, qr = _queries(g, 2, 3, H, rank, 16, dtype)
    _check(dev, q, qr, cache, table, positions, store, scale=scale)
    _check(dev, q, qr, cache, table, positions, store, scale=scale, ancestors=torch.tensor([[1, 2, 5], [0, 3, 6]]))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("store", [E4M3, BF16])
@pytest.mark.parametrize("H", [2, 40])
def test_more_sequences_than_are_shared_out(dev, dtype, store, H):
    g = torch.Generator().manual_seed(H)
    B, page, width = 1100, 16, 16
    cache = ref.random_cache(g, 60, page, 64, 16, store)
    table = torch.randint(0, 60, (B, width), generator=g, dtype=torch.int32)
    positions = torch.randint(-1, page * width, (B, 1), generator=g, dtype=torch.int32)
    q, qr = _queries(g, B, 1, H, 64, 16, dtype)
    _check(dev, q, qr, cache, table, positions, store)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,rank,B,most", [(16, 512, 20, 3000), (70, 64, 300, 200), (40, 256, 7, 5000), (4, 128, 600, 150)])
def test_shares_of_many_uneven_sequences(dev, dtype, H, rank, B, most):
    """Parts that begin and end inside a sequence, hold several whole ones, or are empty; one sequence sees nothing."""
    g = torch.Generator().manual_seed(B)
    page, width = 32, 160
    cache = ref.random_cache(g, 200, page, rank, 16, E4M3)
    table = torch.randint(0, 200, (B, width), generator=g, dtype=torch.int32)
    positions = (torch.rand(B, 1, generator=g) ** 2 * most).to(torch.int32)
    positions[B // 2] = -1
    q, qr = _queries(g, B, 1, H, rank, 16, dtype)
    _check(dev, q, qr, cache, table, positions, E4M3)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("store", [E4M3, BF16])
@pytest.mark.parametrize("H,rank,page", [(8, 64, 1), (70, 64, 1), (40, 512, 3)])
def test_small_pages_of_a_long_sequence(dev, dtype, store, H, rank, page):
    """More pages than are looked up at a time, in one block's share and over the chip; one of them missing."""
    g = torch.Generator().manual_seed(page)
    n = 2500
    width = -(-n // page)
    cache, table = ref.random_cache(g, width + 3, page, rank, 16, store), ref.random_table(g, 1, width, width + 3)
    positions = torch.tensor([[n - 2, n - 1]], dtype=torch.int32)
    q, qr = _queries(g, 1, 2, H, rank, 16, dtype)
    _check(dev, q, qr, cache, table, positions, store)
    # Many short-lived units make a block's share as long as a sequence.
    many = 300
    at = torch.full((many, 1), n - 1, dtype=torch.int32)
    at[3:] = torch.randint(0, 900, (many - 3, 1), generator=g, dtype=torch.int32)
    q, qr = _queries(g, many, 1, H, rank, 16, dtype)
    _check(dev, q, qr, cache, table.expand(many, width).contiguous(), at, store)
    table[0, 777] = -1
    _check(dev, q[:4], qr[:4], cache, table.expand(4, width).contiguous(), at[:4], store)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("store,rank,rope,H", [(E4M3, 512, 64, 16), (E4M3, 512, 64, 64), (BF16, 256, 32, 40), (E4M3, 64, 16, 24)])
@pytest.mark.parametrize("size", [2 ** 32 - 2 ** 20, 2 ** 32 + 2 ** 28])
def test_a_large_cache(dev, dtype, store, rank, rope, H, size):
    """Pages all over a cache of just under 4 GiB, and of more, give bit for bit what they give in a small one."""
    g = torch.Generator().manual_seed(rank)
    page, width, row = 64, 10, ref.row_bytes(rank, rope, store)
    small, table = ref.random_cache(g, 2 * width, page, rank, rope, store).to(dev), ref.random_table(g, 2, width, 2 * width)
    pages = size // (page * row)
    large = torch.empty(pages, page, row, dtype=torch.uint8, device=dev)
    far = (torch.arange(2 * width) * ((pages - 1) // (2 * width - 1))).flip(0)
    far[0] = pages - 1
    large[far.to(dev)] = small
    q, qr = (t.to(dev) for t in _queries(g, 2, 2, H, rank, rope, dtype))
    positions = torch.tensor([[630, 631], [200, 201]], dtype=torch.int32, device=dev)
    expect = _c().latent_attention(q, qr, small, table.to(dev), positions, 0.05)
    got = _c().latent_attention(q, qr, large, far[table.long()].to(torch.int32).to(dev), positions, 0.05)
    assert torch.isfinite(expect).all() and torch.equal(got, expect)
    # What append writes there, read gives back.
    x, words = torch.randn(2, 1, rank, generator=g).to(dtype).to(dev), torch.randn(2, 1, rope, generator=g).to(dtype).to(dev)
    at = positions[:, 1:].contiguous()
    for cache, ids in ((small, table.to(dev)), (large, far[table.long()].to(torch.int32).to(dev))):
        _c().latent_append(x, words, cache, ids, at)
    one = _c().latent_read(small, table.to(dev), at, rank, rope, dtype)
    two = _c().latent_read(large, far[table.long()].to(torch.int32).to(dev), at, rank, rope, dtype)
    assert all(torch.equal(a, b) for a, b in zip(one, two))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,rank", [(5, 64), (40, 512), (70, 128)])
def test_one_token_carries_all_the_weight(dev, dtype, H, rank):
    """Scores of thousands, so that a row's result is one latent (its weight and the result rounded, to bf16 at the coarsest);
    and a query of zeros, whose result is their mean."""
    g = torch.Generator().manual_seed(H)
    cache, table = ref.random_cache(g, 20, 32, rank, 32, E4M3), ref.random_table(g, 2, 10, 20)
    positions = torch.tensor([[318, 319], [0, 77]], dtype=torch.int32)
    q, qr = _queries(g, 2, 2, H, rank, 32, dtype)
    _check(dev, q * 0, qr * 0, cache, table, positions, E4M3)
    got = _c().latent_attention((q * 512).to(dev), (qr * 512).to(dev), cache.to(dev), table.to(dev), positions.to(dev), 1.0).double().cpu()
    latent, words = ref.contents(cache, rank, 32, E4M3)
    for b in range(2):
        for i in range(2):
            n = int(positions[b, i]) + 1
            c, r = latent[table[b].long()].flatten(0, 1)[:n], words[table[b].long()].flatten(0, 1)[:n]
            score = 512 * (q[b, i].double() @ c.t() + qr[b, i].double() @ r.t())
            best = score.topk(min(2, n), -1)
            sure = torch.ones(H, dtype=torch.bool) if n == 1 else best.values[:, 0] - best.values[:, 1] > 60
            expect = c[best.indices[:, 0]]
            assert sure.any() and ((got[b, i] - expect).abs()[sure] <= 2.02 * ref.half_step(BF16) * expect.abs()[sure] + 1e-12).all()


@pytest.mark.parametrize("B,L", [(0, 1), (2, 0), (0, 0)])
def test_empty_calls(dev, B, L):
    c = _c()
    cache = c.latent_cache(2, 16, 64, 16, E4M3, dev)
    at, table = torch.zeros(B, L, dtype=torch.int32, device=dev), torch.zeros(B, 2, dtype=torch.int32, device=dev)
    for dtype in (F32, BF16):
        q, qr = torch.zeros(B, L, 3, 64, dtype=dtype, device=dev), torch.zeros(B, L, 3, 16, dtype=dtype, device=dev)
        assert c.latent_attention(q, qr, cache, table, at, 1.0).shape == (B, L, 3, 64)
        assert c.latent_attention(q, qr, cache, table, at, 1.0, torch.zeros(B, L, dtype=torch.int64, device=dev)).shape == (B, L, 3, 64)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_tensors_of_one_storage_and_expanded_ones(dev, dtype):
    """Every sequence with the same table, positions and queries, expanded without a copy."""
    g = torch.Generator().manual_seed(12)
    cache, table = ref.random_cache(g, 8, 16, 64, 16, BF16), ref.random_table(g, 1, 8, 8)
    positions = torch.tensor([[99, 100, 101]], dtype=torch.int32)
    q, qr = _queries(g, 1, 1, 6, 64, 16, dtype)
    spread = lambda t, *s: t.to(dev).expand(*s)
    got = _c().latent_attention(spread(q, 4, 3, 6, 64), spread(qr, 4, 3, 6, 16), cache.to(dev), spread(table, 4, 8), spread(positions, 4, 3), 0.1)
    one = _check(dev, q.expand(1, 3, 6, 64), qr.expand(1, 3, 6, 16), cache, table, positions, BF16, scale=0.1)
    out, size, span = ref.attention(q.expand(1, 3, 6, 64), qr.expand(1, 3, 6, 16), cache, table, positions, 0.1, BF16)
    bound = ref.attention_bound(size, span, out, 102, 80, dtype)
    for b in range(4):
        _within(got[b:b + 1], out, bound)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("store", [E4M3, BF16])
@pytest.mark.parametrize("name", [-1, -2, -3, 4, 5, 2 ** 30])
def test_every_number_outside_the_pages_is_a_missing_page(dev, dtype, store, name):
    """In a whole tile, in a tile that ends with the sequence, and where no token sees it."""
    g = torch.Generator().manual_seed(12)
    cache = ref.random_cache(g, 4, 64, 64, 16, store)
    table = torch.tensor([[name, 1, 2], [0, name, 3], [2, 3, name]], dtype=torch.int32)
    positions = torch.tensor([[63, 130, 5], [63, 64, 191], [127, 128, 150]], dtype=torch.int32)
    q, qr = _queries(g, 3, 3, 4, 64, 16, dtype)
    got = _check(dev, q, qr, cache, table, positions, store)
    assert torch.isnan(got).all(-1).all(-1).tolist() == [[True, True, True], [False, True, True], [False, True, True]]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("store", [E4M3, BF16])
@pytest.mark.parametrize("H", [2, 40])
@pytest.mark.parametrize("B,n,width", [(2, 40, 1), (1, 5000, 80), (20, 1500, 32)])
def test_scores_of_minus_infinity_alone(dev, dtype, store, H, B, n, width):
    """Every second head's scores are -2^160 or less, which fp32 holds as -infinity: NaN as of a softmax over nothing but
    minus infinities, in one piece and in parts; zeros stay with what sees no token. The other heads weigh all tokens alike."""
    g = torch.Generator().manual_seed(n)
    pages = B * width
    cache, table = ref.random_cache(g, pages, 64, 64, 16, store), ref.random_table(g, B, width, pages)
    if store == E4M3:
        cache[..., 0] = 254  # -448
        cache[..., 96:100] = torch.tensor([2.0 ** 92]).view(torch.uint8)
    else:
        cache[..., :2] = torch.tensor([-2.0 ** 100], dtype=BF16).view(torch.uint8)
    positions = torch.tensor([[n - 1, -1]] * B, dtype=torch.int32)
    q, qr = torch.zeros(B, 2, H, 64), torch.zeros(B, 2, H, 16)
    q[:, :, ::2, 0] = 2.0 ** 60
    q, qr = q.to(dtype), qr.to(dtype)
    got = _c().latent_attention(q.to(dev), qr.to(dev), cache.to(dev), table.to(dev), positions.to(dev), 1.0)
    assert torch.isnan(got[:, 0, ::2]).all() and (got[:, 1] == 0).all() and torch.isfinite(got[:, 0, 1::2]).all()
    # Past the table it is NaN, in a tree that sees no place zeros.
    positions[:, 0], positions[:, 1] = 64 * width, 0
    got = _c().latent_attention(q.to(dev), qr.to(dev), cache.to(dev), table.to(dev), positions.to(dev), 1.0,
                                torch.tensor([[1, 1]] * B).to(dev))
    assert torch.isnan(got[:, 0]).all() and (got[:, 1] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("store", [E4M3, BF16])
@pytest.mark.parametrize("H", [2, 40])
@pytest.mark.parametrize("n", [1, 128, 4096])
def test_the_largest_latents_that_sums_hold(dev, dtype, store, H, n):
    """n tokens of +-2^126 / n (bf16: 2^110 / n), the scores of all but the first 64 of them 2^15.87 times theirs, which is less
    than what a maximum may grow by unnoticed. All latents of a column are alike, and so is their mean: it is off by the
    softmax's rounding, which attention_bound derives, and by no infinity."""
    g = torch.Generator().manual_seed(n)
    width, most = -(-n // 64), 2.0 ** (126 if dtype == F32 else 110) / n
    table = ref.random_table(g, 1, width, width)
    sign = torch.where(torch.rand(64, generator=g) < 0.5, -1.0, 1.0)
    cache = torch.zeros(width, 64, ref.row_bytes(64, 16, store), dtype=torch.uint8)
    if store == E4M3:
        cache[..., :64] = (256 * sign).to(E4M3).view(torch.uint8)
        cache[..., 96:100] = torch.tensor([most / 256]).view(torch.uint8)
    else:
        cache[..., :128] = (most * sign).to(BF16).view(torch.uint8)
    flat = cache[table[0].long()].flatten(0, 1)
    first = 64 if store == E4M3 else 128
    flat[64:, first:first + 2] = torch.tensor([1.0], dtype=BF16).view(torch.uint8)
    cache[table[0].long()] = flat.view(width, 64, -1)
    q, qr = torch.zeros(1, 1, H, 64, dtype=dtype), torch.zeros(1, 1, H, 16, dtype=dtype)
    qr[..., 0] = 11.0
    _check(dev, q, qr, cache, table, torch.tensor([[n - 1]], dtype=torch.int32), store, scale=1.0)

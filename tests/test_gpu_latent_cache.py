"""The latent cache on the GPU: what is written and read back, exactly, in both formats."""

from __future__ import annotations

import pytest
import torch

import latent_reference as ref

pytestmark = pytest.mark.gpu

F32, BF16, E4M3 = torch.float32, torch.bfloat16, torch.float8_e4m3fn


def _c():
    from montlok import _C

    return _C


def _same(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a[~torch.isnan(a)], b[~torch.isnan(b)])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("store", [E4M3, BF16])
@pytest.mark.parametrize("B,L,rank,rope,page,width", [(1, 1, 64, 16, 1, 1), (3, 5, 64, 32, 48, 3), (2, 130, 128, 64, 64, 4), (5, 1, 512, 64, 256, 2),
                                                      (1, 37, 256, 32, 7, 9), (4, 33, 512, 16, 32, 2), (2, 70, 64, 64, 1000, 1)])
def test_append_then_read(dev, dtype, store, B, L, rank, rope, page, width):
    """Bit for bit the definition's values; every row that no token was written to as it was."""
    g = torch.Generator().manual_seed(B * 1000 + L * 10 + rank)
    pages = B * width + 2
    cache0 = ref.random_cache(g, pages, page, rank, rope, store, garbage=True)
    table = ref.random_table(g, B, width, pages)
    both = (torch.randn(B, L, rank + rope + 3, generator=g) * torch.exp(3 * torch.randn(B, L, 1, generator=g))).to(dtype)
    positions = torch.stack([torch.randperm(width * page, generator=g)[:L] for _ in range(B)]).to(torch.int32) if L > 1 else \
        torch.randint(0, width * page, (B, 1), generator=g).to(torch.int32)
    positions[torch.rand(B, L, generator=g) < 0.15] = -1
    cache, d = cache0.to(dev), both.to(dev)
    _c().latent_append(d[..., 1:1 + rank], d[..., 1 + rank:1 + rank + rope], cache, table.to(dev), positions.to(dev))
    latent, words = _c().latent_read(cache, table.to(dev), positions.to(dev), rank, rope, dtype)
    shown = (positions >= 0)[..., None]
    assert latent.dtype == words.dtype == dtype
    assert _same(latent, torch.where(shown, ref.nearest(both[..., 1:1 + rank], store), 0.0))
    assert _same(words, torch.where(shown, both[..., 1 + rank:1 + rank + rope].to(BF16).double(), 0.0))
    kept, kept_words = ref.contents(cache, rank, rope, store)
    now = cache.cpu()
    for b in range(B):
        for i in range(L):
            at = int(positions[b, i])
            if at >= 0:
                p, o = int(table[b, at // page]), at % page
                assert _same(kept[p, o], latent[b, i]) and _same(kept_words[p, o], words[b, i])
                now[p, o] = cache0[p, o]
    assert torch.equal(now, cache0)


@pytest.mark.parametrize("rank", [64, 512])
def test_rounding_at_every_border(dev, rank):
    """Values on, next to and halfway between the codes' values under every kind of scale, both signs."""
    grid = ref.E4M3_VALUES[:127].float()
    middle = (grid[1:] + grid[:-1]) / 2
    near = torch.cat([grid, middle, torch.nextafter(middle, torch.tensor(0.0)), torch.nextafter(middle, torch.tensor(1000.0))])
    rows = []
    for e in (-125, -118, -117, -116, -60, 0, 1, 60, 118, 119):
        for start in range(0, len(near), rank - 1):
            part = near[start:start + rank - 1].double()
            row = torch.zeros(rank, dtype=torch.float64)
            row[:len(part)] = part
            row[rank - 1] = 448 if start == 0 else 256.0000305  # the row's largest: on its border, and just past the power below
            rows += [row * 2.0 ** e, -row * 2.0 ** e]
    rows += [torch.full((rank,), 3.4e38, dtype=torch.float64), torch.full((rank,), 1e-44, dtype=torch.float64),
             torch.zeros(rank, dtype=torch.float64), -torch.zeros(rank, dtype=torch.float64)]
    for e in range(-30, 30):  # a largest value around the border of two scales
        for most in (448.0, 448.00003, 447.99997):
            row = near[:rank].double().clone().clamp(max=400) * 0.37
            row = torch.cat([row, torch.zeros(rank - len(row), dtype=torch.float64)])
            row[0] = most
            rows.append(row * 2.0 ** e)
    x = torch.stack(rows)[None].float()
    x = torch.where(torch.isfinite(x), x, 1.0)
    n = x.shape[1]
    table = torch.arange(-(-n // 16), dtype=torch.int32)[None].to(dev)
    positions = torch.arange(n, dtype=torch.int32)[None].to(dev)
    cache = _c().latent_cache(table.shape[1], 16, rank, 16, device=dev)
    _c().latent_append(x.to(dev), torch.zeros(1, n, 16, device=dev), cache, table, positions)
    latent, _ = _c().latent_read(cache, table, positions, rank, 16)
    assert torch.equal(latent.double().cpu(), ref.nearest(x, E4M3))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("store", [E4M3, BF16])
def test_rows_that_are_no_numbers_become_nan_alone(dev, dtype, store):
    x = torch.randn(1, 5, 128, generator=torch.Generator().manual_seed(1)).to(dtype)
    x[0, 0, 5], x[0, 1, 64], x[0, 2, 127] = torch.nan, torch.inf, -torch.inf
    x[0, 3, 0] = 3.4028e38 if dtype == F32 else 3.38e38  # in fp32 it rounds to an infinity of bf16
    words = torch.randn(1, 5, 16, generator=torch.Generator().manual_seed(2)).to(dtype)
    words[0, 4, 3], words[0, 4, 4] = torch.nan, torch.inf  # the key part keeps its own
    table, positions = torch.zeros(1, 1, dtype=torch.int32, device=dev), torch.arange(5, dtype=torch.int32, device=dev)[None]
    cache = _c().latent_cache(1, 16, 128, 16, store, dev)
    _c().latent_append(x.to(dev), words.to(dev), cache, table, positions)
    latent, kept = _c().latent_read(cache, table, positions, 128, 16, dtype)
    assert _same(latent, ref.nearest(x, store)) and _same(kept, words.to(BF16))
    assert torch.isnan(latent).all(-1)[0].tolist()[:3] == [True] * 3 and not torch.isnan(latent[0, 4]).any()


@pytest.mark.parametrize("store", [E4M3, BF16])
def test_tokens_without_a_page_are_dropped_and_read_as_nan(dev, store):
    g = torch.Generator().manual_seed(3)
    cache0 = ref.random_cache(g, 4, 16, 64, 32, store)
    table = torch.tensor([[1, -1, 4], [2, 2 ** 31 - 1, -2 ** 31]], dtype=torch.int32)
    positions = torch.tensor([[0, 17, 32, 47, 48, 2 ** 31 - 1], [15, 16, 40, -1, -2 ** 31, 1000]], dtype=torch.int32)
    x, words = torch.randn(2, 6, 64, generator=g), torch.randn(2, 6, 32, generator=g)
    cache = cache0.to(dev)
    _c().latent_append(x.to(dev), words.to(dev), cache, table.to(dev), positions.to(dev))
    latent, kept = _c().latent_read(cache, table.to(dev), positions.to(dev), 64, 32)
    expect, expect_words = ref.nearest(x, store), words.to(BF16).double()
    for t in (expect, expect_words):
        t[0, 1:] = torch.nan
        t[1, 1:3], t[1, 3:5], t[1, 5] = torch.nan, 0, torch.nan
    assert _same(latent, expect) and _same(kept, expect_words)
    changed = (cache.cpu() != cache0).any(-1)
    assert changed.sum() == 2 and changed[1, 0] and changed[2, 15]


def test_pages_past_four_gigabytes(dev):
    """A cache of more than 2^32 bytes: its last rows written and read, and seen by a query."""
    rank, rope, page = 512, 64, 4096
    pages = 2 ** 32 // (page * 1168) + 3
    cache = torch.empty(pages, page, 1168, dtype=torch.uint8, device=dev)
    table = torch.tensor([[pages - 1, 0]], dtype=torch.int32, device=dev)
    x = torch.randn(1, 3, rank, generator=torch.Generator().manual_seed(4)).to(BF16).to(dev)
    words = torch.zeros(1, 3, rope, dtype=BF16, device=dev)
    positions = torch.tensor([[0, 1, 2]], dtype=torch.int32, device=dev)
    _c().latent_append(x, words, cache, table, positions)
    latent, _ = _c().latent_read(cache, table, positions, rank, rope, BF16)
    assert torch.equal(latent, x)
    out = _c().latent_attention(torch.zeros(1, 1, 2, rank, dtype=BF16, device=dev), torch.zeros(1, 1, 2, rope, dtype=BF16, device=dev),
                                cache, table, positions[:, 2:], 1.0)
    mean = x.double().mean(1)
    assert ((out[0, 0].double() - mean).abs() <= 2 * 2.0 ** -8 * x.double().abs().mean(1) + 1e-6).all()


def test_empty_calls(dev):
    cache = _c().latent_cache(2, 16, 64, 16, device=dev)
    for batch, length in ((0, 3), (2, 0)):
        at, table = torch.zeros(batch, length, dtype=torch.int32, device=dev), torch.zeros(batch, 1, dtype=torch.int32, device=dev)
        _c().latent_append(torch.zeros(batch, length, 64, device=dev), torch.zeros(batch, length, 16, device=dev), cache, table, at)
        latent, words = _c().latent_read(cache, table, at, 64, 16)
        assert latent.shape == (batch, length, 64) and words.shape == (batch, length, 16)
        out = _c().latent_attention(torch.zeros(batch, length, 3, 64, device=dev), torch.zeros(batch, length, 3, 16, device=dev), cache, table, at, 1.0)
        assert out.shape == (batch, length, 3, 64)

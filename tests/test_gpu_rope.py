"""rope on the GPU against float64: layouts, parts of the head, far positions, padding, strides."""

from __future__ import annotations

import pytest
import torch

import latent_reference as ref

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _c():
    from montlok import _C

    return _C


def _check(got, x, frequencies, positions, interleaved, magnitude):
    expect = ref.rotate(x, frequencies, positions, interleaved, magnitude)
    assert got.shape == x.shape and got.dtype == x.dtype and got.is_contiguous()
    off = (got.double().cpu() - expect).abs() / ref.rope_bound(expect, x.cpu(), x.dtype, magnitude)
    assert float(off.max()) <= 1.0, f"{float(off.max()):.3g} of the bound"


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,L,H,Hkv,D,rope", [(1, 1, 1, 1, 64, 64), (3, 5, 4, 1, 16, 16), (2, 33, 12, 2, 96, 32), (2, 7, 16, 16, 128, 128),
                                              (1, 130, 8, 1, 64, 32), (2, 3, 3, 5, 10, 6), (1, 2, 1, 1, 2, 2), (1, 4, 2, 1, 1024, 1024),
                                              (2, 2, 5, 1, 30, 8), (40, 60, 40, 3, 32, 16), (1, 3, 200, 7, 256, 64)])
def test_against_float64(dev, dtype, interleaved, B, L, H, Hkv, D, rope):
    g = torch.Generator().manual_seed(B + 10 * L + D)
    q, k = torch.randn(B, L, H, D, generator=g).to(dtype), torch.randn(B, L, Hkv, D, generator=g).to(dtype)
    positions = torch.randint(0, 5000, (B, L), generator=g).to(torch.int32)
    positions[torch.rand(B, L, generator=g) < 0.2] = -3
    frequencies, magnitude = _c().rope_frequencies(rope, factor=8.0, original_length=4096, device=dev)
    got = _c().rope(q.to(dev), k.to(dev), frequencies, positions.to(dev), interleaved, magnitude)
    if B * L > 1000:  # the reference walks over tokens: some of them
        keep = torch.randperm(L, generator=g)[:3]
        q, k, positions, got = q[:4, keep], k[:4, keep], positions[:4, keep], [t[:4, keep.to(dev)].contiguous() for t in got]
    for out, x in zip(got, (q, k)):
        _check(out, x, frequencies, positions, interleaved, magnitude)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_far_positions_keep_their_angles(dev, dtype, interleaved):
    """Up to the last int32 position at one radian a position, where a float32 angle would be off by whole turns."""
    positions = torch.tensor([[0, 1, 2 ** 20 + 1, 10 ** 8 + 7, 2 ** 31 - 1, 2 ** 31 - 2, -1, -2 ** 31]], dtype=torch.int32)
    x = torch.randn(1, 8, 2, 32, generator=torch.Generator().manual_seed(1)).to(dtype)
    frequencies = torch.tensor([1.0, 0.731, 0.5, 1e-3, 1e-7, 3.0e-9, 0.0, 1.9999, -0.25, 0.1, 0.2, 0.3, 0.4, 0.6, 0.7, 0.8],
                               dtype=torch.float64)
    for out in _c().rope(x.to(dev), x.to(dev), frequencies.to(dev), positions.to(dev), interleaved, 1.5):
        _check(out, x, frequencies, positions, interleaved, 1.5)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_views_at_any_alignment(dev, dtype):
    """Slices of wider rows at odd elements, keys that every query head shares expanded with stride 0, an empty batch."""
    g = torch.Generator().manual_seed(2)
    wide, keys = torch.randn(2, 9, 3, 71, generator=g).to(dtype), torch.randn(2, 9, 1, 67, generator=g).to(dtype)
    q, k = wide[:, :, :, 7:], keys[:, :, :, 3:].expand(2, 9, 4, 64)
    positions = torch.arange(18, dtype=torch.int32).view(9, 2).t()
    frequencies, _ = _c().rope_frequencies(32, device=dev)
    dq, dk = wide.to(dev)[:, :, :, 7:], keys.to(dev)[:, :, :, 3:].expand(2, 9, 4, 64)
    for interleaved in (False, True):
        for out, x in zip(_c().rope(dq, dk, frequencies, positions.to(dev), interleaved), (q, k)):
            _check(out, x, frequencies, positions, interleaved, 1.0)
    empty = _c().rope(dq[:0], dk[:0], frequencies, positions[:0].to(dev))
    assert empty[0].shape == (0, 9, 3, 64) and empty[1].shape == (0, 9, 4, 64)


def test_values_that_are_no_numbers_stay_in_their_pair(dev):
    x = torch.ones(1, 1, 1, 16, device=dev)
    x[..., 9] = torch.nan
    frequencies, _ = _c().rope_frequencies(8, device=dev)
    at = torch.tensor([[3]], dtype=torch.int32, device=dev)
    half, _ = _c().rope(x, x, frequencies, at)
    pairs, _ = _c().rope(x, x, frequencies, at, True)
    assert torch.isnan(half).nonzero()[:, 3].tolist() == [9, 13] and torch.isnan(pairs).nonzero()[:, 3].tolist() == [8, 9]
    padded, _ = _c().rope(x, x, frequencies, -at)
    assert (padded == 0).all()

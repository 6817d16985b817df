"""head_linear on the GPU against float64: both ways round, types, odd sizes, views."""

from __future__ import annotations

import pytest
import torch

import latent_reference as ref

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
TYPES = [(F32, F32), (F32, BF16), (BF16, BF16)]


def _c():
    from montlok import _C

    return _C


def _check(got, x, w):
    """A sum of K products, K u of the sum of their magnitudes (u = 2^-24, three more for a product of split numbers), and a
    rounding to the result's type."""
    x, w = x.double().cpu(), w.double().cpu()
    expect = torch.stack([x[..., h, :] @ w[h].t() for h in range(w.shape[0])], -2)
    size = torch.stack([x[..., h, :].abs() @ w[h].abs().t() for h in range(w.shape[0])], -2)
    bound = (w.shape[2] + 3) * ref.U * size + ref.half_step(got.dtype) * expect.abs() * 1.01 + 1e-37
    assert got.shape == expect.shape and got.is_contiguous()
    off = ((got.double().cpu() - expect).abs() / bound).max() if got.numel() else torch.zeros(())
    assert float(off) <= 1.0, f"{float(off):.3g} of the bound"


@pytest.mark.parametrize("dtype,wtype", TYPES)
@pytest.mark.parametrize("inner_dense", [True, False])
@pytest.mark.parametrize("T,H,K,N", [(1, 1, 16, 64), (1, 64, 128, 512), (3, 8, 512, 128), (24, 5, 192, 256), (17, 16, 32, 64), (64, 3, 64, 96),
                                     (130, 4, 96, 512), (600, 2, 512, 96), (33, 2, 40, 24), (5, 3, 7, 5), (65, 2, 1, 1), (129, 3, 33, 65),
                                     (2, 7, 513, 130), (1000, 1, 256, 32)])
def test_against_float64(dev, dtype, wtype, inner_dense, T, H, K, N):
    g = torch.Generator().manual_seed(T + H + K)
    x = torch.randn(T, H, K, generator=g).to(dtype)
    w = (torch.randn(H, N, K, generator=g) * K ** -0.5).to(wtype)
    d = w.to(dev) if inner_dense else w.transpose(1, 2).contiguous().to(dev).transpose(1, 2)
    got = _c().head_linear(x.to(dev), d)
    assert got.dtype == dtype
    _check(got, x, w)


@pytest.mark.parametrize("dtype,wtype", TYPES)
@pytest.mark.parametrize("shift", [0, 1, 8])
def test_parts_of_one_projection(dev, dtype, wtype, shift):
    """The rows [H, 2 K, R] of one projection in both directions, x as a part of wider heads at odd elements, heads before
    tokens, several leading dimensions, an empty batch."""
    g = torch.Generator().manual_seed(3)
    H, K, R = 6, 32, 64
    w = torch.randn(H, 2 * K, R + 2 * shift, generator=g).to(wtype)
    part, d = w[:, :, shift:shift + R], w.to(dev)[:, :, shift:shift + R]
    x = torch.randn(2, 9, H, K + 19, generator=g).to(dtype)
    dx = x.to(dev)
    _check(_c().head_linear(dx[..., 3:3 + K], d[:, :K].transpose(1, 2)), x[..., 3:3 + K], part[:, :K].transpose(1, 2))
    y = torch.randn(H, 2, 9, R, generator=g).to(dtype)
    _check(_c().head_linear(y.to(dev).permute(1, 2, 0, 3), d[:, K:]), y.permute(1, 2, 0, 3), part[:, K:])
    assert _c().head_linear(dx[:0, ..., :K], d[:, :K].transpose(1, 2)).shape == (0, 9, H, R)
    one = _c().head_linear(dx[0, 0, :, :K], d[:, :K].transpose(1, 2))  # no leading dimension but the heads
    _check(one, x[0, 0, :, :K], part[:, :K].transpose(1, 2))


@pytest.mark.parametrize("dtype,wtype", TYPES)
def test_values_that_are_no_numbers_stay_in_their_row_and_column(dev, dtype, wtype):
    x, w = torch.ones(40, 2, 64, dtype=dtype, device=dev), torch.ones(2, 48, 64, dtype=wtype, device=dev)
    x[7, 0, 3], x[20, 1, 63] = torch.nan, torch.inf
    w[1, 5, 0] = torch.nan
    got = _c().head_linear(x, w)
    bad = ~torch.isfinite(got)
    expect = torch.zeros(40, 2, 48, dtype=torch.bool, device=dev)
    expect[7, 0], expect[20, 1], expect[:, 1, 5] = True, True, True
    assert torch.equal(bad, expect) and (got[~bad] == 64).all()


@pytest.mark.parametrize("dtype,wtype", TYPES)
@pytest.mark.parametrize("inner_dense", [True, False])
@pytest.mark.parametrize("T,H,K,N", [(5001, 8, 32, 256), (3000, 16, 61, 300), (3001, 16, 128, 520), (2999, 16, 200, 256), (3000, 16, 500, 130),
                                     (300, 16, 600, 100)])
def test_many_tokens(dev, dtype, wtype, inner_dense, T, H, K, N):
    """Blocks that go over several tiles of tokens, the last of them short."""
    g = torch.Generator().manual_seed(T + K)
    x = torch.randn(T, H, K, generator=g).to(dtype)
    w = (torch.randn(H, N, K, generator=g) * K ** -0.5).to(wtype)
    d = w.to(dev) if inner_dense else w.transpose(1, 2).contiguous().to(dev).transpose(1, 2)
    _check(_c().head_linear(x.to(dev), d), x, w)


def test_in_a_graph_and_on_streams(dev):
    """Captured calls of both directions, replayed on other inputs with eager calls between; each equals the eager call's."""
    c, g = _c(), torch.Generator().manual_seed(2)
    w = torch.randn(16, 256, 128, generator=g).to(BF16).to(dev)
    x = torch.randn(24, 16, 128, generator=g).to(BF16).to(dev)
    call = lambda: c.head_linear(c.head_linear(x, w), w.transpose(1, 2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for replay in range(3):
        x.copy_(torch.randn(x.shape, generator=g).to(BF16))
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call()), f"replay {replay}"


@pytest.mark.parametrize("dtype,wtype", TYPES)
@pytest.mark.parametrize("N,K", [(1, 1), (1, 5), (5, 1)])
def test_weights_of_one_input_or_output_in_any_order(dev, dtype, wtype, N, K):
    """Parts of a tensor whose heads lie side by side, which count as contiguous where both sizes are 1."""
    g = torch.Generator().manual_seed(13)
    w = torch.randn(8, 7, 3, generator=g).to(wtype)
    x = torch.randn(40, 3, K, generator=g).to(dtype)
    _check(_c().head_linear(x.to(dev), w.to(dev).permute(2, 0, 1)[:, :N, :K]), x, w.permute(2, 0, 1)[:, :N, :K])

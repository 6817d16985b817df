"""RMSNorm and rotation of query and key heads against float64."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _reference(x, weight, eps, cos, sin, positions):
    x = x.double()
    y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * weight.double()
    rope = cos.shape[1]
    at = positions.long().clamp(0, max(len(cos) - 1, 0))
    if rope:
        turn = y[..., y.shape[-1] - rope:].clone()
        a, b = turn.chunk(2, -1)
        c, s = cos.double()[at][:, :, None], sin.double()[at][:, :, None]
        y[..., y.shape[-1] - rope:] = turn * c + torch.cat([-b, a], -1) * s
    y[positions >= len(cos)] = torch.nan
    y[positions < 0] = 0
    return y


def _check(got, expect, dtype):
    """One rounding of a result formed in float64: half a step of the type, and float64's own error on the parts of a
    rotation, which may cancel: 2^-48 of the row's largest."""
    got, step = got.double().cpu(), torch.finfo(dtype).eps / 2
    assert torch.equal(torch.isnan(got), torch.isnan(expect))
    fine = ~torch.isnan(expect)
    largest = torch.where(fine, expect.abs(), 0.0).amax(-1, keepdim=True).expand_as(expect)
    assert ((got - expect).abs()[fine] <= (step * expect.abs() + 2.0 ** -48 * largest + 1e-38)[fine]).all()


def _tables(g, rows, rope):
    angle = torch.rand(rows, rope // 2, generator=g) * 7
    angle = torch.cat([angle, angle], 1)
    return angle.cos(), angle.sin()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,L,H,Hkv,D,rope", [(1, 1, 1, 1, 2, 2), (2, 3, 4, 2, 64, 64), (3, 5, 32, 8, 128, 64), (1, 7, 3, 3, 32, 32), (2, 2, 2, 1, 256, 256),
                                              (1, 4, 5, 2, 10, 6), (2, 3, 2, 2, 96, 32), (1, 2, 3, 1, 1024, 512), (1, 3, 2, 1, 33, 0),
                                              (4, 50, 12, 4, 64, 32), (2, 3, 2, 1, 128, 4), (1, 2, 1, 1, 7, 6), (2, 3, 4, 2, 512, 128),
                                              (1, 3, 4, 1, 256, 120), (7, 1, 16, 2, 32, 16)])
def test_against_float64(dev, dtype, B, L, H, Hkv, D, rope):
    from montlok import _C

    g = torch.Generator().manual_seed(D * 10 + H)
    qkv = (torch.randn(B, L, H + 2 * Hkv, D, generator=g) * torch.exp(2 * torch.randn(B, L, H + 2 * Hkv, 1, generator=g))).to(dtype)
    weights = 1 + 0.3 * torch.randn(2, D, generator=g)
    cos, sin = _tables(g, 40, rope)
    positions = torch.randint(-1, 42, (B, L), generator=g, dtype=torch.int32)
    d = qkv.to(dev)
    q, k = _C.qk_norm_rope(d[:, :, :H], d[:, :, H:H + Hkv], weights[0].to(dev), weights[1].to(dev), 1e-5, cos.to(dev), sin.to(dev), positions.to(dev))
    assert q.dtype == k.dtype == dtype and q.is_contiguous() and k.is_contiguous()
    assert torch.equal(d.cpu(), qkv)
    _check(q, _reference(qkv[:, :, :H], weights[0], 1e-5, cos, sin, positions), dtype)
    _check(k, _reference(qkv[:, :, H:H + Hkv], weights[1], 1e-5, cos, sin, positions), dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D,rope", [(64, 64), (128, 64), (32, 16), (256, 256), (96, 32)])
def test_views_give_the_copys_bits(dev, dtype, D, rope):
    """Strides and alignments of the operands."""
    from montlok import _C

    g = torch.Generator().manual_seed(D)
    wide = torch.randn(3, 4, 6, D + 3, generator=g).to(dtype).to(dev)
    cos, sin = (t.to(dev) for t in _tables(g, 10, rope))
    w, at = torch.randn(D + 1, generator=g).to(dev), torch.arange(12, dtype=torch.int32, device=dev).view(3, 4) - 1
    expect = _C.qk_norm_rope(wide[:, :, :4, :D].contiguous(), wide[:, :, 4:, :D].contiguous(), w[:D].clone(), w[:D].clone(), 1e-6, cos, sin, at)
    for lead in (0, 1, 2, 3):
        x = torch.roll(wide, lead, -1)[..., lead:lead + D]  # the same values at another alignment
        got = _C.qk_norm_rope(x[:, :, :4], x[:, :, 4:], w[:D], w[:D], 1e-6, cos, sin, at)
        assert all(torch.equal(torch.nan_to_num(a, 77.0), torch.nan_to_num(b, 77.0)) for a, b in zip(got, expect))
    turned = wide[..., :D].transpose(0, 1).contiguous().transpose(0, 1)
    w1 = torch.empty(D + 1, device=dev)[1:].copy_(w[:D])  # a weight 4 bytes off
    wide_cos = torch.cat([cos, sin], 1)
    got = _C.qk_norm_rope(turned[:, :, :4], turned[:, :, 4:], w1, w1, 1e-6, wide_cos[:, :rope], wide_cos[:, rope:], at.t().contiguous().t())
    assert all(torch.equal(torch.nan_to_num(a, 77.0), torch.nan_to_num(b, 77.0)) for a, b in zip(got, expect))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [32, 64, 100, 128, 256])
def test_values_at_the_ends_of_the_range(dev, dtype, D):
    """Rows of zeros, of the largest and smallest numbers; a NaN or an infinity in one head stays in it."""
    from montlok import _C

    g = torch.Generator().manual_seed(2)
    x = torch.randn(1, 6, 2, D, generator=g)
    x[0, 0] = 0
    x[0, 1] *= 1e37
    x[0, 2] *= 1e-38
    x[0, 3, 0, 5] = torch.nan
    x[0, 4, 1, 9] = torch.inf
    x = x.to(dtype)
    w, at = torch.ones(D), torch.arange(6, dtype=torch.int32)[None]
    cos, sin = _tables(g, 8, D // 2)
    d = x.to(dev)
    for eps in (1e-5, 0.0):
        q, k = _C.qk_norm_rope(d[:, :, :1], d[:, :, 1:], w.to(dev), w.to(dev), eps, cos.to(dev), sin.to(dev), at.to(dev))
        _check(q, _reference(x[:, :, :1], w, eps, cos, sin, at), dtype)
        _check(k, _reference(x[:, :, 1:], w, eps, cos, sin, at), dtype)


def test_many_rows(dev):
    """More rows than one wave of blocks, ragged: every element."""
    from montlok import _C

    g = torch.Generator().manual_seed(4)
    B, L, H, Hkv, D = 3, 1037, 8, 2, 64
    qkv = torch.randn(B, L, H + Hkv, D, generator=g)
    w = 1 + 0.1 * torch.randn(2, D, generator=g)
    cos, sin = _tables(g, L, 32)
    at = torch.arange(L, dtype=torch.int32).expand(B, L).clone()
    at[1, 700:] = -1
    d = qkv.to(dev)
    q, k = _C.qk_norm_rope(d[:, :, :H], d[:, :, H:], w[0].to(dev), w[1].to(dev), 1e-5, cos.to(dev), sin.to(dev), at.to(dev))
    _check(q, _reference(qkv[:, :, :H], w[0], 1e-5, cos, sin, at), F32)
    _check(k, _reference(qkv[:, :, H:], w[1], 1e-5, cos, sin, at), F32)


def test_no_tokens_and_no_table(dev):
    from montlok import _C

    w = torch.ones(64, device=dev)
    t = torch.zeros(0, 32, device=dev)
    x = torch.ones(1, 2, 2, 64, device=dev)
    at = torch.tensor([[-1, 0]], dtype=torch.int32, device=dev)
    q, k = _C.qk_norm_rope(x, x, w, w, 1e-5, t, t, at)  # a table without rows: every position is past it
    assert not q[:, 0].any() and torch.isnan(q[:, 1]).all() and not k[:, 0].any() and torch.isnan(k[:, 1]).all()
    e = torch.ones(0, 2, 2, 64, device=dev)
    assert _C.qk_norm_rope(e, e, w, w, 1e-5, t, t, at[:0])[0].shape == e.shape


def test_refusals(dev):
    from montlok import _C

    x, w, t = torch.ones(1, 2, 2, 64, device=dev), torch.ones(64, device=dev), torch.ones(4, 32, device=dev)
    at = torch.zeros(1, 2, dtype=torch.int32, device=dev)
    for call, text in ((lambda: _C.qk_norm_rope(x.half(), x, w, w, 1e-5, t, t, at), "q must be float32 or bfloat16"),
                       (lambda: _C.qk_norm_rope(x, x.bfloat16(), w, w, 1e-5, t, t, at), "k must be of q's dtype"),
                       (lambda: _C.qk_norm_rope(x, x[..., :32], w, w, 1e-5, t, t, at), "k must be"),
                       (lambda: _C.qk_norm_rope(x, x[:, :1], w, w, 1e-5, t, t, at), "k must be"),
                       (lambda: _C.qk_norm_rope(x[0], x[0], w, w, 1e-5, t, t, at), "q must have 4 dimensions"),
                       (lambda: _C.qk_norm_rope(x, x, w[:32], w, 1e-5, t, t, at), "head_dim elements"),
                       (lambda: _C.qk_norm_rope(x, x, w.double(), w, 1e-5, t, t, at), "q_weight must be float32"),
                       (lambda: _C.qk_norm_rope(x, x, w, w, 1e-5, t, t[:3], at), "cos and sin must be"),
                       (lambda: _C.qk_norm_rope(x, x, w, w, 1e-5, t[:, :5], t[:, :5], at), "rope_dim must be even"),
                       (lambda: _C.qk_norm_rope(x, x, w, w, 1e-5, t.repeat(1, 3), t.repeat(1, 3), at), "rope_dim must be even"),
                       (lambda: _C.qk_norm_rope(x, x, w, w, 1e-5, t, t, at.long()), "positions must be int32"),
                       (lambda: _C.qk_norm_rope(x, x, w, w, 1e-5, t, t, at[:, :1]), r"positions must be \[batch, length\]"),
                       (lambda: _C.qk_norm_rope(x, x, w, w.cpu(), 1e-5, t, t, at), "k_weight must be on the same GPU")):
        with pytest.raises(RuntimeError, match=text):
            call()


def _nearest_bf16(y):
    """The bf16 values next to float64 ones of ordinary size, straight from them: torch's cast rounds to float32 on its way."""
    step = 2.0 ** (torch.floor(torch.log2(y.abs())) - 7)
    return (torch.round(y / step) * step).to(torch.float32).to(BF16)  # ties, which torch.round gives the even one, as bf16's are


@pytest.mark.parametrize("D,rope", [(32, 0), (32, 32), (64, 32), (128, 128), (256, 256), (512, 256), (96, 32), (100, 100)])
def test_bf16_results_next_to_a_tie_are_rounded_once(dev, D, rope):
    """Weights, or cosines, that bring each result within 2^-23 of the middle between two bf16 values, where a rounding to
    float32 before that to bf16 lands on the middle and then on the wrong side."""
    from montlok import _C

    g = torch.Generator().manual_seed(D + rope)
    wrong = 0
    for _ in range(4):
        x = torch.randn(1, 1, 1, D, generator=g).to(BF16)
        x[x == 0] = 1
        middle = (1 + (2 * torch.randint(0, 64, (D,), generator=g) + 1).double() / 256) * (1 - 2.0 * torch.randint(0, 2, (D,), generator=g))
        by = (x[0, 0, 0].double() / torch.sqrt(x.double().square().mean() + 1e-6))
        weight = (middle / by).float()
        cos, sin = torch.ones(1, rope), torch.zeros(1, rope)
        if rope:  # rotated lanes: cos = (middle + what the sine takes) / own
            y = (by * weight)[D - rope:]
            a, b = y.chunk(2)
            sin = (torch.rand(1, rope, generator=g) - 0.5)
            other = torch.cat([-b, a]) * sin[0].double()
            cos = ((middle[D - rope:] - other) / y).float()[None]
        at = torch.zeros(1, 1, dtype=torch.int32)
        expect = _reference(x, weight, 1e-6, cos, sin, at)
        q, k = _C.qk_norm_rope(x.to(dev), x.to(dev), weight.to(dev), weight.to(dev), 1e-6, cos.to(dev), sin.to(dev), at.to(dev))
        nearest = _nearest_bf16(expect)
        clear = (expect - torch.round(expect * 256) / 256).abs() > 2.0 ** -44  # of the middles, by more than float64's own error
        wrong += int((expect.float().to(BF16) != nearest)[clear].sum())
        assert torch.equal(q.cpu()[clear], nearest[clear]) and torch.equal(k.cpu()[clear], nearest[clear])
    assert wrong >= D // 4


def _rows_a_wave(tokens, H, Hkv, D, dtype):
    """How many head rows a lane group takes: the rule of the launch."""
    groups = 64 // (D // (4 if dtype == F32 else 8))
    slots = lambda r: sum(-(-heads // (groups * r)) for heads in (H, Hkv)) * r
    for r in (4, 2):
        if tokens * slots(r) >= 4096 * r and 4 * slots(r) <= 5 * slots(1):
            return r
    return 1


@pytest.mark.parametrize("dtype,each,B,L,H,Hkv,D,rope", [
    (BF16, 4, 3, 700, 30, 8, 128, 64), (BF16, 4, 2, 1030, 60, 50, 32, 16), (BF16, 4, 1, 2051, 7, 8, 256, 256), (BF16, 4, 1, 1400, 7, 4, 512, 0),
    (BF16, 2, 2, 1030, 15, 10, 64, 32), (BF16, 2, 1, 2077, 8, 5, 128, 128), (BF16, 1, 3, 1037, 8, 2, 64, 32),
    (F32, 4, 2, 500, 30, 7, 128, 128), (F32, 4, 3, 700, 16, 15, 64, 64), (F32, 4, 1, 1400, 7, 4, 256, 128), (F32, 4, 1, 1030, 60, 50, 32, 0),
    (F32, 2, 2, 1030, 7, 6, 64, 32), (F32, 2, 1, 2077, 4, 3, 128, 32), (F32, 2, 5, 411, 16, 9, 32, 32)])
def test_several_rows_a_wave(dev, dtype, each, B, L, H, Hkv, D, rope):
    """Heads that leave a group's last turns empty, padding, positions past the tables, a head with a NaN and one with an
    infinity, q and k as views."""
    from montlok import _C

    assert _rows_a_wave(B * L, H, Hkv, D, dtype) == each
    g = torch.Generator().manual_seed(D + H + L)
    qkv = torch.randn(B, L, H + 2 * Hkv, D, generator=g)
    qkv[0, 3, H - 1, D - 1], qkv[B - 1, L - 1, H, 0] = torch.nan, torch.inf
    qkv = qkv.to(dtype)
    weights = 1 + 0.3 * torch.randn(2, D, generator=g)
    cos, sin = _tables(g, L, rope)
    positions = torch.arange(L, dtype=torch.int32).expand(B, L).clone()
    positions[torch.rand(B, L, generator=g) < 0.1] = -1
    positions[torch.rand(B, L, generator=g) < 0.05] = L
    positions[0, 3], positions[B - 1, L - 1] = 1, 2
    d = qkv.to(dev)
    q, k = _C.qk_norm_rope(d[:, :, :H], d[:, :, H:H + Hkv], weights[0].to(dev), weights[1].to(dev), 1e-5, cos.to(dev), sin.to(dev), positions.to(dev))
    _check(q, _reference(qkv[:, :, :H], weights[0], 1e-5, cos, sin, positions), dtype)
    _check(k, _reference(qkv[:, :, H:H + Hkv], weights[1], 1e-5, cos, sin, positions), dtype)

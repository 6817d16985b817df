"""The linear with 4-bit weights against float64."""

from __future__ import annotations

import pytest
import torch

import kv4_reference as ref

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _weights(g, n, k, low=120, high=124):
    return (torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8),
            torch.randint(low, high, (n, k // 32), generator=g, dtype=torch.uint8))


def _check(got, x, codes, scales, bias, dtype):
    """Products are exact; the sum of a float32 row has three parts a product, each addition u = 2^-24 of what is summed,
    the bias one more; bf16 rounds the result (2^-8)."""
    w = ref.value_of(codes, scales)
    rows = x.double().reshape(-1, x.shape[-1])
    out, size = rows @ w.t(), rows.abs() @ w.abs().t()
    if bias is not None:
        out, size = out + bias.double(), size + bias.double().abs()
    bound = (3 * x.shape[-1] + 8) * 2.0 ** -24 * size + 1e-37
    if dtype == BF16:
        bound = bound + 2.0 ** -8 * out.abs() * 1.01
    got = got.double().cpu().reshape(out.shape)
    off = float(((got - out).abs() / bound).max())
    assert off <= 1.0, f"{off:.3g} of the bound"
    # What sums of many terms are off by in earnest: far below the bound above.
    assert float((got - out).norm() / out.norm()) <= (3e-3 if dtype == BF16 else 2e-6)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 2, 5, 15, 16, 17, 33, 64, 65, 100, 129, 300])
@pytest.mark.parametrize("k,n", [(32, 16), (64, 1), (96, 17), (128, 64), (160, 130), (512, 100), (1056, 257), (4096, 48)])
def test_against_float64(dev, dtype, rows, k, n):
    from montlok import _C

    g = torch.Generator().manual_seed(rows * 7 + k + n)
    codes, scales = _weights(g, n, k)
    x = torch.randn(rows, k, generator=g).to(dtype)
    bias = torch.randn(n, generator=g) if (rows + n) % 2 else None
    got = _C.linear_fp4(x.to(dev), codes.to(dev), scales.to(dev), None if bias is None else bias.to(dev))
    assert got.shape == (rows, n) and got.dtype == dtype
    _check(got, x, codes, scales, bias, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,k,n", [(1, 8192, 4096), (3, 2048, 9000), (24, 4096, 4100), (200, 1024, 2051), (520, 512, 1000)])
def test_larger_shapes(dev, dtype, rows, k, n):
    from montlok import _C

    g = torch.Generator().manual_seed(n)
    codes, scales = _weights(g, n, k)
    x, bias = torch.randn(rows, k, generator=g).to(dtype), torch.randn(n, generator=g)
    _check(_C.linear_fp4(x.to(dev), codes.to(dev), scales.to(dev), bias.to(dev)), x, codes, scales, bias, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_views_and_leading_dimensions(dev, dtype):
    """Row strides, alignments and shapes of x: the same bits as a contiguous copy."""
    from montlok import _C

    g = torch.Generator().manual_seed(3)
    codes, scales = (t.to(dev) for t in _weights(g, 70, 96))
    wide = torch.randn(2, 5, 7, 131, generator=g).to(dtype).to(dev)
    for x in (wide[..., 1:97], wide[..., 3:99], wide[:, 1:4, ::2, 8:104], wide[0, 0, :, 2:98].t().contiguous().t(), wide[0, 0, 0, 5:101],
              wide[:0, 0, 0, :96]):
        got = _C.linear_fp4(x, codes, scales)
        assert got.shape == (*x.shape[:-1], 70)
        assert torch.equal(got, _C.linear_fp4(x.contiguous(), codes, scales))


@pytest.mark.parametrize("rows", [1, 40])
def test_range_of_values(dev, rows):
    """The largest and smallest scales and inputs: every product that float32 holds."""
    from montlok import _C

    g = torch.Generator().manual_seed(5)
    for low, high, size in ((3, 4, 2.0 ** 90), (240, 252, 2.0 ** -100), (100, 150, 2.0 ** -20), (127, 128, 2.0 ** 120), (200, 210, 2.0 ** -80)):
        codes, scales = _weights(g, 33, 64, low, high)
        x = torch.randn(rows, 64, generator=g) * size
        _check(_C.linear_fp4(x.to(dev), codes.to(dev), scales.to(dev)), x, codes, scales, None, F32)
    codes, scales = _weights(g, 33, 64, 100, 110)
    x = torch.full((rows, 64), 3.4028234663852886e38)  # no part of a value overflows
    x[:, ::2] *= -1
    _check(_C.linear_fp4(x.to(dev), codes.to(dev), scales.to(dev)), x, codes, scales, None, F32)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [3, 40])
def test_infinities_and_nan(dev, dtype, rows):
    """Rows and groups that hold them, as IEEE sums have them; the other rows and columns keep their bits."""
    from montlok import _C

    g = torch.Generator().manual_seed(7)
    codes, scales = _weights(g, 40, 160)
    codes |= 0x11  # no weight is zero: an infinity gives an infinity
    x = torch.randn(rows, 160, generator=g).to(dtype)
    clean = _C.linear_fp4(x.to(dev), codes.to(dev), scales.to(dev)).cpu()
    x[0, 3], x[1, 100], x[2, 159] = torch.inf, -torch.inf, torch.nan
    scales[9, 2] = 255
    got = _C.linear_fp4(x.to(dev), codes.to(dev), scales.to(dev)).cpu()
    expect = x.double() @ ref.value_of(codes, scales).t()
    assert torch.equal(torch.isnan(got), torch.isnan(expect)) and torch.equal(torch.isinf(got), torch.isinf(expect))
    assert torch.equal(torch.sign(got[:2, :9].double()), torch.sign(expect[:2, :9]))
    keep = torch.ones(40, dtype=torch.bool)
    keep[9] = False
    assert torch.equal(got[3:][:, keep], clean[3:][:, keep])


def test_refusals(dev):
    from montlok import _C

    x, codes, scales = torch.zeros(2, 64, device=dev), torch.zeros(8, 32, dtype=torch.uint8, device=dev), torch.zeros(8, 2, dtype=torch.uint8, device=dev)
    for call, text in ((lambda: _C.linear_fp4(x.half(), codes, scales), "input must be float32 or bfloat16"),
                       (lambda: _C.linear_fp4(x[:, :32], codes, scales), "input must end in in_features=64"),
                       (lambda: _C.linear_fp4(x, codes.int(), scales), "codes must be uint8"),
                       (lambda: _C.linear_fp4(x, codes[:, :24], scales), "codes must be"),
                       (lambda: _C.linear_fp4(x, codes[:0], scales), "codes must be"),
                       (lambda: _C.linear_fp4(x, codes, scales[:, :1]), "scales must be"),
                       (lambda: _C.linear_fp4(x, codes, scales.float()), "scales must be uint8"),
                       (lambda: _C.linear_fp4(x, codes, scales, torch.zeros(7, device=dev)), "bias must have 8 elements, got 7"),
                       (lambda: _C.linear_fp4(x, codes, scales, torch.zeros(8, device=dev).bfloat16()), "bias must be float32"),
                       (lambda: _C.linear_fp4(x, codes.cpu(), scales), "codes must be on the same GPU"),
                       (lambda: _C.linear_fp4(x, None, scales), "codes must be defined")):
        with pytest.raises(RuntimeError, match=text):
            call()


def test_graph_replays(dev):
    from montlok import _C

    g = torch.Generator().manual_seed(9)
    codes, scales = (t.to(dev) for t in _weights(g, 1000, 512))
    for rows in (1, 100):
        x = torch.randn(rows, 512, generator=g).to(dev)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _C.linear_fp4(x, codes, scales)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _C.linear_fp4(x, codes, scales)
        for replay in range(4):
            x.copy_(torch.randn(x.shape, generator=g))
            out.fill_(float("nan"))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, _C.linear_fp4(x, codes, scales)), f"replay {replay}"


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_weights_are_quantised_alike_on_the_gpu(dev, dtype):
    """The codes and scales of weights on the GPU are those of the same weights on the CPU, and ``linear_fp4`` of the unit
    rows gives their values back."""
    from montlok import _C

    g = torch.Generator().manual_seed(47)
    w = (torch.randn(130, 192, generator=g) * 2.0 ** torch.randint(-30, 30, (130, 1), generator=g)).to(dtype)
    w[3, :32], w[4, 32:64] = 0.0, 2.0 ** -100
    codes, scales = _C.fp4_weights(w)
    on_gpu = _C.fp4_weights(w.to(dev))
    assert torch.equal(on_gpu[0].cpu(), codes) and torch.equal(on_gpu[1].cpu(), scales)
    got = _C.linear_fp4(torch.eye(192, dtype=dtype, device=dev), *on_gpu)
    assert torch.equal(got.cpu().double(), ref.nearest(w).t())


# ------------------------------------------------------------------ every form of the kernel


def _form(rows, n, dtype, stride=0):
    """Which form a call takes: the rule of the launch, by rounds of blocks on 256 compute units."""
    up = lambda a, b: -(-a // b)
    rounds = lambda c, r: up(up(n, c) * up(rows, r), 256)
    full = lambda c: max(1.0, up(n, c) * up(rows, 16) / 256)
    few, tiles = rows <= 4, stride < 1 << 24
    if dtype == F32:
        if tiles and 30 * rounds(128, 32) < 12 * full(64):
            return "tile 128"
        by = {c: t * rounds(c, 16) for c, t in zip((16, 32, 64), (5.2, 6.8, 9.5) if few else (6.7, 8.1, 11.6))}
        columns = 64 if by[64] < min(by[16], by[32]) else 16 if by[16] <= by[32] else 32
    else:
        narrow, wide = 15.5 * rounds(64, 64), 22 * rounds(128, 64)
        if tiles and min(narrow, wide) < 3.7 * full(32):
            return "tile 64" if narrow < wide else "tile 128"
        one, two = (2.9, 3.8) if few else (4.0, 4.9)
        columns = 16 if one * rounds(16, 16) <= two * rounds(32, 16) else 32
    return f"{'few' if few else 'turned'} {columns}"


FORMS = [(F32, "few 16", 3, 3000), (F32, "few 32", 3, 6001), (F32, "few 64", 2, 8199), (F32, "turned 16", 17, 1001), (F32, "turned 32", 70, 1301),
         (F32, "turned 64", 300, 2050), (F32, "tile 128", 600, 1501), (F32, "tile 128", 130, 12290), (F32, "tile 128", 70, 9001),
         (BF16, "few 16", 4, 3003), (BF16, "few 32", 2, 5002), (BF16, "turned 16", 40, 1001), (BF16, "turned 32", 70, 9001),
         (BF16, "tile 64", 257, 2050), (BF16, "tile 64", 600, 1501), (BF16, "tile 64", 2000, 300), (BF16, "tile 128", 256, 4099),
         (BF16, "tile 128", 130, 12290), (BF16, "tile 128", 300, 6004)]


@pytest.mark.parametrize("dtype,form,rows,n", FORMS)
@pytest.mark.parametrize("k", [32, 224, 512, 544])
def test_every_form_against_float64(dev, dtype, form, rows, n, k):
    """Ragged rows, columns and K (whole steps of 256 are one of the four), with and without a bias."""
    from montlok import _C

    assert _form(rows, n, dtype) == form
    g = torch.Generator().manual_seed(rows + n + k)
    codes, scales = _weights(g, n, k)
    x = torch.randn(rows, k, generator=g).to(dtype)
    bias = torch.randn(n, generator=g) if k % 64 else None
    got = _C.linear_fp4(x.to(dev), codes.to(dev), scales.to(dev), None if bias is None else bias.to(dev))
    assert got.shape == (rows, n) and got.dtype == dtype
    _check(got, x, codes, scales, bias, dtype)


@pytest.mark.parametrize("dtype,form,rows,n", [f for f in FORMS if "tile" in f[1]])
def test_tiles_of_views_and_of_infinities(dev, dtype, form, rows, n):
    """Rows of any alignment give a copy's bits; infinities and NaN stay in their rows and columns, also in the last group
    of a K that ends inside a step."""
    from montlok import _C

    g = torch.Generator().manual_seed(rows * 3 + n)
    codes, scales = _weights(g, n, 160)
    codes |= 0x11  # no weight is zero: an infinity gives an infinity
    dc, ds = codes.to(dev), scales.to(dev)
    wide = torch.randn(rows, 171, generator=g).to(dtype)
    x = wide[:, 3:163].contiguous()
    clean = _C.linear_fp4(x.to(dev), dc, ds)
    for lead in (1, 2, 3, 8):
        moved = torch.roll(wide, lead - 3, 1).to(dev)[:, lead:lead + 160]
        assert torch.equal(_C.linear_fp4(moved, dc, ds), clean)
    same = x[:1].to(dev).expand(rows, 160)  # rows at a stride of 0
    assert torch.equal(_C.linear_fp4(same, dc, ds), _C.linear_fp4(same.contiguous(), dc, ds))
    x[0, 3], x[rows // 2, 100], x[rows - 1, 159] = torch.inf, -torch.inf, torch.nan
    scales[9, 2], scales[n - 1, 4] = 255, 255
    got, clean = _C.linear_fp4(x.to(dev), dc, scales.to(dev)).cpu(), clean.cpu()
    expect = x.double() @ ref.value_of(codes, scales).t()
    assert torch.equal(torch.isnan(got), torch.isnan(expect)) and torch.equal(torch.isinf(got), torch.isinf(expect))
    assert torch.equal(torch.sign(got[0, :9].double()), torch.sign(expect[0, :9]))
    rest, keep = torch.ones(rows, dtype=torch.bool), torch.ones(n, dtype=torch.bool)
    rest[[0, rows // 2, rows - 1]], keep[[9, n - 1]] = False, False
    assert torch.equal(got[rest][:, keep], clean[rest][:, keep])


@pytest.mark.parametrize("dtype,rows,n", [(BF16, 257, 2050), (F32, 70, 9001)])
@pytest.mark.parametrize("stride", [(1 << 24) - 1, 1 << 24])
def test_rows_far_apart(dev, dtype, rows, n, stride):
    """The widest stride that tiles address in 32 bits, and the first that goes to the other form."""
    from montlok import _C

    assert _form(rows, n, dtype, stride).startswith("tile") == (stride < 1 << 24) and _form(rows, n, dtype).startswith("tile")
    g = torch.Generator().manual_seed(n)
    codes, scales = _weights(g, n, 160)
    x = torch.randn(rows, 160, generator=g).to(dtype)
    far = torch.empty(rows * stride, dtype=dtype, device=dev).as_strided((rows, 160), (stride, 1)).copy_(x)
    _check(_C.linear_fp4(far, codes.to(dev), scales.to(dev)), x, codes, scales, None, dtype)


@pytest.mark.parametrize("dtype,rows,n", [(BF16, 257, 2050), (BF16, 256, 4099), (F32, 600, 1501)])
def test_tiles_in_a_graph(dev, dtype, rows, n):
    from montlok import _C

    assert _form(rows, n, dtype).startswith("tile")
    g = torch.Generator().manual_seed(rows)
    codes, scales = (t.to(dev) for t in _weights(g, n, 288))
    x = torch.zeros(rows, 288, dtype=dtype, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _C.linear_fp4(x, codes, scales)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _C.linear_fp4(x, codes, scales)
    for replay in range(4):
        x.copy_(torch.randn(x.shape, generator=g).to(dtype))
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, _C.linear_fp4(x, codes, scales)), f"replay {replay}"


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,n", [(3, 40), (40, 40), (600, 1501)])
def test_weights_past_the_largest_number(dev, dtype, rows, n):
    """Bytes 253 and 254: weights below 2^128 are exact, an output with a larger one is infinite or NaN, the others keep
    their bits."""
    from montlok import _C

    g = torch.Generator().manual_seed(rows)
    codes, scales = _weights(g, n, 96)
    x = (torch.randn(rows, 96, generator=g) * 2.0 ** -20).to(dtype)
    clean = _C.linear_fp4(x.to(dev), codes.to(dev), scales.to(dev)).cpu()
    scales[3, 1], scales[4, 2], scales[5, 2], scales[6, 0] = 253, 254, 253, 254
    codes[3, 16:32], codes[4, 32:48] = 0x75, 0x94  # 6 and 3 times 2^126; 2 and -0.5 times 2^127
    codes[5, 32:48], codes[6, :16] = 0xD5, 0x3B  # 3 times 2^126; 1.5 times 2^127: exact
    got = _C.linear_fp4(x.to(dev), codes.to(dev), scales.to(dev)).cpu()
    assert not torch.isfinite(got[:, 3:5]).any()
    _check(got[:, 5:7], x, codes[5:7], scales[5:7], None, dtype)
    rest = torch.ones(n, dtype=torch.bool)
    rest[3:7] = False
    assert torch.equal(got[:, rest], clean[:, rest])


@pytest.mark.parametrize("rows,n", [(2, 33), (40, 33), (600, 1501)])
@pytest.mark.parametrize("power", [-110, -111, -120, -132, -140, -148])
def test_the_smallest_inputs(dev, rows, n, power):
    """float32 values of one power of two, down to the subnormal ones: their parts are exact from 2^-110 on, and lose less
    than 2^-133 of a smaller value."""
    from montlok import _C

    g = torch.Generator().manual_seed(rows - power)
    codes, scales = _weights(g, n, 96, 220, 224)
    x = (1 + torch.rand(rows, 96, generator=g)).double() * (1 - 2.0 * torch.randint(0, 2, (rows, 96), generator=g)) * 2.0 ** power
    x = x.float()
    got = _C.linear_fp4(x.to(dev), codes.to(dev), scales.to(dev)).double().cpu()
    w = ref.value_of(codes, scales)
    bound = (3 * 96 + 8) * 2.0 ** -24 * (x.double().abs() @ w.abs().t())
    if power < -110:
        bound = bound + 2.0 ** -133 * w.abs().sum(1)
    assert ((got - x.double() @ w.t()).abs() <= bound).all()

"""Refusals of the 4-bit cache's operators that need no GPU: of the C ABI before any launch, and of montlok._C."""

from __future__ import annotations

import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from montlok import _C

    return _C.library()


def _cache(lib, name, head_dim=64, page_size=64, pages=4, width=2, kv_heads=2, batch=1, length=1, dtype=1, heads=4, scale=1.0):
    """One call with null tensors: the geometry is checked before the pointers."""
    if name == "append":
        status = lib.mlk_kv4_append(None, None, None, None, dtype, batch, length, kv_heads, head_dim, None, pages, page_size, None,
                                    width, None, None)
    elif name == "read":
        status = lib.mlk_kv4_read(None, pages, page_size, None, width, None, batch, length, kv_heads, head_dim, dtype, None, None, None)
    else:
        status = lib.mlk_kv4_attention(None, None, dtype, batch, length, heads, kv_heads, head_dim, None, pages, page_size, None, width,
                                       None, scale, None, None, 0, None)
    return status, lib.mlk_last_error().decode()


@pytest.mark.parametrize("name", ["append", "read", "attention"])
@pytest.mark.parametrize("change,text", [
    (dict(head_dim=48), "head_dim must be"), (dict(head_dim=0), "head_dim must be"), (dict(head_dim=512), "head_dim must be"),
    (dict(page_size=0), "page_size must be"), (dict(page_size=24), "page_size must be"), (dict(page_size=1040), "page_size must be"),
    (dict(page_size=-16), "page_size must be"),
    (dict(pages=0), "between 1 and"), (dict(pages=2 ** 31), "between 1 and"),
    (dict(width=0), "page_table must hold"), (dict(width=2 ** 24 + 1), "page_table must hold"),
    (dict(kv_heads=0), "invalid cache geometry"), (dict(batch=-1), "invalid cache geometry"), (dict(length=-1), "invalid cache geometry"),
    (dict(dtype=2), "dtype must be"), (dict(), "null tensor pointer"),
])
def test_cache_geometry_is_refused_before_a_launch(lib, name, change, text):
    status, message = _cache(lib, name, **change)
    assert status == 1 and text in message


@pytest.mark.parametrize("change,text", [
    (dict(heads=3), "multiple of kv_heads"), (dict(heads=0), "multiple of kv_heads"), (dict(heads=-2), "multiple of kv_heads"),
    (dict(length=2 ** 30), "too many tokens"),
])
def test_attention_geometry_is_refused_before_a_launch(lib, change, text):
    status, message = _cache(lib, "attention", **change)
    assert status == 1 and text in message


@pytest.mark.parametrize("name", ["append", "read", "attention"])
@pytest.mark.parametrize("change", [dict(batch=0), dict(length=0)])
def test_calls_without_tokens_do_nothing(lib, name, change):
    assert _cache(lib, name, **change)[0] == 0


def test_workspace_is_bounded_and_zero_for_what_is_refused(lib):
    size = lib.mlk_kv4_attention_workspace_bytes
    assert size(1, 1, 32, 8, 128, 64, 2048) > 0  # one long stream is split
    assert size(1024, 1, 32, 8, 128, 64, 2048) == 0  # many streams are not
    assert size(1, 1, 32, 8, 128, 64, 1) == 0
    for bad in ((0, 1, 32, 8, 128, 64, 64), (1, 1, 31, 8, 128, 64, 64), (1, 1, 32, 8, 48, 64, 64), (1, 1, 32, 8, 128, 0, 64),
                (1, 1, 32, 8, 128, 64, 0), (1, 1, 32, 8, 128, 64, 2 ** 40), (1, 0, 32, 8, 128, 64, 64), (1, 1, 32, 0, 128, 64, 64)):
        assert size(*bad) == 0
    for batch in (1, 3, 64):
        for length in (1, 7, 500):
            assert size(batch, length, 32, 8, 256, 16, 2 ** 26) <= 2 ** 28


def _norm(lib, dtype=0, rows=8, rope=4, batch=1, length=1, heads=2, kv_heads=1, dim=8):
    status = lib.mlk_qk_norm_rope(None, None, None, None, dtype, None, None, 1e-5, None, None, rows, rope, None, batch, length, heads,
                                  kv_heads, dim, None, None, None)
    return status, lib.mlk_last_error().decode()


@pytest.mark.parametrize("change,text", [
    (dict(rope=3), "rope_dim must be"), (dict(rope=10), "rope_dim must be"), (dict(rope=-2), "rope_dim must be"),
    (dict(dim=0), "head_dim must be"), (dict(dim=1025), "head_dim must be"), (dict(heads=0), "invalid norm geometry"),
    (dict(kv_heads=0), "invalid norm geometry"), (dict(rows=-1), "invalid norm geometry"), (dict(dtype=7), "dtype must be"),
    (dict(length=2 ** 34), "too many"), (dict(), "null tensor pointer"),
])
def test_norm_geometry_is_refused_before_a_launch(lib, change, text):
    status, message = _norm(lib, **change)
    assert status == 1 and text in message


def _linear(lib, rows=1, k=64, n=8, dtype=0, codes=None):
    status = lib.mlk_linear_fp4(None, rows, k, k, dtype, codes, None, None, n, None, None)
    return status, lib.mlk_last_error().decode()


@pytest.mark.parametrize("change,text", [
    (dict(k=0), "multiple of 32"), (dict(k=48), "multiple of 32"), (dict(n=0), "invalid linear"), (dict(rows=-1), "invalid linear"),
    (dict(dtype=3), "dtype must be"), (dict(rows=2 ** 31), "too many"), (dict(), "null tensor pointer"),
])
def test_linear_geometry_is_refused_before_a_launch(lib, change, text):
    status, message = _linear(lib, **change)
    assert status == 1 and text in message


def test_calls_without_rows_do_nothing(lib):
    assert _linear(lib, rows=0)[0] == 0
    assert _norm(lib, batch=0)[0] == 0 and _norm(lib, length=0)[0] == 0


def test_operators_refuse_host_tensors():
    from montlok import _C

    x, c, i = torch.ones(1, 1, 2, 32), torch.zeros(1, 2, 16 * 34, dtype=torch.uint8), torch.zeros(1, 1, dtype=torch.int32)
    for call, text in ((lambda: _C.qk_norm_rope(x, x, x, x, 1e-5, x, x, i), "q must be on the GPU"),
                       (lambda: _C.kv4_append(x, x, c, i, i), "k must be on the GPU"),
                       (lambda: _C.kv4_append(None, x, c, i, i), "k must be defined"),
                       (lambda: _C.kv4_read(c, i, i, 32), "cache must be on the GPU"),
                       (lambda: _C.kv4_read(c, i, i, 32, torch.float16), "dtype must be float32 or bfloat16"),
                       (lambda: _C.kv4_attention(x, c, i, i, 1.0), "q must be on the GPU"),
                       (lambda: _C.linear_fp4(x, c, c), "input must be on the GPU"),
                       (lambda: _C.linear_fp4(None, c, c), "input must be defined")):
        with pytest.raises(RuntimeError, match=text):
            call()


@pytest.mark.parametrize("args", [(4, 2, 64, 48), (4, 2, 24, 64), (4, 2, 0, 64), (0, 2, 64, 64), (4, 0, 64, 64), (4, 2, 2048, 64)])
def test_cache_allocation_is_refused(args):
    from montlok import _C

    with pytest.raises(RuntimeError):
        _C.kv4_cache(*args, device="cpu")


def test_cache_allocation():
    from montlok import _C

    cache = _C.kv4_cache(3, 2, 48, 64, device="cpu")
    assert cache.shape == (3, 2, 48 * 68) and cache.dtype == torch.uint8 and not cache.any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,k", [(1, 32), (7, 96), (33, 256)])
def test_weights_in_four_bits(dtype, n, k):
    """The nearest values of the format, by groups of every size, among them halves between codes, zeros, the smallest and
    largest numbers, infinities and NaN."""
    import kv4_reference as ref
    from montlok import _C

    g = torch.Generator().manual_seed(n + k)
    w = torch.randn(n, k, generator=g) * 2.0 ** torch.randint(-20, 20, (n, k // 32, 1), generator=g).expand(-1, -1, 32).flatten(1)
    w[0, :32] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 4) * torch.tensor([1.0, -1.0]).repeat(16)
    if n > 1:
        w[1, :32], w[2, :32], w[3, :32], w[4, 3], w[5, 40] = 0.0, 2.0 ** -140, 3e38, torch.inf, torch.nan
        w[6, :32] = w[0, :32] * 2.0 ** -124
    w = w.to(dtype)
    codes, scales = _C.fp4_weights(w)
    assert codes.shape == (n, k // 2) and scales.shape == (n, k // 32) and codes.dtype == scales.dtype == torch.uint8
    assert codes.is_contiguous() and scales.is_contiguous()
    assert torch.equal(ref.value_of(codes, scales).nan_to_num(nan=1e300), ref.nearest(w).nan_to_num(nan=1e300))
    nan = ~torch.isfinite(w).unflatten(1, (-1, 32)).all(-1)
    assert (scales[nan] == 255).all() and (scales[~nan] < 253).all()


@pytest.mark.parametrize("w", [torch.ones(4), torch.ones(4, 48), torch.ones(4, 0), torch.ones(0, 32), torch.ones(4, 32, dtype=torch.float16)])
def test_weights_that_do_not_fit_are_refused(w):
    from montlok import _C

    with pytest.raises(RuntimeError, match="weight must be"):
        _C.fp4_weights(w)


def test_calls_past_a_launch_are_refused(lib):
    """More threads than a grid holds, with pointers that nothing reads before the refusal."""
    memory = (C.c_uint8 * 64)()
    at = C.c_void_p((C.addressof(memory) + 15) & ~15)
    strides = (C.c_int64 * 3)(64, 64, 64)
    for status in (
            lib.mlk_kv4_append(at, strides, at, strides, 1, 1, 2 ** 26, 8, 64, at, 4, 64, at, 2, at, None),
            lib.mlk_kv4_read(at, 4, 64, at, 2, at, 1, 2 ** 26, 8, 64, 1, at, at, None),
            lib.mlk_kv4_attention(at, strides, 1, 1, 2 ** 24, 16, 16, 64, at, 4, 64, at, 2, at, 1.0, at, None, 0, None),
            lib.mlk_qk_norm_rope(at, strides, at, strides, 1, at, at, 1e-5, at, at, 8, 4, at, 1, 2 ** 22, 32, 8, 64, at, at, None),
            lib.mlk_linear_fp4(at, 2 ** 19, 64, 64, 1, at, at, None, 2 ** 16, at, None)):
        assert status == 1 and "too many" in lib.mlk_last_error().decode()


def test_negative_row_strides_are_refused(lib):
    memory = (C.c_uint8 * 64)()
    at = C.c_void_p((C.addressof(memory) + 15) & ~15)
    assert lib.mlk_linear_fp4(at, 2, 64, -64, 1, at, at, None, 8, at, None) == 1
    assert "x_stride" in lib.mlk_last_error().decode()


def test_attention_is_refused_by_blocks(lib):
    """2^23 blocks of up to 16 rows of a (sequence, key head), however few of the rows there are."""
    memory = (C.c_uint8 * 64)()
    at = C.c_void_p((C.addressof(memory) + 15) & ~15)
    strides = (C.c_int64 * 3)(64, 64, 64)
    for batch, length, heads, kv_heads in ((2 ** 20, 1, 32, 8), (2 ** 23, 1, 1, 1), (2 ** 19, 17, 8, 8), (2 ** 19 + 1, 1, 255, 15)):
        assert batch * kv_heads * -(-(length * heads // kv_heads) // 16) >= 2 ** 23
        assert lib.mlk_kv4_attention(at, strides, 1, batch, length, heads, kv_heads, 64, at, 4, 64, at, 2, at, 1.0, at, None, 0, None) == 1
        assert "too many" in lib.mlk_last_error().decode()

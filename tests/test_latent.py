"""Refusals of the latent attention's operators that need no GPU: of the C ABI before any launch, and of montlok._C; and the
frequencies of the rotation, which are formed on the host."""

from __future__ import annotations

import ctypes as C
import math

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from montlok import _C

    return _C.library()


def _cache(lib, name, rank=64, rope=16, page_size=64, pages=4, width=2, batch=1, length=1, dtype=1, store=2, heads=4, tree=False):
    """One call with null tensors: the geometry is checked before the pointers."""
    if name == "append":
        status = lib.mlk_latent_append(None, None, None, None, dtype, batch, length, rank, rope, None, store, pages, page_size, None, width,
                                       None, None)
    elif name == "read":
        status = lib.mlk_latent_read(None, store, pages, page_size, None, width, None, batch, length, rank, rope, dtype, None, None, None)
    else:
        status = lib.mlk_latent_attention(None, None, None, None, dtype, batch, length, heads, rank, rope, None, store, pages, page_size, None,
                                          width, None, 16 if tree else None, 1.0, None, None, 0, None)
    return status, lib.mlk_last_error().decode()


@pytest.mark.parametrize("name", ["append", "read", "attention"])
@pytest.mark.parametrize("change,text", [
    (dict(rank=48), "rank must be"), (dict(rank=0), "rank must be"), (dict(rank=1024), "rank must be"),
    (dict(rope=8), "rope_dim must be"), (dict(rope=0), "rope_dim must be"), (dict(rope=48), "rope_dim must be"), (dict(rope=128), "rope_dim must be"),
    (dict(page_size=0), "page_size must be"), (dict(page_size=65537), "page_size must be"), (dict(page_size=-16), "page_size must be"),
    (dict(pages=0), "pages must be"), (dict(pages=2 ** 31), "pages must be"),
    (dict(width=0), "page_table must hold"), (dict(width=2 ** 24), "page_table must hold"), (dict(width=2 ** 62), "page_table must hold"),
    (dict(batch=-1), "invalid cache geometry"), (dict(length=-1), "invalid cache geometry"), (dict(batch=2 ** 40), "invalid cache geometry"),
    (dict(dtype=2), "dtype must be"), (dict(store=0), "cache's dtype must be"), (dict(store=3), "cache's dtype must be"),
    (dict(), "null tensor pointer"),
])
def test_cache_geometry_is_refused_before_a_launch(lib, name, change, text):
    status, message = _cache(lib, name, **change)
    assert status == 1 and text in message


@pytest.mark.parametrize("name", ["append", "read"])
def test_copies_past_a_launch_are_refused(lib, name):
    assert "too many tokens" in _cache(lib, name, batch=2, length=2 ** 25)[1]
    assert "null tensor pointer" in _cache(lib, name, batch=1, length=2 ** 26 - 1)[1]


@pytest.mark.parametrize("change,text", [
    (dict(heads=0), "heads must be"), (dict(heads=65536), "heads must be"), (dict(heads=-2), "heads must be"),
    (dict(length=2 ** 30), "too many tokens"), (dict(length=2 ** 24), "too many tokens for one launch"),
    (dict(batch=2 ** 22), "too many tokens for one launch"), (dict(length=65, tree=True), "at most 64"),
])
def test_attention_geometry_is_refused_before_a_launch(lib, change, text):
    status, message = _cache(lib, "attention", **change)
    assert status == 1 and text in message


@pytest.mark.parametrize("name", ["append", "read", "attention"])
@pytest.mark.parametrize("change", [dict(batch=0), dict(length=0)])
def test_calls_without_tokens_do_nothing(lib, name, change):
    assert _cache(lib, name, **change)[0] == 0


def test_workspace_is_bounded_and_zero_for_what_is_refused(lib):
    size = lib.mlk_latent_attention_workspace_bytes
    assert size(1, 1, 16, 512, 64, 1, 2, 64, 2048) > 0  # one long stream is split
    assert size(2048, 1, 16, 512, 64, 1, 2, 64, 2048) == 0  # many streams are not
    assert size(1, 1, 16, 512, 64, 1, 2, 64, 1) == 0
    for bad in ((0, 1, 16, 512, 64, 1, 2, 64, 64), (1, 0, 16, 512, 64, 1, 2, 64, 64), (1, 1, 0, 512, 64, 1, 2, 64, 64), (1, 1, 16, 500, 64, 1, 2, 64, 64),
                (1, 1, 16, 512, 65, 1, 2, 64, 64), (1, 1, 16, 512, 64, 2, 2, 64, 64), (1, 1, 16, 512, 64, 1, 0, 64, 64),
                (1, 1, 16, 512, 64, 1, 2, 0, 64), (1, 1, 16, 512, 64, 1, 2, 64, 2 ** 40)):
        assert size(*bad) == 0
    for batch in (1, 3, 64):
        for length in (1, 7, 500):
            for dtype in (0, 1):
                assert size(batch, length, 128, 512, 64, dtype, 2, 16, 2 ** 24) <= 2 ** 30


def _rope(lib, dtype=0, rope=4, batch=1, length=1, heads=2, kv_heads=1, dim=8):
    status = lib.mlk_rope(None, None, None, None, dtype, None, rope, 0, 1.0, None, batch, length, heads, kv_heads, dim, None, None, None)
    return status, lib.mlk_last_error().decode()


@pytest.mark.parametrize("change,text", [
    (dict(dtype=2), "dtype must be"), (dict(rope=0), "rope_dim must be"), (dict(rope=3), "rope_dim must be"), (dict(rope=10), "rope_dim must be"),
    (dict(dim=0), "head_dim must be"), (dict(dim=1025), "head_dim must be"), (dict(heads=0), "invalid rotation geometry"),
    (dict(kv_heads=0), "invalid rotation geometry"), (dict(batch=-1), "invalid rotation geometry"), (dict(heads=2 ** 20), "too many heads"),
    (dict(batch=2 ** 16, length=2 ** 15), "too many tokens"), (dict(length=2 ** 28), "for one launch"), (dict(), "null tensor pointer"),
])
def test_rotation_geometry_is_refused_before_a_launch(lib, change, text):
    status, message = _rope(lib, **change)
    assert status == 1 and text in message


def _head(lib, tokens=1, heads=2, k=8, n=8, dtype=0, wtype=0, strides=(64, 8, 1), null=True):
    xs, ws = (C.c_int64 * 2)(16, 8), (C.c_int64 * 3)(*strides)
    status = lib.mlk_head_linear(None if null else 16, tokens, heads, k, xs, dtype, None if null else 16, ws, wtype, n, None if null else 16, None)
    return status, lib.mlk_last_error().decode()


@pytest.mark.parametrize("change,text", [
    (dict(dtype=2), "dtype must be"), (dict(dtype=1, wtype=0), "weight must be"), (dict(wtype=2), "weight must be"),
    (dict(tokens=-1), "geometry"), (dict(heads=0), "geometry"), (dict(k=0), "geometry"), (dict(n=0), "geometry"),
    (dict(heads=2 ** 20), "below 2^20"), (dict(k=2 ** 20), "below 2^20"), (dict(n=2 ** 20), "below 2^20"), (dict(tokens=2 ** 31), "too many tokens"),
    (dict(tokens=2 ** 30), "for one launch"), (dict(), "null tensor pointer"), (dict(null=False, strides=(64, 16, 2)), "dense along"),
])
def test_head_linear_geometry_is_refused_before_a_launch(lib, change, text):
    status, message = _head(lib, **change)
    assert status == 1 and text in message


def test_nothing_to_multiply(lib):
    assert _head(lib, tokens=0)[0] == 0


@pytest.mark.parametrize("call", [
    lambda c, t: c.rope(t, t, t, t), lambda c, t: c.latent_append(t, t, t, t, t), lambda c, t: c.latent_read(t, t, t, 64, 16),
    lambda c, t: c.latent_attention(t, t, t, t, t, 1.0), lambda c, t: c.head_linear(t, t)])
def test_tensors_on_the_cpu_are_refused(call):
    from montlok import _C

    with pytest.raises(RuntimeError, match="must be on the GPU"):
        call(_C, torch.zeros(1, 1, 1, 64))


def test_cache_arguments_are_refused():
    from montlok import _C

    for args, text in (((0, 16, 64, 16), "pages"), ((1, 0, 64, 16), "page_size"), ((1, 65537, 64, 16), "page_size"), ((1, 16, 65, 16), "rank"),
                       ((1, 16, 64, 8), "rope_dim"), ((1, 16, 64, 16, torch.float32), "dtype")):
        with pytest.raises(RuntimeError, match=text):
            _C.latent_cache(*args)
    assert _C.latent_cache(2, 3, 64, 16, device="cpu").shape == (2, 3, 64 + 32 + 16)
    assert _C.latent_cache(2, 3, 64, 16, torch.bfloat16, "cpu").shape == (2, 3, 2 * 80 + 16)
    with pytest.raises(RuntimeError, match="dtype"):
        _C.latent_read(torch.zeros(1, 1, 112, dtype=torch.uint8), None, None, 64, 16, torch.float16)


def test_frequencies():
    from montlok import _C

    for bad in (dict(rope_dim=0), dict(rope_dim=7), dict(rope_dim=8, theta=1.0), dict(rope_dim=8, factor=0.5),
                dict(rope_dim=8, factor=2.0, original_length=-1), dict(rope_dim=8, factor=2.0, original_length=10, fast=1.0)):
        with pytest.raises(RuntimeError):
            _C.rope_frequencies(device="cpu", **bad)
    plain, one = _C.rope_frequencies(64, device="cpu")
    assert one == 1.0 and plain.dtype == torch.float64
    assert all(abs(f - 10000.0 ** (-2 * i / 64)) <= 1e-15 * f for i, f in enumerate(plain.tolist()))
    linear, one = _C.rope_frequencies(64, factor=4.0, device="cpu")
    assert one == 1.0 and torch.equal(linear, plain / 4)
    # By parts: pairs that turn more than 32 times over 4096 positions are kept, those below once slowed down, the rest between.
    parts, magnitude = _C.rope_frequencies(64, factor=40.0, original_length=4096, device="cpu")
    assert abs(magnitude - (0.1 * math.log(40) + 1)) < 1e-15
    turns = 4096 * plain / (2 * math.pi)
    ratio = parts / plain
    assert (ratio[turns > 33] > 0.97).all() and torch.allclose(ratio[turns < 0.9], torch.tensor(1 / 40.0, dtype=torch.float64), rtol=1e-12)
    assert (ratio[1:] <= ratio[:-1] + 1e-15).all() and ((ratio < 0.97) & (ratio > 0.03)).sum() > 5
    assert torch.equal(_C.rope_frequencies(64, factor=1.0, original_length=4096, device="cpu")[0], plain)


@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf, 1e300, -3e38])
def test_scales_that_fp32_does_not_hold_are_refused(lib, scale):
    status = lib.mlk_latent_attention(None, None, None, None, 1, 1, 1, 4, 64, 16, None, 2, 4, 64, None, 2, None, None, scale, None, None, 0, None)
    assert status == 1 and "scale must be finite" in lib.mlk_last_error().decode()


@pytest.mark.parametrize("rope_dim,original", [(16, 32768), (64, 131072), (16, 500000), (16, 4096), (64, 4096), (128, 10 ** 6)])
@pytest.mark.parametrize("factor", [4.0, 40.0])
def test_frequencies_where_the_slowest_pair_still_turns(rope_dim, original, factor):
    """Every pair against the ramp written out from how often it turns: the fastest turns original / (2 pi) times, each next
    one theta^(2 / rope_dim) times less often. It ends where a pair would turn once, wherever the last pair lies."""
    from montlok import _C

    plain = _C.rope_frequencies(rope_dim, device="cpu")[0].tolist()
    got = _C.rope_frequencies(rope_dim, factor=factor, original_length=original, device="cpu")[0].tolist()
    fewer = math.log(10000.0) * 2 / rope_dim
    low = max(0, math.floor(math.log(original / (2 * math.pi) / 32) / fewer))
    high = math.ceil(math.log(original / (2 * math.pi)) / fewer)
    assert high < rope_dim
    for i, (f, y) in enumerate(zip(plain, got)):
        slowed = min(1.0, max(0.0, (i - low) / (high - low)))
        assert abs(y / f - (1 - slowed + slowed / factor)) <= 1e-13
        turns = original * f / (2 * math.pi)
        assert turns > 1 or abs(y / f * factor - 1) <= 1e-12
        assert turns <= 1 or y / f > 1 / factor + 1e-3


def test_frequencies_of_a_context_that_no_pair_turns_in_are_refused():
    from montlok import _C

    for bad in (dict(original_length=1), dict(original_length=6), dict(original_length=100, slow=16.0)):
        with pytest.raises(RuntimeError, match="original_length"):
            _C.rope_frequencies(16, factor=4.0, device="cpu", **bad)
    _C.rope_frequencies(16, factor=4.0, original_length=7, device="cpu")
    assert torch.equal(_C.rope_frequencies(16, original_length=1, device="cpu")[0], _C.rope_frequencies(16, device="cpu")[0])


@pytest.mark.parametrize("length,page_size,pages,size", [(480, 64, 8, 60), (512, 64, 8, 64), (20, 16, 2, 10), (33, 7, 5, 7), (5, 64, 1, 5), (1, 1, 1, 1)])
def test_pages_of_a_stream(length, page_size, pages, size):
    """Pages of one size that end with the stream where there are such, else of the size asked for."""
    from types import SimpleNamespace

    from montlok.rdt import MLAHIP

    m = MLAHIP(SimpleNamespace(d_model=64, n_heads=2, head_dim=32, nope_head_dim=16, rope_head_dim=16, kv_lora_rank=64, q_lora_rank=0))
    state = m.new_state(3, length, torch.float8_e4m3fn, page_size, "cpu")
    assert state["cache"].shape == (3 * pages, size, 64 + 32 + 16) and state["max_length"] == length
    assert state["page_table"].flatten().tolist() == list(range(3 * pages)) and state["length"].tolist() == [[0]] * 3

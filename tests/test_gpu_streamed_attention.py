"""A streamed attention layer of the operators with 4-bit weights and a 4-bit cache: projection, norm and rotation of the
heads, the cache, attention over it, projection."""

from __future__ import annotations

import pytest
import torch

import kv4_reference as ref
from test_gpu_linear_fp4 import _check as check_linear
from test_gpu_qk_norm import _check as check_norm, _reference as norm_reference

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
B, H, HKV, D, PAGE, WIDTH, EMBED = 2, 6, 2, 128, 64, 256, 192


class _Layer:
    def __init__(self, g, dev):
        from montlok import _C

        self.c, self.dev = _C, dev
        weight = lambda n, k: torch.randn(n, k, generator=g) * k ** -0.5
        self.w_in, self.b_in = _C.fp4_weights(weight((H + 2 * HKV) * D, EMBED)), torch.randn((H + 2 * HKV) * D, generator=g)
        self.w_out = _C.fp4_weights(weight(EMBED, H * D))
        self.norm = 1 + 0.2 * torch.randn(2, D, generator=g)
        angle = torch.arange(400)[:, None] * 10000.0 ** (-torch.arange(0, D, 2) / D)
        self.cos, self.sin = torch.cat([angle, angle], 1).cos(), torch.cat([angle, angle], 1).sin()
        # Room for many more tokens than there are: the chunks below then have waves that share the keys.
        self.table = torch.full((B, WIDTH), -1, dtype=torch.int32)
        self.table[:, :4] = torch.randperm(B * 4, generator=g).view(B, 4)
        for name in ("w_in", "w_out"):
            setattr(self, "d_" + name, [t.to(dev) for t in getattr(self, name)])
        for name in ("b_in", "norm", "cos", "sin", "table"):
            setattr(self, "d_" + name, getattr(self, name).to(dev))

    def cache(self):
        return self.c.kv4_cache(B * 4, HKV, PAGE, D, self.dev)

    def __call__(self, x, cache, at, keep=None):
        qkv = self.c.linear_fp4(x, *self.d_w_in, self.d_b_in).unflatten(-1, (H + 2 * HKV, D))
        q, k = self.c.qk_norm_rope(qkv[:, :, :H], qkv[:, :, H:H + HKV], self.d_norm[0], self.d_norm[1], 1e-6, self.d_cos, self.d_sin, at)
        self.c.kv4_append(k, qkv[:, :, H + HKV:], cache, self.d_table, at)
        seen = self.c.kv4_attention(q, cache, self.d_table, at, D ** -0.5)
        out = self.c.linear_fp4(seen.flatten(2), *self.d_w_out)
        if keep is not None:
            keep.update(qkv=qkv, q=q, k=k, seen=seen, out=out)
        return out


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_layer_step_by_step(dev, dtype):
    """A prompt in two chunks, then tokens one by one, one sequence shorter than the other: every operator's result against
    float64 from what it was given, the cache's contents against the nearest values of all keys and values so far."""
    g = torch.Generator().manual_seed(3)
    layer = _Layer(g, dev)
    cache = layer.cache()
    lengths, keys, values = [203, 130], [torch.zeros(0, HKV, D)] * B, [torch.zeros(0, HKV, D)] * B
    for begin, end in [(0, 110), (110, 200)] + [(i, i + 1) for i in range(200, 203)]:
        x = torch.randn(B, end - begin, EMBED, generator=g).to(dtype)
        at = torch.tensor([[i if i < n else -1 for i in range(begin, end)] for n in lengths], dtype=torch.int32)
        got = {}
        layer(x.to(dev), cache, at.to(dev), got)
        got = {name: t.cpu() for name, t in got.items()}
        check_linear(got["qkv"].flatten(2), x, *layer.w_in, layer.b_in, dtype)
        check_norm(got["q"], norm_reference(got["qkv"][:, :, :H], layer.norm[0], 1e-6, layer.cos, layer.sin, at), dtype)
        check_norm(got["k"], norm_reference(got["qkv"][:, :, H:H + HKV], layer.norm[1], 1e-6, layer.cos, layer.sin, at), dtype)
        for b in range(B):
            new = at[b] >= 0
            keys[b] = torch.cat([keys[b], got["k"][b, new].float()])
            values[b] = torch.cat([values[b], got["qkv"][b, new, H + HKV:].float()])
        kept, kept_values = ref.contents(cache, PAGE, D)
        for b in range(B):
            n = len(keys[b])
            pages = layer.table[b, :-(-n // PAGE)].long()
            for now, expect in ((kept, keys[b]), (kept_values, values[b])):
                assert torch.equal(now[pages].transpose(0, 1).flatten(1, 2)[:, :n].transpose(0, 1), ref.nearest(expect))
        out, size, spread = ref.attention(got["q"], kept, kept_values, layer.table, at, D ** -0.5)
        bound = ref.attention_bound(size, spread, out, end, D, dtype)
        assert ((got["seen"].double() - out).abs() <= bound).all()
        check_linear(got["out"], got["seen"].flatten(2), *layer.w_out, None, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("length", [1, 140])
def test_a_layer_in_a_graph(dev, dtype, length):
    """One captured layer, replayed on new tokens at further positions, against the eager layer on a copy of the cache."""
    g = torch.Generator().manual_seed(5 + length)
    layer = _Layer(g, dev)
    x, cache, eager = torch.zeros(B, length, EMBED, dtype=dtype, device=dev), layer.cache(), layer.cache()
    at = (torch.arange(length, dtype=torch.int32)[None] + torch.tensor([[3], [40]], dtype=torch.int32)).to(dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(x, layer.cache(), at)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(x, cache, at)
    for replay in range(4):
        x.copy_(torch.randn(x.shape, generator=g).to(dtype))
        at += min(length, 17)
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, layer(x, eager, at)) and torch.equal(cache, eager), f"replay {replay}"

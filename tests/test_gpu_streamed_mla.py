"""MLAHIP.step: the streamed layer of rope, latent_append, head_linear and latent_attention, against float64 and against the
module's whole-window forward."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

import latent_reference as ref

pytestmark = pytest.mark.gpu

F32, BF16, E4M3 = torch.float32, torch.bfloat16, torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def kernels_on(monkeypatch):
    monkeypatch.setenv("MONTLOK_CPP", "1")
    monkeypatch.delenv("MONTLOK_CPP_LAYERS", raising=False)


def _module(dev, heads=8, head_dim=32, nope=16, rank=64, q_rank=0, weights=F32, seed=0):
    from montlok.rdt import MLAHIP

    torch.manual_seed(seed)
    cfg = SimpleNamespace(d_model=heads * head_dim, n_heads=heads, head_dim=head_dim, nope_head_dim=nope, rope_head_dim=head_dim - nope,
                          kv_lora_rank=rank, q_lora_rank=q_rank)
    m = MLAHIP(cfg).eval()
    with torch.no_grad():
        m.kv_norm.weight.uniform_(0.5, 1.5)
        m.kv_norm.bias.uniform_(-0.3, 0.3)
    for name in ("q_proj", "q_down", "q_up", "kv_down", "kv_up", "k_rope_proj", "o_proj"):
        if hasattr(m, name):
            getattr(m, name).to(weights)
    return m.to(dev)


def _rows(state, stream, n):
    """What the cache holds of a stream's first n tokens, latents and key parts in float64."""
    cache = state["cache"].cpu()
    rows = cache[state["page_table"][stream].cpu().long()].flatten(0, 1)[:n]
    return rows


def _reference(m, x, latents, words):
    """The last len(x) tokens of a stream in float64, from what the cache holds of all of them."""
    w = lambda t: t.weight.detach().double().cpu()
    n, past = len(x), len(latents) - len(x)
    x = x.double().cpu()
    if m.q_lora_rank:
        down = x @ w(m.q_down).t()
        q = torch.nn.functional.layer_norm(down, (m.q_lora_rank,), w(m.q_norm), m.q_norm.bias.detach().double().cpu(), m.q_norm.eps) @ w(m.q_up).t()
    else:
        q = x @ w(m.q_proj).t()
    q = q.view(1, n, m.n_heads, m.head_dim)
    at = torch.arange(past, past + n)[None]
    turned = ref.rotate(q[..., m.nope_dim:], m.rope.freqs, at, False, 1.0)[0]
    kv = (latents @ w(m.kv_up).t()).view(-1, m.n_heads, m.nope_dim + m.head_dim)
    out = []
    for i in range(n):
        score = torch.einsum("hd,khd->hk", q[0, i, :, :m.nope_dim], kv[:past + i + 1, :, :m.nope_dim]) + turned[i] @ words[:past + i + 1].t()
        out.append(torch.einsum("hk,khd->hd", torch.softmax(score * m.scale, -1), kv[:past + i + 1, :, m.nope_dim:]).flatten())
    return torch.stack(out) @ w(m.o_proj).t()


@pytest.mark.parametrize("store", [BF16, E4M3])
@pytest.mark.parametrize("geometry", [dict(), dict(heads=4, head_dim=64, nope=32), dict(heads=3, head_dim=48, nope=32, rank=128, q_rank=40)])
def test_tokens_and_chunks_in_turn(dev, store, geometry):
    """A chunk, tokens one by one, another chunk across a page's end, against float64 from what the cache holds. The products
    are fp32 with K up to 144 terms, so that the layer's 6 steps stay under 1e-5 of its largest output (FP32_TOL)."""
    m = _module(dev, **geometry)
    g = torch.Generator().manual_seed(1)
    state, fed = m.new_state(2, 100, store, 16), 0
    xs = torch.zeros(2, 0, m.d_model)
    with torch.no_grad():
        for n in (13, 1, 1, 30, 1):
            x = torch.randn(2, n, m.d_model, generator=g)
            y = m.step(x.to(dev), state) if n > 1 else m.step(x[:, 0].to(dev), state)[:, None]
            xs, fed = torch.cat([xs, x], 1), fed + n
            assert y.shape == x.shape and state["length"].flatten().tolist() == [fed, fed]
            for b in range(2):
                latents, words = ref.contents(_rows(state, b, fed), m.kv_lora_rank, m.rope_dim, store)
                expect = _reference(m, x[b], latents, words)
                assert (y[b].double().cpu() - expect).abs().max() <= 1e-5 * expect.abs().max()
                # The cache holds the normed latents and the rotated key parts: to one step of their format and fp32's errors.
                down = xs[b].double() @ m.kv_down.weight.detach().double().cpu().t()
                normed = torch.nn.functional.layer_norm(down, (m.kv_lora_rank,), m.kv_norm.weight.detach().double().cpu(),
                                                        m.kv_norm.bias.detach().double().cpu(), m.kv_norm.eps)
                most = normed.abs().amax(-1, keepdim=True)
                step = 2.0 ** -8 if store == BF16 else 2.0 ** -4
                assert ((latents - normed).abs() <= step * normed.abs() * 1.001 + (1e-5 if store == BF16 else 2.0 ** -17) * most).all()
                key = (xs[b].double() @ m.k_rope_proj.weight.detach().double().cpu().t())[None, :, None]
                turned = ref.rotate(key, m.rope.freqs, torch.arange(fed)[None], False, 1.0)[0, :, 0]
                assert ((words - turned).abs() <= 2.0 ** -8 * turned.abs() * 1.001 + 1e-5 * turned.abs().max()).all()


@pytest.mark.parametrize("weights", [F32, BF16])
def test_a_stream_is_the_whole_windows_forward(dev, weights):
    """Token by token against ``forward``: off by what bf16 loses of the cached latents (2^-8 of a value in each of 64 of a
    score's and an output's terms, independent of each other) and, with bf16 weights, of ``forward``'s activations: the
    package's bound for bf16 (2e-2 of the largest output)."""
    m = _module(dev, weights=weights)
    x = torch.randn(3, 70, m.d_model, generator=torch.Generator().manual_seed(2)).to(dev)
    state = m.new_state(3, 70)
    with torch.no_grad():
        whole = m(x)
        stream = torch.stack([m.step(x[:, i], state) for i in range(70)], 1)
    assert (stream - whole).abs().max() <= 2e-2 * whole.abs().max()


def test_in_a_graph(dev):
    """A captured step replayed token by token, an eager twin beside it; bit for bit, the cache too."""
    m = _module(dev)
    g = torch.Generator().manual_seed(3)
    state, twin, other = (m.new_state(4, 40, E4M3, 8) for _ in range(3))
    x = torch.randn(4, m.d_model, generator=g).to(dev)
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            m.step(x, other)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = m.step(x, state)
        for i in range(12):
            x.copy_(torch.randn(4, m.d_model, generator=g))
            y.fill_(float("nan"))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, m.step(x, twin)) and torch.equal(state["cache"], twin["cache"])
            assert torch.equal(state["length"], twin["length"]) and state["length"][0].item() == i + 1


def test_past_the_end_and_refusals(dev):
    m = _module(dev)
    x = torch.randn(2, m.d_model, generator=torch.Generator().manual_seed(4)).to(dev)
    state = m.new_state(2, 16, page_size=16)
    with torch.no_grad():
        for _ in range(16):
            assert torch.isfinite(m.step(x, state)).all()
        assert torch.isnan(m.step(x, state)).all()
        with pytest.raises(ValueError, match="expects"):
            m.step(x[:, :-1], state)
        with pytest.raises(RuntimeError, match="positions must be"):  # three streams, a state of two
            m.step(x[:1].repeat(3, 1), state)
        with pytest.raises(RuntimeError, match="float32"):
            m.step(x.to(BF16), state)
    with pytest.raises(RuntimeError, match="inference only"):
        m.step(x, state)
    for bad in ((0, 16), (2, 0), (2, 16, BF16, 0)):
        with pytest.raises(ValueError):
            m.new_state(*bad)
    with pytest.raises(RuntimeError, match="rank must be"):
        _module(dev, rank=48).new_state(1, 16)


def test_no_tokens_leave_the_state(dev):
    m = _module(dev)
    x = torch.randn(2, 3, m.d_model, generator=torch.Generator().manual_seed(5)).to(dev)
    state, twin = m.new_state(2, 16), m.new_state(2, 16)
    with torch.no_grad():
        assert m.step(x[:, :0], state).shape == (2, 0, m.d_model)
        assert torch.equal(m.step(x, state), m.step(x, twin)) and torch.equal(state["cache"], twin["cache"])


@pytest.mark.parametrize("store", [BF16, E4M3])
@pytest.mark.parametrize("length,page_size", [(20, 16), (9, 64), (33, 7)])
def test_the_end_inside_a_page(dev, store, length, page_size):
    """max_length holds to the token where pages reach beyond it: token by token, in a chunk that passes it, and behind it.
    Against float64 from what the cache holds, as test_tokens_and_chunks_in_turn."""
    m = _module(dev)
    x = torch.randn(2, length + 5, m.d_model, generator=torch.Generator().manual_seed(6))
    state = m.new_state(2, length, store, page_size)
    cuts = [0, 4, 5, length - 2, length + 2, length + 5]
    with torch.no_grad():
        y = torch.cat([m.step(x[:, i:j].to(dev), state) for i, j in zip(cuts, cuts[1:])], 1)
        assert torch.isnan(y[:, length:]).all() and torch.isnan(m.step(x[:, 0].to(dev), state)).all()
    for b in range(2):
        latents, words = ref.contents(_rows(state, b, length), m.kv_lora_rank, m.rope_dim, store)
        expect = _reference(m, x[b, :length], latents, words)
        assert (y[b, :length].double().cpu() - expect).abs().max() <= 1e-5 * expect.abs().max()


@pytest.mark.parametrize("store", [BF16, E4M3])
def test_heads_that_are_rotated_whole(dev, store):
    """nope_head_dim 0, which forward has too: scores are of the key parts alone. Against float64 from what the cache holds, as
    test_tokens_and_chunks_in_turn, and against forward, as test_a_stream_is_the_whole_windows_forward."""
    m = _module(dev, nope=0)
    x = torch.randn(2, 20, m.d_model, generator=torch.Generator().manual_seed(7))
    state = m.new_state(2, 20, store, 16)
    with torch.no_grad():
        y = torch.cat([m.step(x[:, :19].to(dev), state), m.step(x[:, 19].to(dev), state)[:, None]], 1)
        whole = m(x.to(dev))
    for b in range(2):
        latents, words = ref.contents(_rows(state, b, 20), m.kv_lora_rank, m.rope_dim, store)
        expect = _reference(m, x[b], latents, words)
        assert (y[b].double().cpu() - expect).abs().max() <= 1e-5 * expect.abs().max()
    if store == BF16:
        assert (y - whole).abs().max() <= 2e-2 * whole.abs().max()


def test_frequencies_of_a_module_that_was_cast(dev):
    """Casting a module's weights casts its buffers as well; the rotation keeps its frequencies, as forward does."""
    m, cast = _module(dev, weights=BF16), _module(dev, weights=BF16).to(BF16)
    cast.kv_norm.float()
    cast.kv_norm.load_state_dict(m.kv_norm.state_dict())
    x = torch.randn(2, 30, m.d_model, generator=torch.Generator().manual_seed(8)).to(dev)
    state, other = m.new_state(2, 30), cast.new_state(2, 30)
    assert torch.equal(state["frequencies"], other["frequencies"])
    with torch.no_grad():
        assert torch.equal(m(x), cast(x)) and torch.equal(m.step(x, state), cast.step(x, other))

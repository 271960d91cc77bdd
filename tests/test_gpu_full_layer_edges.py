"""FullMultiHeadAttention over the life of a program: inference before training,
captured decoding, packed prompts in caches of their own size."""

import pytest
import torch

from full_attention_reference import rel
from test_gpu_full_attention import layer

pytestmark = pytest.mark.gpu


def test_training_after_inference_mode():
    """Tables formed under inference_mode serve a training step."""
    m = layer(64, torch.float32)
    x = torch.randn(1, 40, 96, device="cuda")
    with torch.inference_mode():
        want = m(x)
    y = m(x)
    y.square().sum().backward()
    assert torch.equal(y.detach(), want.clone()) and bool(m.in_proj.weight.grad.isfinite().all())


def prompt_and_graph(m, n, capacity, graph=True):
    """A cache with a prompt of n tokens, a token's input, and the captured step over it."""
    c = m.new_cache(2, capacity, torch.float32, "cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    with torch.no_grad():
        m(torch.randn(2, n, 96, generator=g, device="cuda"), cache=c)
    x = torch.randn(2, 1, 96, generator=g, device="cuda")
    if not graph:
        return c, x
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m.decode(x, c)
    torch.cuda.current_stream().wait_stream(side)
    cuda_graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(cuda_graph):
        y = m.decode(x, c)
    return c, x, cuda_graph, y


def test_a_captured_step_runs_to_the_end_of_its_cache():
    """Positions far past those that were known at the capture."""
    m = layer(64, torch.float32)
    c, x, g, y = prompt_and_graph(m, 5, 300)
    d, x2 = prompt_and_graph(m, 5, 300, graph=False)
    m.decode(x2, d)
    for _ in range(294):
        g.replay()
        want = m.decode(x2, d)
    torch.cuda.synchronize()
    assert c.lengths.tolist() == d.lengths.tolist() == [300, 300]
    # the replay's plan of splits is another: fp32 sums
    assert rel(y, want) <= 1e-5


def test_a_captured_step_keeps_its_tables():
    """A longer prompt through the layer, and memory taken and filled behind it,
    change nothing for a step that was captured before."""
    m = layer(64, torch.float32)
    c, x, g, y = prompt_and_graph(m, 50, 128)
    g.replay()
    torch.cuda.synchronize()
    want = y.clone()
    c.lengths -= 1
    with torch.no_grad():
        m(torch.randn(1, 3000, 96, device="cuda"))
    junk = [torch.full((1 << i,), float("nan"), device="cuda") for i in range(8, 22) for _ in range(4)]
    g.replay()
    torch.cuda.synchronize()
    assert len(junk) == 56 and torch.equal(y, want)


def test_tables_are_not_formed_in_a_capture():
    m = layer(64, torch.float32)
    x = torch.randn(1, 16, 96, device="cuda")
    with torch.no_grad():
        layer(64, torch.float32)(x)  # kernels and status word
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before a capture"):
        with torch.cuda.graph(g), torch.no_grad():
            m(x)
    torch.cuda.synchronize()
    with torch.no_grad():
        assert bool(m(x).isfinite().all())


def test_tables_are_there_for_any_stream():
    """Formed by a call on one stream, used at once by a call on another."""
    x = torch.randn(1, 4000, 96, device="cuda")
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    with torch.no_grad():
        for i in range(5):
            m = layer(64, torch.float32)
            torch.cuda.synchronize()
            with torch.cuda.stream(streams[0]):
                torch.cuda._sleep(20_000_000)
                m(x[:, :1])
                m(x)
            with torch.cuda.stream(streams[1]):
                y = m(x)
            torch.cuda.synchronize()
            assert torch.equal(y, m(x))


@pytest.mark.parametrize("store", ["int8", "fp8"])
def test_packed_prompts_longer_than_the_cache_together(store):
    """Eight prompts in a row of 520 tokens, a cache of 100 slots: each example has to
    fit, the row need not.  Then tokens, then the same cache for another batch."""
    from test_gpu_full_attention import layer as make

    m = make(64, torch.float32, cache_store=store)
    cache = m.new_cache(8, 100, torch.float32, "cuda")
    for lens in ([65] * 8, [95, 1, 40, 7, 95, 95, 95, 92]):
        cache.clear()
        assert cache.lengths.tolist() == [0] * 8 and cache.max_length == 0
        xs = [torch.randn(1, n + 3, 96, device="cuda") for n in lens]
        packed = torch.cat([x[:, :n] for x, n in zip(xs, lens)], 1)
        ids = torch.cat([torch.full((n,), i, device="cuda") for i, n in enumerate(lens)])[None]
        with torch.no_grad():
            m(packed, seq_idx=ids, cache=cache, max_tokens=max(lens))
            assert cache.lengths.tolist() == lens and cache.max_length == max(lens)
            full = [m(x) for x in xs]
            for s in range(3):
                out = m.decode(torch.cat([x[:, n + s: n + s + 1] for x, n in zip(xs, lens)]), cache)
                for i, n in enumerate(lens):  # as in test_layer_prompt_then_tokens
                    assert rel(out[i, 0], full[i][0, n + s]) <= (0.03 if store == "int8" else 0.08)
    with pytest.raises(ValueError, match="capacity"):
        m(packed, seq_idx=ids, cache=cache)  # the default bound is the row

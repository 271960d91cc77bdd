"""Captured steps of the cached attention: graphs that replay beside each other and
beside other calls, with the workspace of none of them.

A replay runs the kernels of the same call outside a graph on the same plan: equal
bits."""

import pytest
import torch

from test_gpu_kv_cache import rand

pytestmark = pytest.mark.gpu


def filled(seed, B=3, N=2900, H=4, D=128, room=400):
    """A cache of rows of different lengths that splits into many chunks, and a step's inputs."""
    from telescope_cache_b200 import init_kv_cache, write_kv_cache

    lengths = torch.tensor([N - 61 * seed, 1 + seed, N // 2])
    ids = torch.where(torch.arange(N) < lengths[:, None], torch.arange(B)[:, None], -1)
    c = init_kv_cache(B, N + room, H, D)
    write_kv_cache(c, rand(B, N, H, D, seed=seed), rand(B, N, H, D, seed=seed + 9), seq_idx=ids.cuda())
    return c, [rand(B, 1, h, D, dtype=torch.bfloat16, seed=20 + seed + h) for h in (16, H, H)]


def eager(c, x, steps):
    """Results of `steps` steps planned for the length at the first, as a replay is."""
    from telescope_cache_b200 import cached_attention_step

    most = c.max_length
    for _ in range(steps):
        c.max_length = most
        out, lse = cached_attention_step(*x, c)
    torch.cuda.synchronize()
    return out, lse, c.lengths.clone()


def test_two_graphs_of_one_stream_replay_on_two_streams():
    from telescope_cache_b200 import cached_attention_step

    capture, streams = torch.cuda.Stream(), [torch.cuda.Stream() for _ in range(2)]
    steps, graphs, kept, want = 200, [], [], []
    for seed in (1, 2):
        want.append(eager(*filled(seed), steps))
        c, x = filled(seed)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=capture):
            out, lse = cached_attention_step(*x, c)
        graphs.append(g)
        kept.append((c, x, out, lse))
    extra, ex = filled(3)
    extra_want = eager(*filled(3), steps)
    torch.cuda.synchronize()
    most = extra.max_length
    for _ in range(steps):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(capture):  # and calls outside a graph on the stream of the captures
            extra.max_length = most
            e = cached_attention_step(*ex, extra)
    torch.cuda.synchronize()
    for (c, _, out, lse), (o, l, n) in zip(kept + [(extra, None, *e)], want + [extra_want]):
        assert torch.equal(c.lengths, n) and torch.equal(out, o) and torch.equal(lse, l)


def test_the_usual_recipe_of_a_capture():
    """Warm up on a side stream, capture on the default capture stream, with more
    than one call in the graph."""
    from telescope_cache_b200 import cached_attention, cached_attention_step

    c, x = filled(4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cached_attention_step(*x, c, advance=False)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        first = cached_attention(x[0], c)
        out, lse = cached_attention_step(*x, c)
        second = cached_attention_step(*x, c)
    d, y = filled(4)
    for i in range(3):
        g.replay()
        n = d.max_length
        want = cached_attention(y[0], d)
        want_step = cached_attention_step(*y, d)
        want_second = cached_attention_step(*y, d)
        d.max_length = n
        torch.cuda.synchronize()
        assert torch.equal(c.lengths, d.lengths)
        for a, b in zip((*first, out, lse, *second), (*want, *want_step, *want_second)):
            assert torch.equal(a, b)


def test_nothing_to_attend_in_a_capture():
    from telescope_cache_b200 import cached_attention_step, init_kv_cache

    c = init_kv_cache(2, 10, 2, 64)
    x = [rand(0, 1, 2, 64, dtype=torch.bfloat16) for _ in range(3)]
    cached_attention_step(*x, c)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = cached_attention_step(*x, c)
    g.replay()
    torch.cuda.synchronize()
    assert out.shape == (0, 1, 2, 64) and lse.shape == (0, 1, 2) and c.lengths.tolist() == [0, 0]


def test_calls_of_a_graph_that_need_more_and_more():
    """Counts that grow inside a capture, and branches of a capture side by side."""
    from telescope_cache_b200 import cached_attention, init_kv_cache, write_kv_cache

    caches = []
    for B, H, N in ((1, 4, 300), (700, 8, 130), (2, 2, 700)):
        c = init_kv_cache(B, N, H, 64)
        write_kv_cache(c, rand(B, N, H, 64, seed=B), rand(B, N, H, 64, seed=B + 1))
        caches.append((c, rand(B, 1, 2 * H, 64, dtype=torch.bfloat16, seed=B + 2)))
    want = [cached_attention(q, c) for c, q in caches]
    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        got = [cached_attention(q, c) for c, q in caches]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            branch = [cached_attention(q, c) for c, q in reversed(caches)]
        again = [cached_attention(q, c) for c, q in caches]
        torch.cuda.current_stream().wait_stream(side)
    for _ in range(20):
        g.replay()
    torch.cuda.synchronize()
    for r in (got, branch[::-1], again):
        for (a, b), (o, l) in zip(r, want):
            assert torch.equal(a, o) and torch.equal(b, l)

"""GPU: the serving operators in CUDA graphs captured as torch.cuda.graph does
by default, on a stream of its own: every graph keeps its own counters and
partial results, whatever was captured, replayed or called beside it.

Compared bit for bit with eager calls, whose results do not depend on timing.
"""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _problem(cuda, lens, new, heads, kv_heads, dim, page, seed):
    import torch
    g = torch.Generator(device=cuda).manual_seed(seed)
    width = -(-max(lens) // page)
    pages = len(lens) * width
    kc, vc = (torch.randint(-127, 128, (pages, kv_heads, page, dim), generator=g, device=cuda).to(torch.int8)
              for _ in range(2))
    ks, vs = (torch.full((pages, kv_heads), 2.0 ** -6, device=cuda) for _ in range(2))
    i = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device=cuda)  # noqa: E731
    table = torch.randperm(pages, generator=g, device=cuda).to(torch.int32).view(len(lens), width)
    q = torch.randn(sum(new), heads, dim, generator=g, device=cuda).half()
    cu = i(np.concatenate([[0], np.cumsum(new)]))
    return dict(q=q, k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, block_table=table, kv_lens=i(lens), cu_tokens=cu,
                max_new=max(new), return_lse=True)


def _calls(cuda):
    """Calls whose items or rows are split over CTAs and joined: few rows, prompts, log probabilities."""
    import torch
    from exl3_b200.kv_cache import kv_attend
    from exl3_b200.logprobs import token_logprobs
    few = [_problem(cuda, [5000, 70, 900], [1, 1, 1], 8, 2, 128, 16, s) for s in (0, 1)]
    many = [_problem(cuda, [900, 1700], [300, 650], 8, 2, d, 32, d) for d in (64, 128)]
    logits = [torch.randn(3, 120001, device=cuda) * 3 for _ in range(2)]
    tok = torch.tensor([1, 2, 3], device=cuda)
    return [[lambda p=p: kv_attend(**p) for p in few], [lambda p=p: kv_attend(**p) for p in many],
            [lambda x=x: token_logprobs(x, tok, top=20) for x in logits]]


def _dirty_pool(cuda):
    """A graph memory pool whose free memory holds ones."""
    import torch
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for n in (1 << 19, 1 << 21, 1 << 23, 1 << 25, 3 << 25):
            torch.full((n,), 0x01010101, dtype=torch.int32, device=cuda)
    graph.replay()
    torch.cuda.synchronize()
    return graph


def _same(a, b):
    import torch
    return all(torch.equal(x, y) for x, y in zip(a, b))


def _clear(outs):
    for o in outs:
        o.zero_()


@pytest.mark.parametrize("kind", ["few rows", "prompts", "log probabilities"])
def test_graphs_on_the_default_capture_stream(native, cuda, kind):
    """Warm-up on the current stream; the later graph replayed first, then both in turn, with eager calls between."""
    import torch
    calls = _calls(cuda)[["few rows", "prompts", "log probabilities"].index(kind)]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    dirt = _dirty_pool(cuda)
    graphs, outs = [], []
    for c in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], pool=dirt.pool()):
            outs.append(c())
    for i in (1, 0, 1, 1, 0, 0, 1):
        _clear(outs[i])
        graphs[i].replay()
        torch.cuda.synchronize()
        assert _same(outs[i], want[i]), i
        assert _same(calls[1 - i](), want[1 - i])


def test_graphs_run_beside_one_another(native, cuda):
    """Graphs captured on one stream and replayed on several, beside eager calls on another."""
    import torch
    calls = [c for kind in _calls(cuda) for c in kind]
    want = [c() for c in calls]
    graphs, outs = [], []
    for c in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(c())
    streams = [torch.cuda.Stream(cuda) for _ in graphs]
    for _ in range(20):
        for o in outs:
            _clear(o)
        for s, g in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        eager = [c() for c in calls]
        torch.cuda.synchronize()
        for o, e, w in zip(outs, eager, want):
            assert _same(o, w) and _same(e, w)


def test_a_whole_step_in_a_graph(native, cuda):
    """Plan, append, attend and log probabilities of one step in one graph, replayed as the cache grows."""
    import torch
    from exl3_b200.kv_cache import Exl3KvCache
    from exl3_b200.logprobs import token_logprobs
    n, heads = 3, 2
    caches = [Exl3KvCache(1, 90, heads, 64, requests=n, max_len=400, page_size=16, device=cuda) for _ in range(2)]
    new = torch.ones(n, dtype=torch.int32, device=cuda)
    k, v, q = (torch.zeros(n, h, 64, dtype=torch.bfloat16, device=cuda) for h in (heads, heads, 6))
    head = torch.randn(6 * 64, 90001, device=cuda).bfloat16()

    def step(cache):
        plan = cache.plan(new, n)
        cache.append(0, k, v, plan)
        y = cache.attend(0, q, plan, 1)
        cache.commit(plan)
        return (y, *token_logprobs(y.flatten(1) @ head, torch.zeros(n, dtype=torch.int64, device=cuda), top=5))

    step(Exl3KvCache(1, 90, heads, 64, requests=n, max_len=400, page_size=16, device=cuda))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(caches[0])
    g = torch.Generator(device=cuda).manual_seed(0)
    for _ in range(300):
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=g, device=cuda))
        graph.replay()
        assert _same(out, step(caches[1]))
    assert caches[0].lens.tolist() == [300] * n


def test_status_survives_replays(native, cuda):
    """A status recorded by an eager call, or by a replay, stands until it is read."""
    import torch
    from exl3_b200.kv_cache import kv_attend
    good, bad = _calls(cuda)[0][0], _problem(cuda, [5000, 70, 900], [1, 1, 1], 8, 2, 128, 16, 3)
    bad["block_table"][0, 3] = -1
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    kv_attend(**bad)
    good()
    assert native.device_status(clear=True) == 7
    for g, call in zip(graphs, (good, lambda: kv_attend(**bad))):
        with torch.cuda.graph(g):
            call()
    assert native.device_status(clear=True) == 0
    kv_attend(**bad)
    graphs[0].replay()
    assert native.device_status(clear=True) == 7
    graphs[0].replay()
    assert native.device_status(clear=True) == 0
    graphs[1].replay()
    graphs[0].replay()
    assert native.device_status(clear=False) == 7 and native.device_status(clear=True) == 7
    assert native.device_status(clear=True) == 0


def test_workspaces_return_when_their_graph_is_gone(native, cuda):
    """Capturing again and again does not use more and more memory."""
    import gc
    import time

    import torch
    from exl3_b200 import _native
    calls = [kind[0] for kind in _calls(cuda)]
    want = [c() for c in calls]

    def once():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = [c() for c in calls]
        graph.replay()
        torch.cuda.synchronize()
        assert all(_same(o, w) for o, w in zip(outs, want))

    sizes = []
    for _ in range(6):
        once()
        gc.collect()
        time.sleep(0.1)  # the driver tells of a destroyed graph on a thread of its own
        sizes.append(sum(b.numel() for b in _native.device_workspaces(cuda)))
    assert sizes[-1] == sizes[2], sizes


def test_a_call_that_does_not_fit_grows_within_a_capture(native, cuda):
    """A small call first, a larger one after it in the same capture, without any call before."""
    import torch
    few, many, lp = (kind[1] for kind in _calls(cuda))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [lp(), few(), many(), few(), lp()]
    for _ in range(3):
        for o in outs:
            _clear(o)
        graph.replay()
        torch.cuda.synchronize()
        for o, c in zip(outs, (lp, few, many, few, lp)):
            assert _same(o, c())


def test_counters_are_renewed_after_a_wait_ran_out(native, cuda):
    """Items given up leave their counters; clearing the status makes the workspace fit again, captured ones too.
    The state is written by hand."""
    import torch
    from exl3_b200 import _native
    calls = [c for kind in _calls(cuda) for c in kind]
    want = [c() for c in calls]
    graphs, outs = [], []
    for c in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(c())
    torch.cuda.synchronize()
    assert native.device_status(clear=True) == 0
    for buf in _native._serve_buffers:
        buf[:4].view(torch.int32).fill_(4)
        buf[256:2048].view(torch.int32).fill_(1)  # as after a piece that was counted and one that was not
    assert native.device_status(clear=False) == 4 and native.device_status(clear=True) == 4
    assert native.device_status(clear=True) == 0
    for g, o, c, w in zip(graphs, outs, calls, want):
        _clear(o)
        g.replay()
        assert _same(c(), w)
        torch.cuda.synchronize()
        assert _same(o, w)

"""GPU: the paged 8-bit cache (plan, append, attend) against its 64-bit plain forms.

Plan and append are exact: whole numbers, power-of-two scales, one rounding.

Attention, per output value, with p its weights and u the unit roundoff of the
output type (2^-8 bf16, 2^-11 f16):
  u |out|                         the output's rounding
  (2^-11 + 2^-13) sum p |v|       weights enter the product in f16 (2^-11 each); 2^-13 covers
                                  the exponential (2^-22) and scores in fp32 below
  n 2^-24 max |v|                 weights below f16's normal range, n keys
and for lse: D 2^-23 max_j sum |q k| scale (fp32 dot product) + 2^-17 (1 + |lse|).
"""

import numpy as np
import pytest
import serving_ref as ref

pytestmark = pytest.mark.gpu

U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def _torch():
    import torch
    return torch, {"bf16": torch.bfloat16, "f16": torch.float16}, {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def _kv():
    from exl3_b200 import kv_cache
    return kv_cache


# --- plan -------------------------------------------------------------------

def _run_plan(cuda, lens, new, table, free, cursor, page, n_tokens):
    import torch
    t = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device=cuda)  # noqa: E731
    tab = t(table)
    p = _kv().kv_plan(t(lens), t(new), tab, t(free), t([cursor]), page_size=page, n_tokens=n_tokens)
    again = _kv().kv_plan(t(lens), t(new), tab, t(free), t([cursor]), page_size=page, n_tokens=n_tokens)
    for x, y in zip(p, again):
        assert torch.equal(x, y)  # nothing it reads is changed
    got = [x.cpu().numpy() for x in p]
    want = ref.plan(list(lens), list(new), np.asarray(table), list(free), cursor, page, n_tokens)
    for name, g, w in zip(("kv_lens", "cu", "positions", "slots", "cursor"), got, want):
        assert np.array_equal(g, w if name != "cursor" else [w]), name
    assert np.array_equal(tab.cpu().numpy(), want[5])


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("B", [1, 3, 64, 513, 1500])
def test_plan(native, cuda, page, B):
    rng = np.random.default_rng(B + page)
    lens = rng.integers(0, 5 * page, B)
    lens[: min(B, 4)] = [0, page, page - 1, 2 * page + 1][: min(B, 4)]
    new = rng.integers(0, 3, B) if B > 64 else rng.integers(0, 2 * page + 2, B)
    width = 9
    table = rng.permutation(B * width).reshape(B, width)
    free = rng.permutation(5000)[: B * 4 + 8]
    for extra in (0, 37):
        _run_plan(cuda, lens, new, table, free, 5, page, int(new.sum()) + extra)


def test_plan_single_tokens_and_nothing(native, cuda):
    table = np.full((4, 3), -1)
    _run_plan(cuda, [0, 15, 16, 17], [1, 1, 1, 1], table, list(range(50, 60)), 0, 16, 4)
    _run_plan(cuda, [0, 15, 16, 17], [0, 0, 0, 0], table, [], 0, 16, 0)
    _run_plan(cuda, [], [], np.zeros((0, 3)), [1, 2], 1, 16, 0)


def test_plan_out_of_pages_and_table(native, cuda):
    """What runs out gives slots of -1 and status 7; the rest stands."""
    for table, free in ((np.full((2, 6), -1), [7, 8, 9]), (np.full((2, 2), -1), list(range(10, 20)))):
        _run_plan(cuda, [0, 0], [40, 40], table, free, 0, 16, 80)
        assert native.device_status(clear=True) == 7
    import torch
    one = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    p = _kv().kv_plan(one([4, 2]), one([3, 3]), one([[0], [1]]), one([]), one([0]), page_size=16, n_tokens=4)
    assert p.cu_tokens.tolist() == [0, 3, 4] and p.slots.tolist() == [4, 5, 6, 18]  # fewer rows than new tokens
    assert native.device_status(clear=True) == 7


# --- append -----------------------------------------------------------------

def _cache(cuda, pages, heads, page, dim, code, seed=0):
    """(codes tensor, scales tensor) filled with random codes and power-of-two scales."""
    torch, _, codes = _torch()
    g = torch.Generator(device=cuda).manual_seed(seed)
    x = torch.randn(pages, heads, page, dim, generator=g, device=cuda)
    x = (x * (90.0 if code == "e4m3" else 35.0)).clamp(-ref.QMAX[code], ref.QMAX[code])
    c = x.to(codes[code]) if code == "e4m3" else x.round().to(torch.int8)
    s = 2.0 ** torch.randint(-9, -4, (pages, heads), generator=g, device=cuda).float()
    return c, s


def _check_append(cuda, k, v, slots, dim, page, heads, code, pages=40):
    import torch
    kc, ks = _cache(cuda, pages, heads, page, dim, code, 1)
    vc, vs = _cache(cuda, pages, heads, page, dim, code, 2)
    want = [ref.append(x.float().cpu().numpy(), slots, c.float().cpu().numpy(), s.cpu().numpy(), code, other)
            for x, c, s, other in ((k, kc, ks, v.float().cpu().numpy()), (v, vc, vs, None))]
    _kv().kv_append(k, v, torch.tensor(slots, device=cuda), kc, vc, ks, vs)
    for (wc, ws), c, s in zip(want, (kc, vc), (ks, vs)):
        assert np.array_equal(s.cpu().numpy(), ws)
        assert np.array_equal(c.float().cpu().numpy(), wc, equal_nan=True)


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("x", ["bf16", "f16"])
@pytest.mark.parametrize("page,dim,heads", [(16, 128, 4), (32, 64, 3), (64, 128, 1), (128, 64, 2)])
def test_append(native, cuda, code, x, page, dim, heads):
    """Whole pages, part pages, single tokens joining pages (their scale growing or not), skipped rows."""
    torch, kinds, _ = _torch()
    rng = np.random.default_rng(page + dim)
    order = rng.permutation(40)
    slots, at = [], 0
    for start, n in ((0, 2 * page + 5), (3, 1), (page - 1, 2), (0, 1), (page // 2, page), (1, page - 1), (0, page)):
        s = start
        while n:
            m = min(n, page - s)
            slots += [int(order[at]) * page + s + i for i in range(m)]
            at, n, s = at + 1, n - m, 0
        slots.append(-1)
    slots = np.array(slots)
    T = len(slots)
    gain = np.exp2(rng.integers(-6, 7, (T, heads, 1)))
    mk = lambda: torch.tensor(rng.standard_normal((T, heads, dim)) * gain, device=cuda).to(kinds[x])  # noqa: E731
    _check_append(cuda, mk(), mk(), slots, dim, page, heads, code)


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_append_values(native, cuda, code):
    """Zeros, the range's ends, ties between codes, infinities, NaN, tiny and huge rows."""
    import torch
    q = ref.QMAX[code]
    rows = torch.zeros(12, 2, 64, dtype=torch.bfloat16, device=cuda)
    rows[1] = q
    rows[2] = -q
    rows[3, :, :8] = torch.tensor([q, 2.5, 3.5, 0.5, 1.5, -2.5, 17.0, 0.001953125]).bfloat16()
    rows[4, :, 3] = float("inf")
    rows[5, :, 4] = float("-inf")
    rows[6, :, 5] = float("nan")
    rows[6, :, 6] = 3.0
    rows[7] = 1e-30
    rows[8] = 3e38
    rows[9] = 449.0
    rows[10, 0] = 1.75
    rows[10, 1] = 1.7578125
    rows[11] = float("nan")
    slots = np.arange(12) * 16          # each the first of its page
    _check_append(cuda, rows, -rows, slots, 64, 16, 2, code)
    _check_append(cuda, rows, rows.flip(0), slots, 64, 16, 2, code)  # K and V have their NaN in other tokens
    _check_append(cuda, rows, -rows, slots + 5, 64, 16, 2, code)  # each joins a page
    _check_append(cuda, rows, -rows, np.arange(12) + 32, 64, 16, 2, code)  # all of one page


def test_append_strided_and_bad_slots(native, cuda):
    """Slices of a fused projection, offsets that force a copy, slots past the cache (status 7)."""
    import torch
    g = torch.Generator(device=cuda).manual_seed(3)
    fused = torch.randn(50, 14, 64, generator=g, device=cuda).half()
    slots = np.arange(50) + 16
    _check_append(cuda, fused[:, 8:11], fused[:, 11:], slots, 64, 16, 3, "int8")
    wide = torch.randn(50, 3, 67, generator=g, device=cuda).half()
    _check_append(cuda, wide[:, :, 1:65], wide[:, :, 3:], slots, 64, 16, 3, "int8")
    turned = torch.randn(3, 50, 64, generator=g, device=cuda).half().transpose(0, 1)
    _check_append(cuda, turned, turned, slots, 64, 16, 3, "e4m3")
    slots[-4:] = [40 * 16, 40 * 16 + 1, 1 << 40, (1 << 40) + 1]
    _check_append(cuda, turned, turned, slots, 64, 16, 3, "e4m3")
    assert native.device_status(clear=True) == 7


# --- attend -----------------------------------------------------------------

def _problem(cuda, lens, new, *, heads, kv_heads, dim, page, x, code, seed=0, extra_rows=0, gain=1.0):
    torch, kinds, _ = _torch()
    rng = np.random.default_rng(seed)
    width = max(1, -(-max(lens) // page)) + 1
    pages = sum(-(-n // page) for n in lens) + 3
    kc, ks = _cache(cuda, pages, kv_heads, page, dim, code, seed + 1)
    vc, vs = _cache(cuda, pages, kv_heads, page, dim, code, seed + 2)
    table = np.full((len(lens), width), -1)
    order, at = rng.permutation(pages), 0
    for b, n in enumerate(lens):
        m = -(-n // page)
        table[b, :m] = order[at:at + m]
        at += m
    cu = np.concatenate([[0], np.cumsum(new)])
    g = torch.Generator(device=cuda).manual_seed(seed)
    q = (torch.randn(int(cu[-1]) + extra_rows, heads, dim, generator=g, device=cuda) * gain).to(kinds[x])
    return dict(q=q, kc=kc, vc=vc, ks=ks, vs=vs, table=table, lens=np.array(lens), cu=cu, max_new=max(max(new), 1))


def _attend(cuda, p, window=0, scale=None, cu="given"):
    import torch
    i = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    return _kv().kv_attend(p["q"], p["kc"], p["vc"], p["ks"], p["vs"], i(p["table"]), i(p["lens"]),
                           cu_tokens=i(p["cu"]) if cu == "given" else cu, max_new=p["max_new"], window=window,
                           scale=scale, return_lse=True)


def _values(c, s):
    return np.nan_to_num(c.float().cpu().numpy().astype(np.float64)) * s.cpu().numpy()[:, :, None, None]


def _check_attend(cuda, p, x, window=0, scale=None, **kw):
    out, lse = _attend(cuda, p, window, scale, **kw)
    D = p["q"].shape[2]
    q = p["q"].float().cpu().numpy().astype(np.float64)
    want, wlse, amp, vmax, smax = ref.attend(np.nan_to_num(q), (_values(p["kc"], p["ks"]), _values(p["vc"], p["vs"])),
                                             p["table"], p["lens"], p["cu"], D ** -0.5 if scale is None else scale, window)
    got = out.float().cpu().numpy().astype(np.float64)
    n = max(int(p["lens"].max()), 1)
    tol = U[x] * np.abs(want) + (2.0 ** -11 + 2.0 ** -13) * amp + n * 2.0 ** -24 * vmax + (2.0 ** -25 if x == "f16" else 0)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), f"{bad.sum()} of {bad.size}, worst {np.nanmax(np.abs(got - want) / np.maximum(tol, 1e-30)):.2f} of tol"
    glse = lse.cpu().numpy().astype(np.float64)
    empty = np.isinf(wlse)
    assert np.array_equal(np.isneginf(glse), empty)
    ltol = D * 2.0 ** -23 * smax + 2.0 ** -17 * (1 + np.abs(np.where(empty, 0, wlse)))
    assert (np.abs(np.where(empty, 0, glse) - np.where(empty, 0, wlse)) <= ltol).all()
    assert not got[np.broadcast_to(empty[:, :, None], got.shape)].any()  # rows that see nothing are zeros
    return out, lse


SHAPES = [  # heads, kv_heads, dim, page
    (8, 1, 128, 16), (8, 2, 128, 32), (3, 3, 64, 16), (12, 1, 128, 64), (10, 2, 64, 128), (32, 2, 64, 32), (24, 1, 128, 16),
]


@pytest.mark.parametrize("x,code", [("bf16", "e4m3"), ("f16", "int8"), ("f16", "e4m3"), ("bf16", "int8")])
@pytest.mark.parametrize("heads,kv_heads,dim,page", SHAPES)
def test_attend_single_tokens(native, cuda, heads, kv_heads, dim, page, x, code):
    """One row per request: lengths 0, 1, page edges, tile edges, a few hundred."""
    lens = [0, 1, 15, 16, 17, page, page + 1, 127, 128, 129, 333, 700]
    p = _problem(cuda, lens, [1] * len(lens), heads=heads, kv_heads=kv_heads, dim=dim, page=page, x=x, code=code)
    _check_attend(cuda, p, x)
    _check_attend(cuda, p, x, cu=None)


@pytest.mark.parametrize("x,code", [("bf16", "e4m3"), ("f16", "int8")])
@pytest.mark.parametrize("heads,kv_heads,dim,page", SHAPES)
def test_attend_several_tokens(native, cuda, heads, kv_heads, dim, page, x, code):
    """Rows 0 to a few hundred per request in one call, whole prompts among them, a window, rows of no request."""
    lens = [0, 5, 40, 300, 257, 129, 64, 1]
    new = [0, 5, 3, 2, 200, 129, 1, 1]
    p = _problem(cuda, lens, new, heads=heads, kv_heads=kv_heads, dim=dim, page=page, x=x, code=code, extra_rows=4)
    p["q"][-4:] = float("nan")
    for window in (0, 1, 50):
        out, lse = _check_attend(cuda, p, x, window=window)
        assert not out[-4:].any() and bool((lse[-4:] == -float("inf")).all())


@pytest.mark.parametrize("x,code", [("bf16", "int8"), ("f16", "e4m3")])
@pytest.mark.parametrize("dim", [64, 128])
def test_attend_long(native, cuda, dim, x, code):
    """A few long requests: the keys are split over the card and joined; windows that start inside a tile."""
    for lens, new, window in (([5000, 33], [1, 1], 0), ([9000], [3], 0), ([7001, 4096], [2, 40], 1111)):
        p = _problem(cuda, lens, new, heads=4, kv_heads=1, dim=dim, page=32, x=x, code=code)
        _check_attend(cuda, p, x, window=window)


@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 1, 128), (12, 4, 64)])
def test_attend_shares(native, cuda, heads, kv_heads, dim):
    """Items of one and of many steps: the card's shares begin and end at an item's edge, inside it, or have no step at all."""
    lens = [700, 333, 64, 450]
    p = _problem(cuda, lens, lens, heads=heads, kv_heads=kv_heads, dim=dim, page=16, x="f16", code="e4m3")
    for window in (0, 75):
        _check_attend(cuda, p, "f16", window=window)
    lens = [1 + (37 * i * i) % 600 for i in range(150)]
    p = _problem(cuda, lens, [1] * len(lens), heads=heads, kv_heads=kv_heads, dim=dim, page=32, x="bf16", code="int8")
    _check_attend(cuda, p, "bf16")


def test_attend_repeats_streams_graph(native, cuda):
    """Bit-equal repeats, on other streams and from a CUDA graph."""
    import torch
    p = _problem(cuda, [3000, 70, 900], [1, 1, 1], heads=8, kv_heads=2, dim=128, page=16, x="bf16", code="e4m3")
    first = _attend(cuda, p)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(cuda) for _ in range(3)]
    outs = []
    for _ in range(4):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                outs.append(_attend(cuda, p))
    torch.cuda.synchronize()
    assert all(torch.equal(o[0], first[0]) and torch.equal(o[1], first[1]) for o in outs)
    i = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    table, lens = i(p["table"]), i(p["lens"])
    s = streams[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        run = lambda: _kv().kv_attend(p["q"], p["kc"], p["vc"], p["ks"], p["vs"], table, lens)  # noqa: E731
        run()
        with torch.cuda.graph(graph, stream=s):
            got = run()
    for _ in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, first[0])


def test_attend_strided_q_and_scale(native, cuda):
    """q as a slice of a fused projection and as a view that needs a copy; another softmax scale; large and tiny q."""
    import torch
    for dim in (64, 128):
        p = _problem(cuda, [200, 31], [1, 4], heads=6, kv_heads=2, dim=dim, page=16, x="bf16", code="e4m3")
        fused = torch.randn(5, 11, dim, device=cuda).bfloat16()
        p["q"] = fused[:, 2:8]
        _check_attend(cuda, p, "bf16", scale=0.3)
        p["q"] = torch.randn(5, 6, dim + 1, device=cuda).bfloat16()[:, :, 1:]
        _check_attend(cuda, p, "bf16")
        for gain in (2.0 ** -100, 2.0 ** -14, 30.0):
            p["q"] = (torch.randn(5, 6, dim, device=cuda) * gain).bfloat16()
            _check_attend(cuda, p, "bf16")


def test_attend_ignores_what_it_may_not_see(native, cuda):
    """NaN codes past a request's end, in other pages and behind the table's used part do not reach the output."""
    import torch
    for new in ([1, 1], [3, 150]):
        p = _problem(cuda, [37, 300], new, heads=4, kv_heads=2, dim=64, page=32, x="bf16", code="e4m3")
        clean, _ = _attend(cuda, p)
        used = np.zeros((p["kc"].shape[0], 32), bool)
        for b, n in enumerate(p["lens"]):
            for j in range(n):
                used[p["table"][b, j // 32], j % 32] = True
        for c in (p["kc"], p["vc"]):
            raw = c.view(torch.uint8)
            raw[torch.tensor(~used, device=cuda)[:, None, :, None].expand_as(raw)] = 0x7F  # NaN
        for s in (p["ks"], p["vs"]):
            s[torch.tensor(~used.any(1), device=cuda)] = float("nan")
        p["table"][0, 2:] = 1 << 30
        again, _ = _attend(cuda, p)
        assert torch.equal(clean, again)


def test_attend_nan_stays_with_its_token(native, cuda):
    """A NaN in a token's K or V reaches the rows that see the token and no others (e4m3; int8 has none)."""
    import torch
    for new, dim in ((40, 64), (3, 128), (200, 128)):
        cache = _kv().Exl3KvCache(1, 20, 2, dim, requests=1, max_len=320, page_size=16, device=cuda)
        k, v, q = (torch.randn(new, n, dim, device=cuda).bfloat16() for n in (2, 2, 6))
        bad = new // 2
        plan = cache.plan(torch.tensor([new], dtype=torch.int32, device=cuda), new)
        cache.append(0, k, v, plan)
        clean = cache.attend(0, q, plan, new)
        k[bad, 0, 5] = float("nan")
        v[bad, 1, 7] = float("nan")
        cache.append(0, k, v, plan)
        out = cache.attend(0, q, plan, new)
        assert torch.equal(out[:bad], clean[:bad]) and bool(out[bad:].isnan().all())
        windowed = cache.attend(0, q, plan, new, window=2)
        assert not windowed[bad + 2:].isnan().any() and bool(windowed[bad:bad + 2].isnan().all())


def test_attend_bad_page(native, cuda):
    """Keys whose page is not in the cache are not seen; status 7."""
    for new in ([1], [70]):
        p = _problem(cuda, [100], new, heads=2, kv_heads=1, dim=64, page=16, x="f16", code="int8")
        p["table"][0, 2], p["table"][0, 4] = -1, 1 << 20
        _check_attend(cuda, p, "f16")
        assert native.device_status(clear=True) == 7


def test_attend_scales_far_apart(native, cuda):
    """Pages whose V scales differ by powers up to 2^40: their weights keep their place in the sum."""
    p = _problem(cuda, [160], [1], heads=4, kv_heads=1, dim=64, page=16, x="bf16", code="int8")
    for i, e in enumerate((-40, -30, -8, -8, 0, -40, -20, -8, -5, -30)):
        p["vs"][int(p["table"][0, i])] = 2.0 ** e
    _check_attend(cuda, p, "bf16")


def test_attend_past_32_bits(native, cuda):
    """A cache whose byte offsets pass 2^31."""
    import torch
    heads, page, dim = 2, 64, 128
    pages = (1 << 31) // (heads * page * dim) + 70
    kc, vc = (torch.zeros(pages, heads, page, dim, dtype=torch.int8, device=cuda) for _ in range(2))
    ks, vs = (torch.full((pages, heads), 2.0 ** -6, device=cuda) for _ in range(2))
    x = torch.randn(400, 2 * heads, dim, device=cuda).half()
    table = torch.arange(pages - 7, pages, dtype=torch.int32, device=cuda).view(1, 7)
    slots = (table[0].long()[:, None] * page + torch.arange(page, device=cuda)).view(-1)[:400].contiguous()
    _kv().kv_append(x[:, :heads], x[:, heads:], slots, kc, vc, ks, vs)
    kw = dict(kv_lens=torch.tensor([400], dtype=torch.int32, device=cuda))
    small = table - (pages - 7)
    for new in (1, 200):
        cu = torch.tensor([0, new], dtype=torch.int32, device=cuda)
        q = torch.randn(new, 4, dim, device=cuda).half()
        a = _kv().kv_attend(q, kc, vc, ks, vs, table, cu_tokens=cu, max_new=new, **kw)
        b = _kv().kv_attend(q, kc[-7:], vc[-7:], ks[-7:], vs[-7:], small, cu_tokens=cu, max_new=new, **kw)
        assert torch.equal(a, b) and bool(a.any())


# --- the step together --------------------------------------------------------

def test_cache_object_steps(native, cuda):
    """Exl3KvCache over several steps (prompts, then single tokens, a release) against dense attention in 64 bits."""
    import torch
    cache = _kv().Exl3KvCache(1, 40, 2, 64, requests=3, max_len=200, page_size=16, dtype=torch.int8, device=cuda)
    hist = [[], [], []]
    g = torch.Generator(device=cuda).manual_seed(0)
    for step, new in enumerate(([20, 0, 33], [1, 1, 1], [1, 50, 1], [1, 1, 1])):
        if step == 3:
            cache.release(0)
            hist[0] = []
        T = sum(new)
        k, v = (torch.randn(T, 2, 64, generator=g, device=cuda).half() for _ in range(2))
        q = torch.randn(T, 4, 64, generator=g, device=cuda).half()
        plan = cache.plan(torch.tensor(new, dtype=torch.int32, device=cuda), T)
        cache.append(0, k, v, plan)
        out = cache.attend(0, q, plan, max(new)).double().cpu()
        cache.commit(plan)
        at = 0
        for b, n in enumerate(new):
            for i in range(n):
                hist[b].append((k[at].double().cpu(), v[at].double().cpu()))
                ks, vs = (torch.stack([h[j] for h in hist[b]]).repeat_interleave(2, 1) for j in (0, 1))
                p = torch.softmax(torch.einsum("hd,nhd->hn", q[at].double().cpu(), ks) / 8, 1)
                want = torch.einsum("hn,nhd->hd", p, vs)
                # a scale is at most 2 * max|x| / 127: half a step is max|x| / 127 of V, and K's error moves weights alike
                assert (out[at] - want).abs().max() <= 0.08 * vs.abs().max(), (step, b, i)
                at += 1
    assert cache.lens.tolist() == [1, 52, 36]


def test_operators_share_a_workspace(native, cuda):
    """Log probabilities of split rows between attention calls of every kind: each leaves the shared counters zero."""
    import torch
    from exl3_b200.logprobs import token_logprobs
    few = _problem(cuda, [3000, 500], [1, 2], heads=8, kv_heads=2, dim=64, page=16, x="f16", code="int8")
    many = _problem(cuda, [900, 700], [300, 650], heads=8, kv_heads=2, dim=128, page=16, x="bf16", code="e4m3", seed=5)
    logits = torch.randn(3, 120001, device=cuda)
    tok = torch.tensor([1, 2, 3], device=cuda)
    want = [_attend(cuda, few)[0], _attend(cuda, many)[0], token_logprobs(logits, tok, top=20)]
    for order in ((2, 0, 2, 1, 2), (2, 1, 0, 2, 2), (1, 2, 1, 0, 2), (0, 0, 2, 1, 1)):
        for i in order:
            if i == 2:
                got = token_logprobs(logits, tok, top=20)
                assert all(torch.equal(a, b) for a, b in zip(got, want[2]))
            else:
                assert torch.equal(_attend(cuda, (few, many)[i])[0], want[i])


def test_refusals(native, cuda):
    import torch
    kv = _kv()
    p = _problem(cuda, [40], [1], heads=4, kv_heads=2, dim=64, page=16, x="f16", code="int8")
    i = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    table, lens = i(p["table"]), i(p["lens"])
    good = dict(q=p["q"], k_cache=p["kc"], v_cache=p["vc"], k_scale=p["ks"], v_scale=p["vs"], block_table=table, kv_lens=lens)

    def refused(match, exc=ValueError, **kw):
        with pytest.raises(exc, match=match):
            kv.kv_attend(**{**good, **kw})

    refused("CUDA", RuntimeError, q=p["q"].cpu())
    refused("fp16 or bf16", q=p["q"].float())
    refused("multiple of kv_heads", q=p["q"][:, :3])
    refused("both", v_cache=p["vc"].view(torch.uint8))
    refused("contiguous", k_cache=p["kc"][:, :1])
    refused("page must be", k_cache=p["kc"][:, :, :8].contiguous(), v_cache=p["vc"][:, :, :8].contiguous())
    refused("scales", k_scale=p["ks"][:1])
    refused("scales", v_scale=p["vs"].half())
    refused("block_table", block_table=table.long())
    refused("one row of q", max_new=2)
    refused("cu_tokens", cu_tokens=i([0]))
    refused("window", window=-1)
    refused("finite", RuntimeError, scale=float("nan"))
    with pytest.raises(ValueError, match="slots, kv heads"):
        kv.kv_append(p["q"], p["q"], torch.zeros(1, dtype=torch.int64, device=cuda), p["kc"], p["vc"], p["ks"], p["vs"])
    with pytest.raises(ValueError, match="int64"):
        kv.kv_append(p["q"][:, :2], p["q"][:, :2], i([0]), p["kc"], p["vc"], p["ks"], p["vs"])
    with pytest.raises(ValueError, match="page_size"):
        kv.kv_plan(lens, lens, table, i([0]), i([0]), page_size=48, n_tokens=1)
    with pytest.raises(ValueError, match="one row per request"):
        kv.kv_plan(lens, i([1, 1]), table, i([0]), i([0]), page_size=16, n_tokens=1)
    with pytest.raises(RuntimeError, match="requests"):
        kv.kv_plan(i([0] * 20000), i([0] * 20000), torch.zeros(20000, 1, dtype=torch.int32, device=cuda), i([0]), i([0]),
                   page_size=16, n_tokens=1)

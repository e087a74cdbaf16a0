"""GPU: the serving operators on device values that a plan does not give (slots
out of order, lengths beyond the table, offsets outside the rows), and at sizes
where a launch changes.  What is wrong is skipped with status 7; what is right
beside it stands, and nothing is written elsewhere."""

import numpy as np
import pytest
import serving_ref as ref

pytestmark = pytest.mark.gpu


def _kv():
    from exl3_b200 import kv_cache
    return kv_cache


def _kept(slots, page, pages):
    """The slots that are written, -1 for the others, and whether any was refused: rows must continue the row
    before them, or come from another page than the last kept row (up to a page's length back)."""
    slots = [int(s) if 0 <= s < pages * page else -1 for s in slots]
    out, refused, good = [], False, False
    for t, s in enumerate(slots):
        if s >= 0 and not (t and slots[t - 1] >= 0 and s == slots[t - 1] + 1 and s % page):
            before = next((u for u in reversed(slots[max(0, t - page):t]) if u >= 0), None)
            good = before is None or before // page != s // page
            refused |= not good
        out.append(s if good else -1)
    return np.array(out), refused


def _append(cuda, native, slots, *, page, heads, dim, code, pages, guard=4096, seed=0):
    """Appends to caches with guard bytes on both sides; checks codes, scales, guards and the status."""
    import torch
    kinds = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
    rng = np.random.default_rng(seed)
    n = pages * heads * page * dim
    whole = [torch.full((n + 2 * guard,), 0x38, dtype=torch.uint8, device=cuda) for _ in range(2)]
    caches = [w[guard:guard + n].view(kinds[code]).view(pages, heads, page, dim) for w in whole]
    scales = [torch.full((pages, heads), 2.0 ** -6, device=cuda) for _ in range(2)]
    k, v = (torch.tensor(rng.standard_normal((len(slots), heads, dim)) * np.exp2(rng.integers(-6, 3, (len(slots), heads, 1))),
                         device=cuda).half() for _ in range(2))
    kept, refused = _kept(slots, page, pages)
    want = [ref.append(x.float().cpu().numpy(), kept, c.float().cpu().numpy(), s.cpu().numpy(), code, other)
            for x, c, s, other in zip((k, v), caches, scales, (v.float().cpu().numpy(), None))]
    _kv().kv_append(k, v, torch.tensor(np.asarray(slots), dtype=torch.int64, device=cuda), *caches, *scales)
    torch.cuda.synchronize()
    for (wc, ws), c, s, w in zip(want, caches, scales, whole):
        assert np.array_equal(s.cpu().numpy(), ws)
        assert np.array_equal(c.float().cpu().numpy(), wc)
        assert bool((w[:guard] == 0x38).all()) and bool((w[guard + n:] == 0x38).all())
    refused |= bool((np.asarray(slots) >= pages * page).any())
    assert native.device_status(clear=True) == (7 if refused else 0)


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("page,dim", [(16, 128), (32, 64), (64, 128), (128, 64)])
def test_append_stays_within_its_tile(native, cuda, page, dim, code):
    """Slots that repeat, jump, turn back or wrap within a page, at the end of the cache too."""
    P, pages, heads = page, 6, 2
    end = pages * P
    for slots in ([end - 1] * (2 * P), [end - 1, end - P], [end - 2, end - 1, end - 1, end - 1],
                  [end - P + 3, end - P + 5, end - P + 6], list(range(end - 1, end - P - 1, -1)),
                  list(range(end - P // 2, end)) + list(range(end - P, end - P // 2)),
                  [0, 1, -1, 3, -1, 4], [0] + [-1] * (P - 1) + [1], [end - 1, end, end + 1, end - 1],
                  [0, 0, P, P + 1, P + 1, 2 * P, 2 * P + 1] + list(range(3 * P, 4 * P)) * 2 + [5 * P]):
        _append(cuda, native, slots, page=page, heads=heads, dim=dim, code=code, pages=pages)


@pytest.mark.parametrize("page", [16, 64, 128])
def test_append_skipped_rows_between_pages(native, cuda, page):
    """Rows skipped before, between and behind the pages of a padded layout are no fault."""
    P = page
    slots = [-1] * 5 + [3, 4, 5] + [-1] * (P + 40) + [P, P + 1] + [-1] * 3 + list(range(2 * P - 1 + P, 4 * P)) + [-1] * 70
    assert not _kept(slots, P, 8)[1]
    _append(cuda, native, slots, page=P, heads=3, dim=64, code="int8", pages=8)


def test_append_any_slots(native, cuda):
    """Stretches of random kinds, in small and in page-sized windows of a launch.  A page returns only next to itself."""
    rng = np.random.default_rng(7)
    for page, heads, pages, tokens in ((16, 2, 400, 700), (64, 8, 200, 2000), (128, 8, 60, 2500), (32, 4, 300, 1500)):
        order, slots = list(rng.permutation(pages)), []
        while len(slots) < tokens and order:
            p = int(order.pop()) * page
            for _ in range(int(rng.integers(1, 4))):
                a, b = sorted(rng.integers(0, page + 1, 2))
                stretch = list(range(p + int(a), p + int(b)))
                kind = rng.integers(0, 6)
                slots += stretch[::-1] if kind == 0 else stretch[::2] if kind == 1 else stretch[:1] * 5 if kind == 2 else stretch
                if kind == 3:
                    slots += [-1] * int(rng.integers(1, page // 2))
        _append(cuda, native, slots, page=page, heads=heads, dim=128, code="e4m3", pages=pages, seed=page)


# --- attend -----------------------------------------------------------------

def _attend_problem(cuda, lens, new, *, heads=4, kv_heads=2, dim=64, page=16, seed=0):
    import torch
    g = torch.Generator(device=cuda).manual_seed(seed)
    width = max(1, max(-(-n // page) for n in lens))
    pages = len(lens) * width
    kc, vc = (torch.randint(-127, 128, (pages, kv_heads, page, dim), generator=g, device=cuda).to(torch.int8)
              for _ in range(2))
    ks, vs = (torch.full((pages, kv_heads), 2.0 ** -6, device=cuda) for _ in range(2))
    i = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device=cuda)  # noqa: E731
    table = torch.randperm(pages, generator=g, device=cuda).to(torch.int32).view(len(lens), width)
    q = torch.randn(sum(new), heads, dim, generator=g, device=cuda).half()
    return dict(q=q, k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, block_table=table, kv_lens=i(lens),
                cu_tokens=i(np.concatenate([[0], np.cumsum(new)])), max_new=max(new), return_lse=True)


def _plain(p, window=0):
    """The 64-bit form of a problem: out, lse and their bounds (f16 outputs; derived in test_gpu_kv_cache.py)."""
    D, n = p["q"].shape[2], max(int(p["kv_lens"].max()), 1)
    kv = [c.double().cpu().numpy() * s.double().cpu().numpy()[:, :, None, None]
          for c, s in ((p["k_cache"], p["k_scale"]), (p["v_cache"], p["v_scale"]))]
    out, lse, amp, vmax, smax = ref.attend(p["q"].double().cpu().numpy(), kv, p["block_table"].cpu().numpy(),
                                           p["kv_lens"].cpu().numpy(), p["cu_tokens"].cpu().numpy(), D ** -0.5, window)
    tol = 2.0 ** -11 * np.abs(out) + (2.0 ** -11 + 2.0 ** -13) * amp + n * 2.0 ** -24 * vmax + 2.0 ** -25
    ltol = D * 2.0 ** -23 * smax + 2.0 ** -17 * (1 + np.abs(np.where(np.isinf(lse), 0, lse)))
    return out, lse, tol, ltol


def _near(got, want, rows=slice(None)):
    (out, lse), (wout, wlse, tol, ltol) = got, want
    out, lse = out.double().cpu().numpy()[rows], lse.double().cpu().numpy()[rows]
    assert (np.abs(out - wout[rows]) <= tol[rows]).all()
    empty = np.isneginf(wlse[rows])
    assert np.array_equal(np.isneginf(lse), empty)
    assert (np.abs(np.where(empty, 0, lse) - np.where(empty, 0, wlse[rows])) <= ltol[rows]).all()


@pytest.mark.parametrize("new", [[2, 1, 3], [70, 90, 130]])
def test_attend_row_offsets_outside_q(native, cuda, new):
    """cu_tokens that leave q: nothing outside is read or written, rows inside stand, status 7."""
    import torch
    p = _attend_problem(cuda, [150, 200, 170], new)
    want = _plain(p)
    _near(_kv().kv_attend(**p), want)
    n, big = sum(new), 2 ** 31 - 1
    first, second = new[0], new[0] + new[1]
    for cu, stands in (([-5, first, second, n], (first, n)), ([0, first, second, n + 7], (0, second)),
                       ([0, first, second, big], (0, second)), ([-big, first, second, n], (first, n)),
                       ([0, first, n + 3, n + 9], (0, first)), ([-2 ** 31, -4, second, -1], (0, 0)),
                       ([big, big, big, big], (0, 0)), ([0, big, -big, big], (0, 0))):
        bad = {**p, "cu_tokens": torch.tensor(cu, dtype=torch.int32, device=cuda)}
        got = _kv().kv_attend(**bad)
        torch.cuda.synchronize()
        _near(got, want, slice(*stands))
        assert native.device_status(clear=True) == (0 if cu == [big] * 4 else 7), cu
    # a request that q cuts short keeps the positions of all its rows
    cut = {**p, "q": p["q"][:-1]}
    _near(_kv().kv_attend(**cut), [w[:-1] for w in want])
    assert native.device_status(clear=True) == 7


@pytest.mark.parametrize("new", [[5, 1, 3, 2], [70, 64, 90, 5]])
def test_attend_lengths_beyond_the_table(native, cuda, new):
    """Tokens that the block table has no place for are not seen; the rows keep their positions."""
    import torch
    lens = [100, 90, 96, 71]
    p = _attend_problem(cuda, lens, new)
    p["kv_lens"] = torch.tensor([117, 90, 96, 75], dtype=torch.int32, device=cuda)
    p["block_table"] = p["block_table"][:, :4].contiguous()  # places for 64
    wide = torch.full((4, 8), -1, dtype=torch.int32, device=cuda)
    wide[:, :4] = p["block_table"]
    for window in (0, 12, 40):
        got = _kv().kv_attend(**p, window=window)
        _near(got, _plain({**p, "block_table": wide}, window))
        assert native.device_status(clear=True) == 7
    p["kv_lens"] = torch.tensor([64, 60, 64, 7], dtype=torch.int32, device=cuda)
    _kv().kv_attend(**p)
    assert native.device_status(clear=True) == 0
    p["kv_lens"] = torch.full((4,), 2 ** 31 - 1, dtype=torch.int32, device=cuda)
    assert not _kv().kv_attend(**p, window=50)[0].any()  # every row is far behind the table
    assert native.device_status(clear=True) == 7


# --- plan -------------------------------------------------------------------

def test_plan_request_counts(native, cuda):
    """Up to the limit, from small to large in a process of its own: a larger launch must not be what lets a smaller one through."""
    import os
    import subprocess
    import sys

    from conftest import PKG
    code = """
import numpy as np, torch
from exl3_b200.kv_cache import kv_plan
for B in (6000, 6125, 6126, 6130, 6143, 6144, 9000, 16384):
    lens = torch.arange(B, dtype=torch.int32, device="cuda") % 50
    new = torch.ones_like(lens)
    table = torch.arange(B * 4, dtype=torch.int32, device="cuda").view(B, 4)
    free = torch.arange(B * 4, B * 5, dtype=torch.int32, device="cuda")
    p = kv_plan(lens, new, table, free, torch.zeros(1, dtype=torch.int32, device="cuda"), page_size=16, n_tokens=B)
    n = np.arange(B) % 50
    taken = n % 16 == 0
    page = np.where(taken, B * 4 + np.cumsum(taken) - 1, np.arange(B) * 4 + n // 16)
    assert np.array_equal(p.slots.cpu().numpy(), page * 16 + n % 16), B
    assert np.array_equal(p.positions.cpu().numpy(), n) and int(p.cursor) == taken.sum(), B
    assert np.array_equal(p.kv_lens.cpu().numpy(), n + 1) and np.array_equal(p.cu_tokens.cpu().numpy(), np.arange(B + 1)), B
print("planned")
"""
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([PKG, os.environ.get("PYTHONPATH", "")]))
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, env=env, timeout=300)
    assert run.returncode == 0 and "planned" in run.stdout, run.stderr[-2000:]


def test_plan_sums_beyond_32_bits(native, cuda):
    """Lengths whose sums pass 2^31: what is in order stands, nothing outside the table is read or written, status 7."""
    import torch
    big = 2 ** 31 - 1
    i = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    for lens, new in (([3, 5, 0, 7], [2, big, 20, 1]), ([3, 5, 0, 7], [2, big, big, big]),
                      ([3, big, 9, 7], [2, 5, 20, 1]), ([3, big, big - 1, 0], [2, big, 3, big]),
                      ([3, big - 9, 100, 7], [2, big, big, 1])):
        whole = torch.full((3, 4, 6), -5, dtype=torch.int32, device=cuda)
        table = whole[1]
        table.copy_(torch.arange(24, device=cuda).view(4, 6))
        free = torch.arange(100, 140, dtype=torch.int32, device=cuda)
        p = _kv().kv_plan(i(lens), i(new), table, free, i([0]), page_size=16, n_tokens=30)
        torch.cuda.synchronize()
        assert native.device_status(clear=True) == 7
        assert p.positions[:2].tolist() == [3, 4] and p.slots[:2].tolist() == [3, 4]
        assert p.kv_lens.tolist() == [min(a + b, big) for a, b in zip(lens, new)]
        assert p.cu_tokens.tolist()[:2] == [0, 2] and all(0 <= c <= 30 for c in p.cu_tokens.tolist())
        assert bool((whole[0] == -5).all()) and bool((whole[2] == -5).all())
        slots = p.slots.tolist()
        assert all(s == -1 or 0 <= s < 24 * 16 or 100 * 16 <= s < 140 * 16 for s in slots)
        assert int(p.cursor) == (40 if max(new) == big else 1)


@pytest.mark.parametrize("heads,kv_heads", [(64, 1), (128, 1), (98, 2), (600, 1)])
def test_attend_many_heads_per_kv_head(native, cuda, heads, kv_heads):
    """More query columns from one token than the few-row kernel takes, up to several tiles of the prompt kernel."""
    for lens, new in (([1, 40, 333], [1, 1, 1]), ([70, 300], [2, 3])):
        p = _attend_problem(cuda, lens, new, heads=heads, kv_heads=kv_heads)
        _near(_kv().kv_attend(**p), _plain(p))


def test_attend_many_requests(native, cuda):
    """More requests than the kernels have threads, empty ones among them, prompts between single tokens."""
    lens = [(7 * i) % 90 for i in range(1300)]
    new = [min(n, 1) for n in lens]
    p = _attend_problem(cuda, lens, new)
    _near(_kv().kv_attend(**p), _plain(p))
    for b in (3, 600, 601, 1299):
        new[b] = lens[b]
    p = _attend_problem(cuda, lens, new, seed=1)
    _near(_kv().kv_attend(**p), _plain(p))


def test_attend_more_rows_than_tokens(native, cuda):
    """Rows at positions before the first token see nothing; a max_new below or above the rows only selects kernels."""
    for lens, new in (([3, 0, 20], [5, 2, 20]), ([30, 64, 1], [90, 70, 60])):
        p = _attend_problem(cuda, lens, new)
        want = _plain(p)
        for most in (max(new), 1, 5000):
            out, lse = _kv().kv_attend(**{**p, "max_new": most})
            _near((out, lse), want)
            empty = np.isinf(want[1])
            assert empty.any() and not out.cpu().numpy()[empty].any()

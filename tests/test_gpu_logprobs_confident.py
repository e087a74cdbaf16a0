"""GPU: token log probabilities where one entry carries nearly all of the weight.

Error of log p = d - log s, with the largest entry's weight exactly 1 and p its
probability: s has at most 7 fp32 roundings where a row has a few entries (the
others are sums with zeros), the other weights, together 1 - p, are off by 2^-21
each (the exponential 2^-22, its argument's rounding), the logarithm by 2^-22 of
itself: 7 * 2^-24 + (1 - p) 2^-21 + 2^-22 |log p|.
The entropy adds w: 8 roundings of the largest entry's weight times its lag
behind the reference, 4 at most: (7 + 32) 2^-24, and 2^-20 of its own size.
A full row of n entries has 16 + 2 + n / 8192 roundings in a thread and 20 in
the joins instead of the 7 and 8: 64 * 2^-24 and, times the lag, 256 * 2^-24.
Signs are exact: log p <= 0, H >= 0.
"""

import numpy as np
import pytest
import serving_ref as ref

pytestmark = pytest.mark.gpu


def _check(x, tokens, top, sums):
    import torch
    from exl3_b200.logprobs import token_logprobs
    got = token_logprobs(x, torch.tensor(tokens, device=x.device), top=top)
    lp, ent, rank, vals, ids = ref.logprobs(x.double().cpu().numpy(), tokens, top)
    glp, gent, gvals = (t.double().cpu().numpy() for t in (got.logprob, got.entropy, got.top_logprobs))
    assert (glp <= 0).all() and (gvals <= 0).all() and (gent >= 0).all()
    most = np.exp(np.max(vals, 1))
    tol = sums * 2.0 ** -24 + (1 - most) * 2.0 ** -21
    for g, w, t in ((glp, lp, tol), (gvals, vals, tol[:, None])):
        seen = np.isfinite(w)
        assert np.array_equal(g[~seen], w[~seen])
        err = np.abs(np.where(seen, g, 0) - np.where(seen, w, 0))
        assert (err <= t + 2.0 ** -22 * np.abs(np.where(seen, w, 0))).all(), err.max()
    err = np.abs(gent - ent)
    assert (err <= (sums + (32 if sums == 7 else 256)) * 2.0 ** -24 + 2.0 ** -20 * ent).all(), err.max()
    assert np.array_equal(got.rank.cpu().numpy(), rank) and np.array_equal(got.top_ids.cpu().numpy(), ids)


@pytest.mark.parametrize("x", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("start", [0, 1])
def test_two_entries(native, cuda, x, start):
    """Two finite entries that one thread meets one after the other, the larger by up to 20: a vector and the one a
    round later, an entry before the first vector and a vector, a vector and an entry behind the last."""
    import torch
    dt = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[x]
    n, vec = 16411, 4 if x == "f32" else 8
    g = torch.Generator(device=cuda).manual_seed(start)
    wide = torch.full((1500, n + 13), -float("inf"), dtype=dt, device=cuda)
    rows = wide[:, start:start + n]
    low = torch.randn(1500, generator=g, device=cuda) * 3
    gap = torch.rand(1500, generator=g, device=cuda) * 20
    for i, (a, b) in enumerate(((40, 40 + 1024 * vec), (0, 8), (2, 1024 * vec + 8), (40 + 1024 * vec, n - 2), (300, 310))):
        part = slice(300 * i, 300 * i + 300)
        rows[part, a], rows[part, b] = low[part].to(dt), (low + gap)[part].to(dt)
    best = rows.float().argmax(1).cpu().numpy()
    _check(rows, best, 2, 7)


@pytest.mark.parametrize("vocab", [1000, 50257, 131072])
@pytest.mark.parametrize("rows", [1, 3, 600])
def test_one_entry_above_the_rest(native, cuda, rows, vocab):
    """Full rows, one entry 8 to 18 above the largest of the others, in split rows and whole ones."""
    import torch
    if rows * vocab > 1 << 25:
        rows = 100
    g = torch.Generator(device=cuda).manual_seed(vocab + rows)
    x = torch.randn(rows, vocab, generator=g, device=cuda)
    at = torch.randint(0, vocab, (rows,), generator=g, device=cuda)
    up = x.amax(1) + 8 + 10 * torch.rand(rows, generator=g, device=cuda)
    x[torch.arange(rows, device=cuda), at] = up
    _check(x, at.cpu().numpy(), 3, 64)
    _check(x.bfloat16(), at.cpu().numpy(), 3, 64)


def test_rows_that_rise(native, cuda):
    """The maximum grows all the way, by less and by more than the reference lets pass."""
    import torch
    n = 40000
    at = torch.arange(n, device=cuda, dtype=torch.float32)
    x = torch.stack([at / n * s for s in (3.0, 30.0, 300.0)] + [(at // 8192) * 3.9, (at // 8192) * 4.1])
    _check(x, [n - 1] * 5, 3, 64)

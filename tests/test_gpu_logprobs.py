"""GPU: token log probabilities against the 64-bit plain form.

Sums of exponentials carry at most (64 + 16) fp32 roundings of positive terms
and 2^-22 of the exponential: 2^-17 relative, so 2^-16 absolute in a log
probability, plus 2^-22 of its own size (two fp32 differences); the entropy's
second sum weighs the same errors by |d|: 2^-15 (1 + H).  Ranks and ids are exact.
"""

import numpy as np
import pytest
import serving_ref as ref

pytestmark = pytest.mark.gpu


def _run(x, tokens, top):
    from exl3_b200.logprobs import token_logprobs
    return token_logprobs(x, tokens, top=top)


def _check(cuda, x, tokens, top, ids=None):
    import torch
    t = torch.tensor(tokens, dtype=ids or torch.int64, device=cuda)
    got = _run(x, t, top)
    lp, ent, rank, vals, tid = ref.logprobs(x.double().cpu().numpy(), tokens, top)

    def near(a, b, tol):
        a = a.cpu().numpy().astype(np.float64)
        inf = np.isinf(b)
        assert np.array_equal(a[inf], b[inf])
        assert (np.abs(a[~inf] - b[~inf]) <= tol(np.abs(b[~inf]))).all(), np.max(np.abs(a[~inf] - b[~inf]))

    assert np.array_equal(got.rank.cpu().numpy(), rank)
    assert np.array_equal(got.top_ids.cpu().numpy(), tid)
    near(got.logprob, lp, lambda b: 2.0 ** -16 + 2.0 ** -22 * b)
    near(got.top_logprobs, vals, lambda b: 2.0 ** -16 + 2.0 ** -22 * b)
    near(got.entropy, ent, lambda b: 2.0 ** -15 * (1 + b))
    return got


def _dtypes():
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.mark.parametrize("x", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [1, 2, 7, 31, 33, 1000, 4097, 50257, 131072, 200003])
@pytest.mark.parametrize("rows", [1, 5])
def test_sizes(native, cuda, rows, vocab, x):
    import torch
    g = torch.Generator(device=cuda).manual_seed(vocab)
    logits = (torch.randn(rows, vocab, generator=g, device=cuda) * 3).to(_dtypes()[x])
    rng = np.random.default_rng(vocab)
    for top in (0, 1, 20, 32):
        _check(cuda, logits, rng.integers(0, vocab, rows), min(top, vocab))


def test_many_rows(native, cuda):
    import torch
    logits = (torch.randn(700, 9001, device=cuda) * 2).bfloat16()
    best = logits.float().argmax(1).cpu().numpy()
    _check(cuda, logits, best, 3, ids=torch.int32)
    _check(cuda, logits[:400], best[:400], 32)


@pytest.mark.parametrize("x", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [40, 5000, 70000])
def test_ties_and_order(native, cuda, vocab, x):
    """Constant rows, few distinct values, rising and falling rows: ties go to the lowest index."""
    import torch
    at = torch.arange(vocab, device=cuda).float()
    rows = torch.stack([torch.full_like(at, 1.5), (at * 7919 % 5), at / vocab * 8, -at / vocab * 8,
                        torch.where(at % 3 == 0, 0.0, -0.0), (at == vocab - 1) * 4.0])
    for tokens in ([0] * 6, [vocab - 1] * 6, [vocab // 2] * 6):
        _check(cuda, rows.to(_dtypes()[x]), tokens, 32)


@pytest.mark.parametrize("x", ["f32", "f16", "bf16"])
def test_masked_rows(native, cuda, x):
    """-inf masks that leave one, none or some entries; the type's lowest value as a mask; tokens outside."""
    import torch
    dt = _dtypes()[x]
    inf, low = float("inf"), torch.finfo(dt).min
    logits = (torch.randn(8, 6001, device=cuda) * 2).to(dt)
    logits[0] = -inf
    logits[1] = -inf
    logits[1, 77] = 2.0
    logits[2, 100:] = -inf
    logits[3] = low
    logits[4] = low
    logits[4, 5990] = 1.0
    logits[5, ::2] = low
    logits[6, :40] = torch.finfo(dt).max
    tokens = [3, 77, 200, 4000, 5990, 4, 41, 6000]
    _check(cuda, logits, tokens, 5)
    _check(cuda, logits, [-1, 6001, -5, 1 << 40, 0, 1, 2, 3], 5)
    _check(cuda, logits, [0, 0, 99, 0, 0, 0, 39, 0], 32)


def test_nan_and_inf(native, cuda):
    """NaN or +inf in a row makes that row NaN; its neighbours stay."""
    import torch
    logits = torch.randn(3, 5000, device=cuda)
    clean = _run(logits, torch.zeros(3, dtype=torch.int64, device=cuda), 4)
    logits[1, 4321] = float("nan")
    logits[2, 17] = float("inf")
    got = _run(logits, torch.zeros(3, dtype=torch.int64, device=cuda), 4)
    for a, b in zip(got, clean):
        assert torch.equal(a[0], b[0])
    assert got.logprob[1:].isnan().all() and got.entropy[1:].isnan().all()
    assert int(got.top_ids[2, 0]) == 17 and ((got.top_ids >= 0) & (got.top_ids < 5000)).all()
    assert torch.equal(got.top_ids[1], clean.top_ids[1])


def test_strides_and_streams(native, cuda):
    """Rows of a wider buffer at odd offsets, transposed logits (copied), another stream, repeats bit for bit."""
    import torch
    wide = (torch.randn(6, 8203, device=cuda) * 2).half()
    for lo, hi in ((1, 8001), (3, 8203), (8, 5000)):
        _check(cuda, wide[:, lo:hi], [0, 5, 6, 7, 8, 4000], 7)
    _check(cuda, wide[::2, 5:4005], [0, 5, 6], 7)
    _check(cuda, wide.t()[:2000], list(range(6)) * 333 + [0, 1], 2)
    big = torch.randn(2, 150001, device=cuda)
    tok = torch.tensor([5, 9], device=cuda)
    first = _run(big, tok, 20)
    s = torch.cuda.Stream(cuda)
    s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        with torch.cuda.stream(s):
            b = _run(big, tok, 20)
        a = _run(big, tok, 20)
        torch.cuda.synchronize()
        for u, v, w in zip(first, a, b):
            assert torch.equal(u, v) and torch.equal(u, w)


def test_refusals(native, cuda):
    import torch
    from exl3_b200.logprobs import token_logprobs
    x, t = torch.zeros(2, 50, device=cuda), torch.zeros(2, dtype=torch.int64, device=cuda)
    for args, kw, exc, match in (
            ((x.cpu(), t), {}, RuntimeError, "CUDA"), ((x[0], t), {}, ValueError, "rows, vocab"),
            ((x.int(), t), {}, ValueError, "fp32"), ((x.double(), t), {}, ValueError, "fp32"),
            ((x, t[:1]), {}, ValueError, "tokens"), ((x, t.float()), {}, ValueError, "tokens"),
            ((x, t), {"top": 33}, ValueError, "top"), ((x, t), {"top": -1}, ValueError, "top"),
            ((x[:, :3], t), {"top": 4}, ValueError, "top")):
        with pytest.raises(exc, match=match):
            token_logprobs(*args, **kw)
    empty = token_logprobs(x[:0], t[:0], top=3)
    assert empty.top_ids.shape == (0, 3)

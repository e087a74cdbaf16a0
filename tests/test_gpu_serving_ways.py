"""GPU: the serving operators answer alike on the compiled way from Python and on the one written out."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["compiled", "written out"])
def way(request, native, monkeypatch):
    from exl3_b200 import _native
    assert _native.binding() is not _native._NoBinding
    if request.param == "written out":
        monkeypatch.setattr(_native, "_binding", _native._NoBinding)
    return request.param


def _cache(cuda, dtype):
    from exl3_b200.kv_cache import Exl3KvCache
    return Exl3KvCache(1, 40, 2, 64, requests=3, max_len=200, page_size=16, dtype=dtype, device=cuda)


def _steps(cuda, dtype):
    """All that three steps of a cache and their log probabilities return."""
    import torch
    from exl3_b200.logprobs import token_logprobs
    cache, got = _cache(cuda, dtype), []
    g = torch.Generator(device=cuda).manual_seed(0)
    for new in ([20, 0, 33], [1, 1, 1], [1, 90, 2]):
        n = sum(new)
        fused = torch.randn(n, 10, 64, generator=g, device=cuda).bfloat16()
        plan = cache.plan(torch.tensor(new, dtype=torch.int32, device=cuda), n + 2)
        for field in plan:
            got.append(field.clone())
        cache.append(0, fused[:, 6:8], fused[:, 8:], plan._replace(slots=plan.slots[:n]))
        got += cache.attend(0, fused[:, :6], plan, max(new), return_lse=True)
        got.append(cache.attend(0, fused[:, :6], plan, max(new), window=7, scale=0.2))
        cache.commit(plan)
        x = torch.randn(3, 90001, generator=g, device=cuda)
        got += token_logprobs(x, torch.tensor([5, 90001, 7], device=cuda), top=9)
        got += token_logprobs(x.half(), torch.tensor([5, 6, 7], dtype=torch.int32, device=cuda))
    got += [cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale, cache.block_table]
    return got


@pytest.mark.parametrize("dtype", ["float8_e4m3fn", "int8"])
def test_both_ways_are_equal(native, cuda, dtype, monkeypatch):
    import torch
    from exl3_b200 import _native
    one = _steps(cuda, getattr(torch, dtype))
    monkeypatch.setattr(_native, "_binding", _native._NoBinding)
    two = _steps(cuda, getattr(torch, dtype))
    assert len(one) == len(two)
    for a, b in zip(one, two):
        assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b)


@pytest.mark.parametrize("asked", [True, 1, np.True_, "yes", False, 0, np.False_, None])
def test_return_lse_goes_by_truth(native, cuda, way, asked):
    """One tensor or a pair, whatever the flag's type and the layout of q."""
    import torch
    from exl3_b200.kv_cache import kv_attend
    kc = torch.ones(3, 1, 16, 64, dtype=torch.int8, device=cuda)
    s = torch.ones(3, 1, device=cuda)
    table, lens = torch.zeros(2, 1, dtype=torch.int32, device=cuda), torch.tensor([3, 9], dtype=torch.int32, device=cuda)
    wide = torch.ones(2, 4, 65, device=cuda).half()
    for q in (wide[:, :, :64].contiguous(), wide[:, :, 1:]):
        got = kv_attend(q, kc, kc, s, s, table, lens, return_lse=asked)
        if asked:
            out, lse = got
            assert lse.shape == (2, 4) and lse.dtype == torch.float32
        else:
            out = got
        assert isinstance(out, torch.Tensor) and out.shape == (2, 4, 64) and bool((out == 1).all())


def test_a_flag_that_cannot_be_asked_raises(native, cuda, way):
    import torch
    from exl3_b200.kv_cache import kv_attend

    class Odd:
        def __bool__(self):
            raise KeyError("odd")

    kc, s = torch.ones(3, 1, 16, 64, dtype=torch.int8, device=cuda), torch.ones(3, 1, device=cuda)
    table, lens = torch.zeros(2, 1, dtype=torch.int32, device=cuda), torch.tensor([3, 9], dtype=torch.int32, device=cuda)
    with pytest.raises(KeyError, match="odd"):
        kv_attend(torch.ones(2, 4, 64, device=cuda).half(), kc, kc, s, s, table, lens, return_lse=Odd())


def test_a_backward_pass_raises(native, cuda, way):
    """No gradient is left out in silence: results of inputs that want one raise when it is asked for."""
    import torch
    from exl3_b200.kv_cache import kv_attend
    from exl3_b200.logprobs import token_logprobs
    kc, s = torch.ones(3, 1, 16, 64, dtype=torch.int8, device=cuda), torch.ones(3, 1, device=cuda)
    table, lens = torch.zeros(2, 1, dtype=torch.int32, device=cuda), torch.tensor([3, 9], dtype=torch.int32, device=cuda)
    q = torch.ones(2, 4, 64, device=cuda).half()
    x, tok = torch.randn(2, 500, device=cuda), torch.tensor([1, 2], device=cuda)
    plain = [kv_attend(q, kc, kc, s, s, table, lens), *kv_attend(q, kc, kc, s, s, table, lens, return_lse=True)]
    plain += [*token_logprobs(x, tok, top=3), *token_logprobs(x, tok)]
    assert not any(t.requires_grad for t in plain)
    q.requires_grad_()
    x.requires_grad_()

    def again():
        got = [kv_attend(q, kc, kc, s, s, table, lens), *kv_attend(q, kc, kc, s, s, table, lens, return_lse=True)]
        return got + [*token_logprobs(x, tok, top=3), *token_logprobs(x, tok)]

    got = again()
    assert all(torch.equal(a, b) for a, b in zip(plain, got))
    for t in got:
        if t.is_floating_point() and t.numel():
            assert t.requires_grad
            with pytest.raises(RuntimeError, match="inference"):
                t.float().sum().backward()
        else:
            assert not t.requires_grad or not t.numel()
    with torch.no_grad():
        assert not any(t.requires_grad for t in again())
    with torch.inference_mode():
        assert all(torch.equal(a, b) for a, b in zip(plain, again()))


def test_a_cache_without_heads_or_pages_is_refused(native, cuda, way):
    import torch
    from exl3_b200.kv_cache import kv_append, kv_attend
    table, lens = torch.zeros(2, 1, dtype=torch.int32, device=cuda), torch.tensor([3, 9], dtype=torch.int32, device=cuda)
    for shape, exc in (((3, 0, 16, 64), ValueError), ((0, 2, 16, 64), RuntimeError)):
        kc, s = torch.ones(shape, dtype=torch.int8, device=cuda), torch.ones(shape[:2], device=cuda)
        for heads in (0, 4):
            q = torch.ones(2, heads, 64, device=cuda).half()
            with pytest.raises(ValueError if heads == 0 else exc):
                kv_attend(q, kc, kc, s, s, table, lens)
        k = torch.ones(2, shape[1], 64, device=cuda).half()
        with pytest.raises(exc):
            kv_append(k, k, torch.tensor([0, 1], device=cuda), kc, kc, s, s)

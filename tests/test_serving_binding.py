"""CPU: how the compiled way into the serving operators is built and loaded."""

import os
import sysconfig

import pytest


def test_its_file_names_what_it_was_built_against(monkeypatch):
    import torch
    from exl3_b200 import build
    path = build.binding_path()
    assert sysconfig.get_config_var("SOABI") in path and torch.__version__ in path
    monkeypatch.setattr(torch, "__version__", "99.0")
    assert build.binding_path() != path  # another torch does not load this one


def test_builds_at_once_do_not_share_a_file(monkeypatch, tmp_path):
    """Every process compiles into a file of its own and puts it in place whole."""
    from exl3_b200 import build
    monkeypatch.setattr(build, "PKG_DIR", str(tmp_path))
    made = []

    class Done:
        returncode, stderr = 0, "no"

    def compile_(cmd, **kw):
        out = cmd[cmd.index("-o") + 1]
        made.append(out)
        with open(out, "w") as f:
            f.write("built")
        return Done

    monkeypatch.setattr(build.subprocess, "run", compile_)
    path = build.build_binding()
    monkeypatch.setattr(build.os, "getpid", lambda: 12345)
    assert build.build_binding(force=True) == path
    assert made[0] != made[1] and os.listdir(tmp_path) == [os.path.basename(path)]
    assert build.build_binding() == path and len(made) == 2  # up to date
    Done.returncode = 1
    with pytest.raises(RuntimeError, match="g\\+\\+ failed"):
        build.build_binding(force=True)


@pytest.mark.parametrize("why", [RuntimeError("g++ failed"), AttributeError("_GLIBCXX_USE_CXX11_ABI"), OSError("no file"),
                                 ImportError("symbol")])
def test_without_it_the_operators_stand_and_say_so(monkeypatch, why):
    import torch
    from exl3_b200 import _native, logprobs

    def fail():
        raise why

    monkeypatch.setattr(_native, "_binding", None)
    monkeypatch.setattr(_native._build, "build_binding", fail)
    with pytest.warns(RuntimeWarning, match=type(why).__name__):
        assert _native.binding() is _native._NoBinding
    with pytest.raises(RuntimeError, match="CUDA"):
        logprobs.token_logprobs(torch.zeros(1, 4), torch.zeros(1, dtype=torch.int64))


def test_tensors_of_several_gpus_are_refused():
    """Each tensor in turn on another GPU than the others: refused by name, before any address is taken."""
    import torch
    from exl3_b200 import kv_cache, logprobs
    from torch._subclasses.fake_tensor import FakeTensor, FakeTensorMode
    mode = FakeTensorMode()

    def on(gpu, *shape, dtype):
        return FakeTensor(mode, torch.empty(shape, dtype=dtype, device="meta"), torch.device("cuda", gpu))

    i32, i64, f16, f32, i8 = torch.int32, torch.int64, torch.float16, torch.float32, torch.int8
    code, scale = ((3, 2, 16, 64), i8), ((3, 2), f32)
    calls = [
        (lambda t: kv_cache.kv_plan(*t, page_size=16, n_tokens=4),
         [((2,), i32), ((2,), i32), ((2, 3), i32), ((9,), i32), ((1,), i32)]),
        (lambda t: kv_cache.kv_append(*t), [((4, 2, 64), f16), ((4, 2, 64), f16), ((4,), i64), code, code, scale, scale]),
        (lambda t: kv_cache.kv_attend(*t[:-1], cu_tokens=t[-1], max_new=2),
         [((4, 4, 64), f16), code, code, scale, scale, ((2, 3), i32), ((2,), i32), ((3,), i32)]),
        (lambda t: logprobs.token_logprobs(*t), [((2, 50), f32), ((2,), i64)]),
    ]
    for call, shapes in calls:
        for other in range(len(shapes)):
            tensors = [on(int(i == other), *s, dtype=d) for i, (s, d) in enumerate(shapes)]
            with pytest.raises(ValueError, match="different GPUs"):
                call(tensors)

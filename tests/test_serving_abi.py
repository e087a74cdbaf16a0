"""CPU: the serving entries refuse bad arguments on the host, before any launch."""

import pytest

OK, ARG, CUDA, WS = 0, 1, 2, 3
A = 4096  # an aligned address that is never read


def _lib():
    from exl3_b200 import _native
    return _native.load(), _native.last_error


def _pack(name, a):
    from exl3_b200 import _native
    return getattr(_native, name)(*[0 if v is None else v for k, v in a.items() if k != "stream"])


def _attend(**kw):
    a = dict(q=A, qt=512, qh=128, xd=2, rows=1, heads=4, k=A, v=A, ks=A, vs=A, code=0, pages=8, hk=2, page=16, dim=128,
             table=A, width=4, req=1, lens=A, cu=None, max_new=1, scale=1.0, window=0, out=A, lse=None, ws=A,
             wsb=1 << 30, stream=None)
    a.update(kw)
    lib, err = _lib()
    return lib.exl3_kv_attend(_pack("PACK_KV_ATTEND", a), a["stream"]), err()


@pytest.mark.parametrize("kw,match", [
    (dict(k=None), "null"), (dict(vs=None), "null"), (dict(k=A + 8), "16-byte"), (dict(code=2), "code"),
    (dict(page=48), "page"), (dict(dim=96), "dim"), (dict(hk=0), "kv_heads"), (dict(pages=0), "pages"),
    (dict(xd=0), "fp16 or bf16"), (dict(heads=5), "multiple"), (dict(rows=-1), "rows"), (dict(width=-1), "width"),
    (dict(width=1 << 30), "tokens"), (dict(max_new=0), "max_new"), (dict(rows=2), "one row of q"),
    (dict(window=-1), "window"), (dict(scale=float("inf")), "finite"), (dict(q=None), "null"),
    (dict(table=None), "null"), (dict(q=A + 8), "16 bytes"), (dict(qt=516), "16 bytes"), (dict(out=A + 2), "out")])
def test_attend_refuses(kw, match):
    rc, msg = _attend(**kw)
    assert rc == ARG and match in msg


def test_attend_workspace_refused():
    for kw in (dict(wsb=100), dict(ws=None), dict(ws=A + 16)):
        rc, msg = _attend(**kw)
        assert rc == WS and "workspace" in msg
    assert _attend(rows=0, req=0)[0] == OK  # nothing to do
    lib, _ = _lib()
    assert lib.exl3_kv_attend_workspace_size(4, 2, 128, 1, 1, 1) > 0
    assert lib.exl3_kv_attend_workspace_size(5, 2, 128, 1, 1, 1) == 0
    assert lib.exl3_kv_attend_workspace_size(4, 2, 96, 1, 1, 1) == 0


@pytest.mark.parametrize("kw,match", [
    (dict(k=None), "null"), (dict(xd=0), "fp16 or bf16"), (dict(kt=132), "16 bytes"), (dict(v=A + 8), "16 bytes"),
    (dict(tokens=-1), "tokens"), (dict(slots=None), "null"), (dict(page=8), "page"), (dict(kc=None), "null")])
def test_append_refuses(kw, match):
    a = dict(k=A, kt=512, kh=128, v=A, vt=512, vh=128, xd=1, slots=A, tokens=4, kc=A, vc=A, ks=A, vs=A, code=0, pages=8,
             hk=2, page=16, dim=128, status=None, stream=None)
    a.update(kw)
    lib, err = _lib()
    assert lib.exl3_kv_append(_pack("PACK_KV_APPEND", a), None) == ARG and match in err()


@pytest.mark.parametrize("kw,match", [
    (dict(req=-1), "requests"), (dict(req=1 << 20), "requests"), (dict(page=17), "page"), (dict(n=-1), "sizes"),
    (dict(cursor=None), "null"), (dict(free=None), "null"), (dict(slots=None), "null"), (dict(table=None), "null")])
def test_plan_refuses(kw, match):
    a = dict(lens=A, new=A, req=4, table=A, width=4, free=A, n_free=9, cursor=A, page=16, n=8, kv=A, cu=A, pos=A, slots=A,
             cur=A, status=None, stream=None)
    a.update(kw)
    lib, err = _lib()
    assert lib.exl3_kv_plan(_pack("PACK_KV_PLAN", a), None) == ARG and match in err()


@pytest.mark.parametrize("kw,rc,match", [
    (dict(xd=3), ARG, "logits"), (dict(ids=0), ARG, "tokens"), (dict(vocab=0), ARG, "vocab"), (dict(top=33), ARG, "top"),
    (dict(vocab=4, top=5), ARG, "top"), (dict(rows=-1), ARG, "rows"), (dict(stride=99), ARG, "overlap"),
    (dict(x=None), ARG, "null"), (dict(tid=None), ARG, "null"), (dict(x=A + 2, xd=0), ARG, "misaligned"),
    (dict(wsb=8), WS, "workspace"), (dict(rows=0), OK, "")])
def test_logprobs_refuses(kw, rc, match):
    a = dict(x=A, xd=2, rows=2, stride=100, vocab=100, tok=A, ids=4, top=3, lp=A, ent=A, rank=A, tlp=A, tid=A, ws=A,
             wsb=1 << 30, stream=None)
    a.update(kw)
    lib, err = _lib()
    assert lib.exl3_token_logprobs(_pack("PACK_TOKEN_LOGPROBS", a), None) == rc and (rc == OK or match in err())


def test_packed_structs_match_the_header():
    """Every struct of the header has one 8-byte field per packed value, the double where it is packed."""
    import os
    import re
    from conftest import ROOT
    from exl3_b200 import _native
    with open(os.path.join(ROOT, "include", "exl3_b200.h")) as f:
        text = re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)
    found = re.findall(r"typedef struct \w+ \{(.*?)\} exl3_(\w+)_args;", text, flags=re.S)
    assert {n for _, n in found} == {"kv_plan", "kv_append", "kv_attend", "token_logprobs"}
    for body, name in found:
        kinds = []
        for decl in filter(None, (d.strip() for d in body.split(";"))):
            assert re.match(r"(const )?(void|int|float|int32_t|int64_t|double)\b", decl)
            for field in decl.split(","):
                assert "*" in field or "int64_t" in decl or "double" in decl, decl
                kinds.append("d" if "double" in decl else "q")
        pack = getattr(_native, "PACK_" + name.upper())
        fmt = pack.__self__.format
        want = "".join(c * int(n or 1) for n, c in re.findall(r"(\d*)([qd])", fmt))
        assert "".join(kinds) == want, name
    lib, err = _lib()
    for name in ("kv_plan", "kv_append", "kv_attend", "token_logprobs"):
        assert getattr(lib, "exl3_" + name)(None, None) == ARG and "null" in err()


def test_binding_loads_and_steps_aside():
    """The compiled short way is there, and takes nothing it should not: CPU tensors, wrong kinds, wrong counts."""
    import torch
    from exl3_b200 import _native
    short = _native.binding()
    assert short is not _native._NoBinding and short.__name__ == "_serving_py"
    t, f = torch.zeros(1, dtype=torch.int32), torch.zeros(2, 4)
    c, s = torch.zeros(1, 1, 16, 64, dtype=torch.int8), torch.zeros(1, 1)
    assert short.kv_plan(t, t, t.view(1, 1), t, t, 16, 1) is None
    assert short.kv_plan(t, t, t.view(1, 1), t, t, 16, 1.5) is None
    assert short.kv_append(f, f, t, c, c, s, s) is None
    assert short.kv_attend(f, c, c, s, s, t.view(1, 1), t, None, 1, None, 0, False) is None
    assert short.token_logprobs(f, t, 1) is None
    assert short.token_logprobs(f, "tokens", 1) is None
    assert short.token_logprobs(f, t, 1 << 70) is None
    with pytest.raises(TypeError):
        short.kv_plan(t)


def test_cpu_tensors_fail_loudly():
    import torch
    from exl3_b200 import kv_cache, logprobs
    t = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        kv_cache.kv_plan(t, t, t.view(1, 1), t, t, page_size=16, n_tokens=1)
    c, s = torch.zeros(1, 1, 16, 64, dtype=torch.int8), torch.zeros(1, 1)
    x = torch.zeros(1, 1, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        kv_cache.kv_append(x, x, t.long(), c, c, s, s)
    with pytest.raises(RuntimeError, match="CUDA"):
        kv_cache.kv_attend(x, c, c, s, s, t.view(1, 1), t)
    with pytest.raises(RuntimeError, match="CUDA"):
        logprobs.token_logprobs(torch.zeros(1, 4), torch.zeros(1, dtype=torch.int64))


def test_plain_forms_agree_with_hand_values():
    """The oracle itself, on values worked out by hand."""
    import numpy as np
    import serving_ref as ref
    assert [ref.scale_exponent(a, "e4m3") for a in (0, 448, 449, 224, 1)] == [-40, 0, 1, -1, -8]
    assert [ref.scale_exponent(a, "int8") for a in (127, 128, 63.5, 1e30)] == [0, 1, -1, 40]
    assert ref.round_code([17.0, 18.0, 19.0, 0.5 * 2 ** -9, 1.5 * 2 ** -9, 500], "e4m3").tolist() == \
        [16.0, 18.0, 20.0, 0.0, 2 ** -8, 448.0]
    kv, cu, pos, slots, cur, tab = ref.plan([15, 0], [2, 1], np.array([[3, -1], [-1, -1]]), [9, 8, 7], 1, 16, 4)
    assert kv.tolist() == [17, 1] and cu.tolist() == [0, 2, 3] and pos.tolist() == [15, 16, 0, 0]
    assert slots.tolist() == [63, 128, 112, -1] and cur == 3 and tab.tolist() == [[3, 8], [7, -1]]
    lp, ent, rank, vals, ids = ref.logprobs(np.log([[0.5, 0.25, 0.25]]), [2], 3)
    assert np.allclose(lp, np.log(0.25)) and np.allclose(ent, 1.5 * np.log(2)) and rank.tolist() == [3]
    assert ids.tolist() == [[0, 1, 2]]

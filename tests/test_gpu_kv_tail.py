"""GPU: attention where a few keys take nearly all of the weight and hold no
value, and all that comes out is the tail of the others.

Error of an output: a weight enters the product in f16.  Relative to the largest
weight of its part, which is 2^7 at least, it is off by 2^-11 of itself and,
below f16's normal range, by 2^-25 / 2^7 = 2^-32: with the largest weight's share
P of the sum, n keys: (2^-11 + 2^-13) sum p |v| + n 2^-32 P max |v|, and the
output's own rounding u |out| (2^-8 bf16).
"""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("requests,new,keys", [(40, 1, 4096), (24, 5, 3000), (2, 130, 4096), (1, 700, 9000)])
@pytest.mark.parametrize("octaves", [16.0, 22.0, 24.5, 25.25, 28.0])
def test_tail_behind_sinks(native, cuda, octaves, requests, new, keys, dim, code):
    """Every 16th key is a sink with v = 0, the others score `octaves` powers of two less."""
    import torch
    from exl3_b200.kv_cache import kv_attend
    P, kv_heads, heads = 32, 2, 8
    width = -(-keys // P)
    pages = requests * width
    kind = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}[code]
    g = torch.Generator(device=cuda).manual_seed(keys + dim)
    kc = torch.zeros(pages, kv_heads, P, dim, device=cuda)
    kc[:, :, ::16] = 1.0                                           # a sink's score is sum q = dim * q0 * 2^-2
    v = torch.randint(1, 16, (pages, kv_heads, P, dim), generator=g, device=cuda).float()
    v[:, :, ::16] = 0.0
    scale = octaves * float(np.log(2.0)) / dim                     # with q = 4, K scale 2^-2
    q = torch.full((requests * new, heads, dim), 4.0, dtype=torch.bfloat16, device=cuda)
    table = torch.arange(pages, dtype=torch.int32, device=cuda).view(requests, width)
    cu = torch.arange(0, requests * new + 1, new, dtype=torch.int32, device=cuda)
    out, lse = kv_attend(q, kc.to(kind), v.to(kind), torch.full((pages, kv_heads), 0.25, device=cuda),
                         torch.full((pages, kv_heads), 0.5, device=cuda), table,
                         torch.full((requests,), keys, dtype=torch.int32, device=cuda), cu_tokens=cu, max_new=new,
                         scale=scale, return_lse=True)
    got = out.double().view(requests, new, kv_heads, heads // kv_heads, dim)
    vals = v.double().mul(0.5).view(requests, width, kv_heads, P, dim).transpose(2, 3).reshape(requests, -1, kv_heads, dim)
    small = 2.0 ** -octaves
    for i in {0, new // 2, new - 1}:
        seen = keys - new + i + 1
        sinks = -(-seen // 16)
        total = sinks + (seen - sinks) * small
        want = vals[:, :seen].sum(1) * small / total
        tol = 2.0 ** -8 * want + (2.0 ** -11 + 2.0 ** -13) * want + seen * 2.0 ** -32 / total * 7.5
        for h in range(heads // kv_heads):
            assert bool(((got[:, i, :, h] - want).abs() <= tol).all()), (i, h, float((got[:, i, :, h] / want).mean()))
        wl = octaves * np.log(2.0) + np.log(total)
        assert float((lse.double().view(requests, new, heads)[:, i] - wl).abs().max()) <= 2.0 ** -17 * (1 + wl) + dim * 2.0 ** -23 * 20

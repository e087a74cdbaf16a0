"""A small decoder served with the package: paged 8-bit cache, attention over it,
EXL3 routed experts and token log probabilities.

    python examples/decoder_step.py

Three requests with prompts of different lengths are prefilled in one step,
then decoded greedily token by token; every step is kv_plan, and per layer
kv_append, kv_attend and the routed experts, then token_logprobs.  At the end
the finished texts are scored in a single prompt pass, the way a pack's
quality is measured, and the two sets of log probabilities are compared.
Weights are random (seeded); the experts are the synthetic EXL3 packs of the
benchmark's smallest configuration.
"""

import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vllm-exl3_b200"))

from exl3_b200 import moe, synthetic  # noqa: E402
from exl3_b200.kv_cache import Exl3KvCache  # noqa: E402
from exl3_b200.logprobs import token_logprobs  # noqa: E402

HIDDEN, HEADS, KV_HEADS, DIM, VOCAB, LAYERS = 1024, 8, 2, 128, 4096, 2


def norm(x):
    return x * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-6).to(x.dtype)


def rotate(x, positions):
    """Rotary positions on [rows, heads, DIM]."""
    half = DIM // 2
    angle = positions.float()[:, None] * 10000.0 ** (-torch.arange(half, device=x.device) / half)
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    a, b = x[..., :half].float(), x[..., half:].float()
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1).to(x.dtype)


class Decoder:
    def __init__(self, device, seed=0):
        g = torch.Generator(device=device).manual_seed(seed)
        draw = lambda *s: (torch.randn(*s, generator=g, device=device) * s[-1] ** -0.5).bfloat16()  # noqa: E731
        self.embed = draw(VOCAB, HIDDEN) * HIDDEN ** 0.5
        self.head = draw(VOCAB, HIDDEN) * 3.0
        self.layers = []
        for i in range(LAYERS):
            pack, *_ = synthetic.make_config("cfg1", seed=seed + i, tokens=1)
            self.layers.append(dict(qkv=draw((HEADS + 2 * KV_HEADS) * DIM, HIDDEN), out=draw(HIDDEN, HEADS * DIM),
                                    router=draw(len(pack.experts), HIDDEN), experts=moe.layer_from_pack(pack, device)))

    def step(self, tokens, plan, cache, max_new):
        """Logits (fp32) of the step's token rows; their keys and values go into the cache."""
        x = self.embed[tokens]
        for i, layer in enumerate(self.layers):
            qkv = (norm(x) @ layer["qkv"].T).view(-1, HEADS + 2 * KV_HEADS, DIM)
            q, k = rotate(qkv[:, :HEADS], plan.positions), rotate(qkv[:, HEADS:HEADS + KV_HEADS], plan.positions)
            cache.append(i, k, qkv[:, HEADS + KV_HEADS:], plan)
            x = x + cache.attend(i, q, plan, max_new).flatten(1) @ layer["out"].T
            h = norm(x)
            # every expert takes part, so that no near tie of the router can tell two runs apart
            weight, ids = torch.softmax((h @ layer["router"].T).float(), -1).sort(-1, descending=True)
            x = x + layer["experts"].apply(h, weight, ids)
        return (norm(x) @ self.head.T).float()


def new_cache(device, requests, max_len, dtype):
    pages = requests * -(-max_len // 16)
    return Exl3KvCache(LAYERS, pages, KV_HEADS, DIM, requests=requests, max_len=max_len, page_size=16, dtype=dtype,
                       device=device)


def run(device="cuda", steps=12, dtype=torch.float8_e4m3fn, verbose=False):
    """Returns (log probabilities while decoding, the same tokens' when scored in one pass, ranks), per request."""
    device = torch.device(device)
    model = Decoder(device)
    g = torch.Generator().manual_seed(1)
    texts = [torch.randint(0, VOCAB, (n,), generator=g).tolist() for n in (37, 5, 64)]
    B = len(texts)
    prompt = [len(t) for t in texts]
    cache = new_cache(device, B, max(prompt) + steps, dtype)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731

    # the prompts, then single tokens
    tokens = torch.tensor([t for text in texts for t in text], device=device)
    plan = cache.plan(i32(prompt), sum(prompt))
    logits = model.step(tokens, plan, cache, max(prompt))[plan.cu_tokens[1:].long() - 1]
    decoded, ranks = [], []
    for s in range(steps):
        cache.commit(plan)
        best = token_logprobs(logits, logits.argmax(1), top=3)
        tokens = best.top_ids[:, 0].long()
        decoded.append(best.logprob)
        ranks.append(best.rank)
        for text, t in zip(texts, tokens.tolist()):
            text.append(t)
        if verbose:
            print(f"step {s:2d}  tokens {tokens.tolist()}  log p {[f'{v:.3f}' for v in best.logprob.tolist()]}"
                  f"  entropy {[f'{v:.2f}' for v in best.entropy.tolist()]}")
        if s + 1 < steps:
            plan = cache.plan(i32([1] * B), B)
            logits = model.step(tokens, plan, cache, 1)

    # the finished texts in one pass
    lens = [len(t) - 1 for t in texts]
    cache = new_cache(device, B, max(lens), dtype)
    plan = cache.plan(i32(lens), sum(lens))
    rows = torch.tensor([t for text in texts for t in text[:-1]], device=device)
    following = torch.tensor([t for text in texts for t in text[1:]], device=device)
    scored = token_logprobs(model.step(rows, plan, cache, max(lens)), following).logprob.split(lens)
    decoded = list(torch.stack(decoded).T)
    return decoded, [s[-steps:] for s in scored], torch.stack(ranks).T


if __name__ == "__main__":
    decoded, scored, _ = run(verbose=True)
    for b, (d, s) in enumerate(zip(decoded, scored)):
        print(f"request {b}: mean log p {d.mean():.4f} while decoding, {s.mean():.4f} scored in one pass, "
              f"largest difference {(d - s).abs().max():.4f}")

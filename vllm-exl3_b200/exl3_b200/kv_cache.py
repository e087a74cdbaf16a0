"""A decoder step's paged key/value cache, held in 8 bits, on the B200 kernels.

A step is ``kv_plan`` (pages and slots from the requests' lengths), then per
layer ``kv_append`` (the step's keys and values into the cache) and
``kv_attend`` (attention over it).  The caches are codes ``[pages, kv_heads,
page, dim]`` (``torch.float8_e4m3fn`` or ``torch.int8``; page 16, 32, 64 or
128; dim 64 or 128) with one power-of-two scale per (page, kv head) in fp32
``[pages, kv_heads]``: value = code * scale.  Nothing here synchronises; all
three can be captured in a CUDA graph once each shape has run before.

:class:`Exl3KvCache` keeps the tensors of one model's layers together.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native as _n

PAGES = (16, 32, 64, 128)
DIMS = (64, 128)
_CODES = {torch.float8_e4m3fn: 0, torch.int8: 1}
_ROWS = {torch.float16: _n.DT_F16, torch.bfloat16: _n.DT_BF16}


class KvPlan(NamedTuple):
    kv_lens: torch.Tensor    # int32 [requests] tokens held after the step
    cu_tokens: torch.Tensor  # int32 [requests + 1] first token row of each request
    positions: torch.Tensor  # int32 [n_tokens] position of each row in its request
    slots: torch.Tensor      # int64 [n_tokens] page * page_size + offset, -1: none
    cursor: torch.Tensor     # int32 [1] the free list's cursor after the step


def _int32(t: torch.Tensor, name: str, who: str, dim: int = 1) -> None:
    if t.dtype != torch.int32 or t.dim() != dim or not t.is_contiguous():
        raise ValueError(f"{who}: {name} must be a contiguous int32 tensor of {dim} dimension(s)")


def _workspace(dev: torch.device, stream: int, nbytes: int = 0) -> torch.Tensor:
    return _n.zeroed_workspace(dev, nbytes, stream)


def kv_plan(lens: torch.Tensor, new_tokens: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
            cursor: torch.Tensor, *, page_size: int, n_tokens: int) -> KvPlan:
    """Pages, slots and positions of a step in which request b, holding
    ``lens[b]`` tokens, adds ``new_tokens[b]``.

    ``n_tokens`` is the number of token rows of the step (rows past the last
    request get slot -1).  Pages a request lacks are taken from
    ``free_pages[cursor:]`` in request order and entered into ``block_table``
    (int32 [requests, width], updated in place); the inputs ``lens``,
    ``cursor`` and ``free_pages`` stay as they are, the result carries their
    successors.  A free list or a table that runs out gives slots of -1 and
    records status 7 (``_native`` workspaces, ``vllm_exl3_c.device_status``).
    """
    who = "kv_plan"
    _n.require_cuda(lens, new_tokens, block_table, free_pages, cursor, who=who)
    for t, name in ((lens, "lens"), (new_tokens, "new_tokens"), (free_pages, "free_pages"), (cursor, "cursor")):
        _int32(t, name, who)
    _int32(block_table, "block_table", who, 2)
    B = lens.numel()
    if new_tokens.numel() != B or block_table.size(0) != B or cursor.numel() != 1:
        raise ValueError(f"{who}: lens, new_tokens and block_table must have one row per request, cursor one value")
    if page_size not in PAGES:
        raise ValueError(f"{who}: page_size must be one of {PAGES}")
    n_tokens = int(n_tokens)
    if n_tokens < 0:
        raise ValueError(f"{who}: n_tokens must be >= 0")
    dev = lens.device
    with _n.on_device(dev):
        stream = _n.raw_stream(dev)
        # one buffer: slots (8 bytes a token) first, then the int32 results
        buf = torch.empty(3 * n_tokens + 2 * B + 2, dtype=torch.int32, device=dev)
        at = buf.data_ptr()
        p_pos, p_lens = at + 8 * n_tokens, at + 12 * n_tokens
        p_cu = p_lens + 4 * B
        _n.check(_n.load().exl3_kv_plan(
            lens.data_ptr(), new_tokens.data_ptr(), B, block_table.data_ptr(), block_table.size(1),
            free_pages.data_ptr(), free_pages.numel(), cursor.data_ptr(), page_size, n_tokens, p_lens, p_cu, p_pos, at,
            p_cu + 4 * B + 4, _workspace(dev, stream).data_ptr(), stream), who)
    slots, pos, kv_lens, cu, cur = buf.split((2 * n_tokens, n_tokens, B, B + 1, 1))
    return KvPlan(kv_lens, cu, pos, slots.view(torch.int64), cur)


def _check_cache(k_cache, v_cache, k_scale, v_scale, who: str) -> tuple[int, int, int, int, int]:
    _n.require_cuda(k_cache, v_cache, k_scale, v_scale, who=who)
    code = _CODES.get(k_cache.dtype)
    if code is None or v_cache.dtype != k_cache.dtype:
        raise ValueError(f"{who}: the caches must both be float8_e4m3fn or both int8")
    shape = k_cache.shape
    if len(shape) != 4 or v_cache.shape != shape or not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError(f"{who}: the caches must be contiguous [pages, kv_heads, page, dim] of one shape")
    pages, heads, page, dim = shape
    if page not in PAGES or dim not in DIMS:
        raise ValueError(f"{who}: page must be one of {PAGES} and dim one of {DIMS} (got {page}, {dim})")
    for s in (k_scale, v_scale):
        if s.dtype != torch.float32 or s.shape != (pages, heads) or not s.is_contiguous():
            raise ValueError(f"{who}: scales must be contiguous fp32 [pages, kv_heads]")
    return code, pages, heads, page, dim


def _rows(x: torch.Tensor, bytes_: int) -> torch.Tensor:
    """x, or a copy of it, with rows that start at multiples of ``bytes_``."""
    a, b, c = x.stride()
    n = bytes_ // 2
    return x if c == 1 and a % n == 0 and b % n == 0 and x.data_ptr() % bytes_ == 0 else x.contiguous()


def kv_append(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
              k_scale: torch.Tensor, v_scale: torch.Tensor) -> None:
    """Writes new rows ``k``, ``v`` (fp16 or bf16 [tokens, kv_heads, dim],
    slices of a fused projection included) into the cache at ``slots`` (int64,
    from :func:`kv_plan`; negative: skipped).

    A page's scale is set by the call that writes its first token and grows
    when a later token needs it, the older codes being rounded to it again.
    """
    who = "kv_append"
    code, pages, heads, page, dim = _check_cache(k_cache, v_cache, k_scale, v_scale, who)
    _n.require_cuda(k, v, slots, who=who)
    x = _ROWS.get(k.dtype)
    if x is None or v.dtype != k.dtype:
        raise ValueError(f"{who}: k and v must both be fp16 or both bf16")
    n = slots.numel()
    if k.shape != (n, heads, dim) or v.shape != (n, heads, dim):
        raise ValueError(f"{who}: k and v must be [{n}, {heads}, {dim}] (slots, kv heads, dim)")
    if slots.dtype != torch.int64 or not slots.is_contiguous():
        raise ValueError(f"{who}: slots must be contiguous int64")
    if n == 0:
        return
    k, v = _rows(k, 8), _rows(v, 8)
    dev = k_cache.device
    with _n.on_device(dev):
        stream = _n.raw_stream(dev)
        _n.check(_n.load().exl3_kv_append(
            k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), x, slots.data_ptr(), n,
            k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), code, pages, heads, page,
            dim, _workspace(dev, stream).data_ptr(), stream), who)


def kv_attend(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
              v_scale: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor, *,
              cu_tokens: torch.Tensor | None = None, max_new: int = 1, scale: float | None = None, window: int = 0,
              return_lse: bool = False) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Causal attention of ``q`` (fp16 or bf16 [rows, heads, dim]) over the cache.

    Request b's rows are ``cu_tokens[b]:cu_tokens[b + 1]`` (one row per request
    when ``cu_tokens`` is None); they are its last tokens of ``kv_lens[b]``,
    already appended.  ``max_new`` is the most rows of a request.  ``heads`` is
    a multiple of the cache's kv heads.  ``window`` limits a row to the last
    ``window`` keys, its own included (0: no limit); ``scale`` defaults to
    dim ** -0.5.  Rows that see no key are zeros (lse -inf).
    """
    who = "kv_attend"
    code, pages, kv_heads, page, dim = _check_cache(k_cache, v_cache, k_scale, v_scale, who)
    _n.require_cuda(q, block_table, kv_lens, cu_tokens, who=who)
    x = _ROWS.get(q.dtype)
    if x is None or q.dim() != 3 or q.size(2) != dim:
        raise ValueError(f"{who}: q must be fp16 or bf16 [rows, heads, {dim}]")
    rows, heads, _ = q.shape
    if heads == 0 or heads % kv_heads:
        raise ValueError(f"{who}: heads ({heads}) must be a multiple of kv_heads ({kv_heads})")
    _int32(block_table, "block_table", who, 2)
    _int32(kv_lens, "kv_lens", who)
    B = kv_lens.numel()
    if block_table.size(0) != B:
        raise ValueError(f"{who}: block_table must have one row per request")
    if cu_tokens is None:
        if rows != B or max_new != 1:
            raise ValueError(f"{who}: without cu_tokens every request has one row of q")
    else:
        _int32(cu_tokens, "cu_tokens", who)
        if cu_tokens.numel() != B + 1:
            raise ValueError(f"{who}: cu_tokens must have one entry more than there are requests")
    if max_new < 1 or window < 0:
        raise ValueError(f"{who}: max_new must be >= 1 and window >= 0")
    q = _rows(q, 16)
    dev = k_cache.device
    out = torch.empty((rows, heads, dim), dtype=q.dtype, device=dev)
    lse = torch.empty((rows, heads), dtype=torch.float32, device=dev) if return_lse else None
    with _n.on_device(dev):
        lib = _n.load()
        stream = _n.raw_stream(dev)
        ws = _workspace(dev, stream, lib.exl3_kv_attend_workspace_size(heads, kv_heads, dim, max_new, B, rows))
        _n.check(lib.exl3_kv_attend(
            q.data_ptr(), q.stride(0), q.stride(1), x, rows, heads, k_cache.data_ptr(), v_cache.data_ptr(),
            k_scale.data_ptr(), v_scale.data_ptr(), code, pages, kv_heads, page, dim, block_table.data_ptr(),
            block_table.size(1), B, kv_lens.data_ptr(), _n.ptr(cu_tokens), max_new,
            dim ** -0.5 if scale is None else float(scale), int(window), out.data_ptr(), _n.ptr(lse), ws.data_ptr(),
            ws.numel(), stream), who)
    return (out, lse) if return_lse else out


class Exl3KvCache:
    """The cache of a model's attention layers: one (codes, scales) set per
    layer, and one block table, free list and length per request row for all.

    A step: ``plan = cache.plan(new_tokens, n_tokens)``, then for every layer
    ``cache.append(layer, k, v, plan)`` and ``cache.attend(layer, q, plan,
    max_new)``, then ``cache.commit(plan)``.  ``release(row)`` hands a finished
    request's pages back (host side, between steps).
    """

    def __init__(self, layers: int, pages: int, kv_heads: int, dim: int, *, requests: int, max_len: int,
                 page_size: int = 16, dtype: torch.dtype = torch.float8_e4m3fn, device: torch.device | str = "cuda"):
        if page_size not in PAGES or dim not in DIMS or dtype not in _CODES:
            raise ValueError(f"Exl3KvCache: page_size in {PAGES}, dim in {DIMS}, dtype float8_e4m3fn or int8")
        self.page_size = page_size
        shape = (layers, pages, kv_heads, page_size, dim)
        self.k = torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype)
        self.v = torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype)
        self.k_scale = torch.ones(shape[:3], dtype=torch.float32, device=device)
        self.v_scale = torch.ones(shape[:3], dtype=torch.float32, device=device)
        self.lens = torch.zeros(requests, dtype=torch.int32, device=device)
        self.block_table = torch.full((requests, -(-max_len // page_size)), -1, dtype=torch.int32, device=device)
        self.free_pages = torch.arange(pages, dtype=torch.int32, device=device)
        self.cursor = torch.zeros(1, dtype=torch.int32, device=device)

    def plan(self, new_tokens: torch.Tensor, n_tokens: int) -> KvPlan:
        return kv_plan(self.lens, new_tokens, self.block_table, self.free_pages, self.cursor,
                       page_size=self.page_size, n_tokens=n_tokens)

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, plan: KvPlan) -> None:
        kv_append(k, v, plan.slots, self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer])

    def attend(self, layer: int, q: torch.Tensor, plan: KvPlan, max_new: int, **kw):
        return kv_attend(q, self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer], self.block_table,
                         plan.kv_lens, cu_tokens=plan.cu_tokens, max_new=max_new, **kw)

    def commit(self, plan: KvPlan) -> None:
        """The step is done: its lengths and its free list's cursor become the cache's."""
        self.lens.copy_(plan.kv_lens)
        self.cursor.copy_(plan.cursor)

    def release(self, row: int) -> None:
        """Gives the pages of request ``row`` back to the free list and empties the row."""
        held = -(-int(self.lens[row]) // self.page_size)
        pages = self.block_table[row, :held]
        pages = pages[pages >= 0]
        at = int(self.cursor) - pages.numel()
        self.free_pages[at:at + pages.numel()] = pages
        self.cursor.fill_(at)
        self.block_table[row].fill_(-1)
        self.lens[row] = 0


__all__ = ["Exl3KvCache", "KvPlan", "kv_append", "kv_attend", "kv_plan"]

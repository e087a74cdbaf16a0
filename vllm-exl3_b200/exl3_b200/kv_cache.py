"""A decoder step's paged key/value cache, held in 8 bits, on the B200 kernels.

A step is ``kv_plan`` (pages and slots from the requests' lengths), then per
layer ``kv_append`` (the step's keys and values into the cache) and
``kv_attend`` (attention over it).  The caches are codes ``[pages, kv_heads,
page, dim]`` (``torch.float8_e4m3fn`` or ``torch.int8``; page 16, 32, 64 or
128; dim 64 or 128) with one power-of-two scale per (page, kv head) in fp32
``[pages, kv_heads]``: value = code * scale.  Nothing here synchronises, and all
three can be captured in CUDA graphs, each with a workspace of its own (the
first captured call of a graph sets it up on the host).

:class:`Exl3KvCache` keeps the tensors of one model's layers together.
"""

from __future__ import annotations

import functools
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


# The operators run for a few microseconds.  A call whose arguments are as the
# kernels want them goes the compiled way (_native.binding); one that needs a
# copy, another device or a refusal goes the way written out here.  It asks
# whether all is well in one expression; _explain says what is not.

def _explain(who: str, *wrong: tuple[bool, str]):
    for bad, what in wrong:
        if bad:
            raise ValueError(f"{who}: {what}")
    raise ValueError(f"{who}: arguments do not fit together")


def _is_i32(t: torch.Tensor, dim: int = 1) -> bool:
    return t.dtype is torch.int32 and t.dim() == dim and t.is_contiguous()


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
    records status 7 (``vllm_exl3_c.device_status``).
    """
    short = _n.binding().kv_plan(lens, new_tokens, block_table, free_pages, cursor, page_size, n_tokens)
    if short is not None:
        return KvPlan(*short)
    B = lens.numel()
    who = "kv_plan"
    _n.require_one_device(lens, new_tokens, block_table, free_pages, cursor, who=who)
    if not (_is_i32(lens) and _is_i32(new_tokens) and _is_i32(free_pages) and _is_i32(cursor)
            and _is_i32(block_table, 2) and new_tokens.numel() == B and block_table.size(0) == B
            and cursor.numel() == 1 and page_size in PAGES and n_tokens >= 0):
        named = (("lens", lens), ("new_tokens", new_tokens), ("free_pages", free_pages), ("cursor", cursor))
        _explain(who, *((not _is_i32(t), f"{n} must be a contiguous int32 tensor of one dimension") for n, t in named),
                 (not _is_i32(block_table, 2), "block_table must be a contiguous int32 tensor of two dimensions"),
                 (page_size not in PAGES, f"page_size must be one of {PAGES}"),
                 (n_tokens < 0, "n_tokens must be >= 0"),
                 (True, "lens, new_tokens and block_table must have one row per request, cursor one value"))
    dev = lens.device.index
    if dev != _n.current_device():
        with torch.cuda.device(dev):
            return kv_plan(lens, new_tokens, block_table, free_pages, cursor, page_size=page_size, n_tokens=n_tokens)
    stream = _n.raw_stream(dev)
    # one buffer: slots (8 bytes a token) first, then the int32 results
    buf = lens.new_empty(3 * n_tokens + 2 * B + 2)
    at = buf.data_ptr()
    p_lens = at + 12 * n_tokens
    p_cu = p_lens + 4 * B
    rc = _n.load().exl3_kv_plan(_n.PACK_KV_PLAN(
        lens.data_ptr(), new_tokens.data_ptr(), B, block_table.data_ptr(), block_table.size(1), free_pages.data_ptr(),
        free_pages.numel(), cursor.data_ptr(), page_size, n_tokens, p_lens, p_cu, at + 8 * n_tokens, at,
        p_cu + 4 * B + 4, _n.serve_workspace(dev, stream)[0]), stream)
    if rc:
        _n.check(rc, "kv_plan")
    slots, pos, kv_lens, cu, cur = torch.unsafe_split_with_sizes(buf, (2 * n_tokens, n_tokens, B, B + 1, 1))
    return KvPlan(kv_lens, cu, pos, slots.view(torch.int64), cur)


def _bad_cache(who: str, k_cache, v_cache, k_scale, v_scale) -> None:
    """Raises what is wrong with a cache, if anything."""
    shape = k_cache.shape
    four = len(shape) == 4 and v_cache.shape == shape and k_cache.is_contiguous() and v_cache.is_contiguous()
    wrong = [(k_cache.dtype not in _CODES or v_cache.dtype != k_cache.dtype,
              "the caches must both be float8_e4m3fn or both int8"),
             (not four or shape[1] == 0, "the caches must be contiguous [pages, kv_heads, page, dim] of one shape")]
    if four:
        wrong += [(shape[2] not in PAGES or shape[3] not in DIMS,
                   f"page must be one of {PAGES} and dim one of {DIMS} (got {shape[2]}, {shape[3]})")]
        wrong += [(t.dtype != torch.float32 or t.shape != shape[:2] or not t.is_contiguous(),
                   "scales must be contiguous fp32 [pages, kv_heads]") for t in (k_scale, v_scale)]
    for bad, what in wrong:
        if bad:
            raise ValueError(f"{who}: {what}")


def _cache_ok(k_cache, v_cache, k_scale, v_scale) -> bool:
    shape = k_cache.shape
    return (k_cache.dtype in _CODES and v_cache.dtype is k_cache.dtype and len(shape) == 4 and v_cache.shape == shape
            and shape[1] > 0 and shape[2] in PAGES and shape[3] in DIMS and k_cache.is_contiguous()
            and v_cache.is_contiguous() and k_scale.dtype is torch.float32 and v_scale.dtype is torch.float32
            and k_scale.shape == shape[:2] and v_scale.shape == shape[:2]
            and k_scale.is_contiguous() and v_scale.is_contiguous())


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x, or a copy of it, with rows that start at multiples of 16 bytes."""
    a, b, c = x.stride()
    return x if c == 1 and not (a | b) & 7 and not x.data_ptr() & 15 else x.clone(memory_format=torch.contiguous_format)


def kv_append(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
              k_scale: torch.Tensor, v_scale: torch.Tensor) -> None:
    """Writes new rows ``k``, ``v`` (fp16 or bf16 [tokens, kv_heads, dim],
    slices of a fused projection included) into the cache at ``slots`` (int64,
    from :func:`kv_plan`; negative: skipped).

    The tokens of a page in one call must be one stretch of rows at
    consecutive slots, which is how :func:`kv_plan` gives them: rows that
    repeat, jump or turn back within the page of the row before them are
    skipped with status 7, and so is what follows a skipped row inside a page.

    A page's scale is set by the call that writes its first token and grows
    when a later token needs it, the older codes being rounded to it again.
    In e4m3 a NaN of ``v`` is kept in the token's key (attention rows that see
    the token become NaN, others do not); int8 has no NaN and takes 0.
    """
    if _n.binding().kv_append(k, v, slots, k_cache, v_cache, k_scale, v_scale):
        return
    n = slots.numel()
    x = _ROWS.get(k.dtype)
    who = "kv_append"
    _n.require_one_device(k_cache, v_cache, k_scale, v_scale, k, v, slots, who=who)
    if not (_cache_ok(k_cache, v_cache, k_scale, v_scale) and x is not None and v.dtype is k.dtype
            and slots.dtype is torch.int64 and slots.is_contiguous() and k.dim() == 3 and k.size(0) == n
            and k.shape[1:] == k_cache.shape[1::2] and v.shape == k.shape):
        _bad_cache(who, k_cache, v_cache, k_scale, v_scale)
        _, heads, _, dim = k_cache.shape
        _explain(who, (x is None or v.dtype != k.dtype, "k and v must both be fp16 or both bf16"),
                 (slots.dtype != torch.int64 or not slots.is_contiguous(), "slots must be contiguous int64"),
                 (True, f"k and v must be [{n}, {heads}, {dim}] (slots, kv heads, dim)"))
    if n == 0:
        return
    dev = k_cache.device.index
    if dev != _n.current_device():
        with torch.cuda.device(dev):
            return kv_append(k, v, slots, k_cache, v_cache, k_scale, v_scale)
    stream = _n.raw_stream(dev)
    k, v = _rows(k), _rows(v)
    kt, kh, _ = k.stride()
    vt, vh, _ = v.stride()
    rc = _n.load().exl3_kv_append(_n.PACK_KV_APPEND(
        k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, x, slots.data_ptr(), n, k_cache.data_ptr(), v_cache.data_ptr(),
        k_scale.data_ptr(), v_scale.data_ptr(), _CODES[k_cache.dtype], *k_cache.shape,
        _n.serve_workspace(dev, stream)[0]), stream)
    if rc:
        _n.check(rc, "kv_append")


@functools.lru_cache(maxsize=1024)
def _attend_bytes(device: int, heads: int, kv_heads: int, dim: int, max_new: int, requests: int, rows: int) -> int:
    return _n.load().exl3_kv_attend_workspace_size(heads, kv_heads, dim, max_new, requests, rows)


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
    dim ** -0.5.  Rows that see no key are zeros (lse -inf).  For inference: a
    backward pass through the result raises.
    """
    short = _n.binding().kv_attend(q, k_cache, v_cache, k_scale, v_scale, block_table, kv_lens, cu_tokens, max_new,
                                   scale, window, return_lse)
    if short is not None:
        return short
    x = _ROWS.get(q.dtype)
    B = kv_lens.numel()
    who = "kv_attend"
    _n.require_one_device(k_cache, v_cache, k_scale, v_scale, q, block_table, kv_lens, cu_tokens, who=who)
    if not (_cache_ok(k_cache, v_cache, k_scale, v_scale) and x is not None and q.dim() == 3
            and q.size(2) == k_cache.size(3) and q.size(1) and not q.size(1) % k_cache.size(1)
            and _is_i32(block_table, 2) and _is_i32(kv_lens) and block_table.size(0) == B and max_new >= 1 and window >= 0
            and ((q.size(0) == B and max_new == 1) if cu_tokens is None
                 else _is_i32(cu_tokens) and cu_tokens.numel() == B + 1)):
        _bad_cache(who, k_cache, v_cache, k_scale, v_scale)
        _, kv_heads, _, dim = k_cache.shape
        _explain(who, (x is None or q.dim() != 3 or q.size(-1) != dim, f"q must be fp16 or bf16 [rows, heads, {dim}]"),
                 (q.dim() == 3 and (q.size(1) == 0 or q.size(1) % kv_heads != 0),
                  f"heads ({q.size(min(1, q.dim() - 1))}) must be a multiple of kv_heads ({kv_heads})"),
                 (not _is_i32(block_table, 2) or block_table.size(0) != B,
                  "block_table must be contiguous int32 with one row per request"),
                 (not _is_i32(kv_lens), "kv_lens must be a contiguous int32 tensor of one dimension"),
                 (max_new < 1 or window < 0, "max_new must be >= 1 and window >= 0"),
                 (cu_tokens is None, "without cu_tokens every request has one row of q"),
                 (True, "cu_tokens must be contiguous int32 with one entry more than there are requests"))
    dev = k_cache.device.index
    if dev != _n.current_device():
        with torch.cuda.device(dev):
            return kv_attend(q, k_cache, v_cache, k_scale, v_scale, block_table, kv_lens, cu_tokens=cu_tokens,
                             max_new=max_new, scale=scale, window=window, return_lse=return_lse)
    stream = _n.raw_stream(dev)
    rows, heads, dim = shape = q.shape
    pages, kv_heads, page, _ = k_cache.shape
    q = _rows(q)
    qt, qh, _ = q.stride()
    out = q.new_empty(shape)
    lse = q.new_empty((rows, heads), dtype=torch.float32) if return_lse else None
    ws, ws_bytes = _n.serve_workspace(dev, stream, _attend_bytes(dev, heads, kv_heads, dim, max_new, B, rows))
    rc = _n.load().exl3_kv_attend(_n.PACK_KV_ATTEND(
        q.data_ptr(), qt, qh, x, rows, heads, k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(),
        v_scale.data_ptr(), _CODES[k_cache.dtype], pages, kv_heads, page, dim, block_table.data_ptr(),
        block_table.size(1), B, kv_lens.data_ptr(), 0 if cu_tokens is None else cu_tokens.data_ptr(), max_new,
        dim ** -0.5 if scale is None else scale, window, out.data_ptr(), 0 if lse is None else lse.data_ptr(),
        ws, ws_bytes), stream)
    if rc:
        _n.check(rc, "kv_attend")
    out = _n.inference_only("kv_attend", out, q)
    return (out, _n.inference_only("kv_attend", lse, q)) if return_lse else out


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

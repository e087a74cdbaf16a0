"""ctypes binding of ``libexl3_b200.so`` (the C ABI in ``include/exl3_b200.h``).

There is no CPU fallback: if the library is missing or cannot load, every
entry raises.  Tensors are passed as raw device pointers; the stream is
torch's current stream of the tensors' device.
"""

from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
import os
import struct
import threading
import warnings

import torch

from . import build as _build

_lock = threading.Lock()
_lib = None

EXL3_OK, EXL3_ERR_ARG, EXL3_ERR_CUDA, EXL3_ERR_WORKSPACE = 0, 1, 2, 3
DT_F32, DT_F16, DT_BF16, DT_I32, DT_I64 = 0, 1, 2, 3, 4
CB_3INST, CB_MCG, CB_MUL1 = 0, 1, 2
ACT_SILU, ACT_RELU2, ACT_SWIGLU_OAI = 0, 2, 3

_DTYPE_CODE = {
    torch.float32: DT_F32,
    torch.float16: DT_F16,
    torch.bfloat16: DT_BF16,
    torch.int32: DT_I32,
    torch.int64: DT_I64,
}

P = ctypes.c_void_p
I32 = ctypes.c_int
I64 = ctypes.c_int64
SZ = ctypes.c_size_t
F32 = ctypes.c_float

# name -> (restype, argtypes); must cover every function in include/exl3_b200.h
SIGNATURES = {
    "exl3_abi_version": (I32, []),
    "exl3_last_error": (ctypes.c_char_p, []),
    "exl3_device_status": (I32, [P, I32, P, ctypes.POINTER(I32)]),
    "exl3_reconstruct": (I32, [P, P, P, I64, I64, I32, I32, P, P]),
    "exl3_decode_raw": (I32, [P, I64, I64, I32, I32, P, P]),
    "exl3_had128": (I32, [P, P, I64, I64, P, P, F32, P]),
    "exl3_linear_workspace_size": (SZ, [I64, I64, I64, I32]),
    "exl3_linear": (I32, [P, I32, I64, P, P, P, I64, I64, I32, I32, P, I32, P, SZ, P]),
    "exl3_moe_workspace_size": (SZ, [I64, I32, I64, I64, I32, I32]),
    "exl3_moe_forward": (
        I32,
        [P, I32, I64, I64, I64, P, P, P, P, P, P, P, P, P, P, I32, P, I32, I32, P, I64,
         P, P, P, I32, I32, I32, I32, I32, F32, P, P, I32, P, SZ, P],
    ),
    "exl3_batched_linear_workspace_size": (SZ, [I64, I32, I64, I64, I32, I32]),
    "exl3_batched_linear": (I32, [P, I32, I64, P, P, P, I32, P, I32, I64, I64, I32, I32, P, I32, P, SZ, P]),
    "exl3_fat_gemm": (I32, [P, I64, P, P, I64, I64, I32, I32, P, P, P, P, SZ, P]),
    "exl3_linear_noalloc": (I32, [P, I32, I64, P, P, P, I64, I64, I32, I32, P, I32, P]),
    "exl3_ep_dispatch": (I32, [P, I32, I64, I64, P, I32, P, I32, I32, I64, I32, P, P, P, P, P, P, P, I64, P]),
    "exl3_ep_combine": (I32, [P, I32, P, I64, I32, I64, P, P, I32, P]),
    "exl3_ep_window_size": (SZ, [I32, I64, I64, I32, I32, I32]),
    "exl3_ep_window_alloc": (I32, [SZ, ctypes.POINTER(P)]),
    "exl3_ep_window_free": (I32, [P]),
    "exl3_ep_ipc_handle": (I32, [P, P]),
    "exl3_ep_ipc_open": (I32, [P, ctypes.POINTER(P)]),
    "exl3_ep_ipc_close": (I32, [P]),
    "exl3_ep_p2p_dispatch": (I32, [P, I32, I64, I64, P, I32, P, I32, I32, I64, I32, I32, I64, P, P, P, I32, P, P]),
    "exl3_ep_p2p_wait": (I32, [P, I32, I32, P]),
    "exl3_ep_p2p_return": (I32, [P, I32, I32, I32, I64, I64, I32, I32, P, P, P]),
    "exl3_ep_p2p_combine": (I32, [P, I32, I32, I64, I64, I32, I32, I32, P, I64, P, P, I32, P]),
    "exl3_ep_window_recv": (I32, [I32, I64, I64, I32, I32, I32, ctypes.POINTER(SZ), ctypes.POINTER(SZ),
                                  ctypes.POINTER(SZ)]),
    "exl3_ngram_dequant": (I32, [P, I64, I32, P, P, I32, P, I32, P]),
    "exl3_ngram_lookup": (I32, [P, I64, I32, P, I32, I64, P, I32, P, P, I32, P, P]),
    # the serving entries take a packed struct of 8-byte fields (see Args)
    "exl3_kv_plan": (I32, [P, P]),
    "exl3_kv_append": (I32, [P, P]),
    "exl3_kv_attend_workspace_size": (SZ, [I32, I32, I32, I32, I32, I64]),
    "exl3_kv_attend": (I32, [P, P]),
    "exl3_token_logprobs_workspace_size": (SZ, [I64, I64, I32, I32]),
    "exl3_token_logprobs": (I32, [P, P]),
    "exl3_capture_id": (ctypes.c_uint64, [P]),
    "exl3_capture_hold": (I32, [P, ctypes.POINTER(P)]),
    "exl3_capture_gone": (I32, [P]),
    "exl3_capture_mode": (I32, [I32]),
    "exl3_profile_enable": (I32, [I32, ctypes.c_longlong]),
    "exl3_profile_read": (I32, [ctypes.POINTER(F32), I32, ctypes.POINTER(I32)]),
}


# exl3_*_args structs: one 8-byte field per argument, in the header's order
# (pointers and integers "q", the attention scale "d")
PACK_KV_PLAN = struct.Struct("16q").pack
PACK_KV_APPEND = struct.Struct("19q").pack
PACK_KV_ATTEND = struct.Struct("21qd5q").pack
PACK_TOKEN_LOGPROBS = struct.Struct("15q").pack


def lib_path() -> str:
    return _build.LIB_PATH


def load():
    """Load (building first if the sources are newer) and bind the library."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        path = _build.LIB_PATH
        if not _build.up_to_date():
            try:
                _build.build()
            except Exception as exc:  # no nvcc on this machine: use the shipped binary
                if not os.path.exists(path):
                    raise RuntimeError(f"EXL3 CUDA library unavailable: {exc}") from exc
        lib = ctypes.CDLL(path)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _lib = lib
        return lib


class _NoBinding:
    """Stands for the serving binding where it could not be built or loaded: every call takes the long way."""

    @staticmethod
    def _none(*args):
        return None

    kv_plan = kv_append = kv_attend = token_logprobs = _none


_binding = None


def binding():
    """The compiled short way into the serving entries (``_serving_py.*.so``).
    Its functions return None where a call needs the checks or copies of the
    Python function, which is complete without them.  Where it cannot be built
    or loaded, whatever the reason, a warning says so once."""
    global _binding
    if _binding is None:
        lib = load()
        try:
            path = _build.build_binding()
            loader = importlib.machinery.ExtensionFileLoader("_serving_py", path)
            mod = importlib.util.module_from_spec(importlib.util.spec_from_loader("_serving_py", loader))
            loader.exec_module(mod)
            names = ("kv_plan", "kv_append", "kv_attend", "kv_attend_workspace_size", "token_logprobs",
                     "token_logprobs_workspace_size", "capture_id")
            mod.setup(*(ctypes.cast(getattr(lib, "exl3_" + n), P).value for n in names), serve_workspace, check)
            _binding = mod
        except Exception as e:
            warnings.warn(f"exl3_b200: no compiled way into the serving operators, their calls take some 10 us more on "
                          f"the host ({type(e).__name__}: {e})", RuntimeWarning, stacklevel=2)
            _binding = _NoBinding
    return _binding


def last_error() -> str:
    return load().exl3_last_error().decode(errors="replace")


def check(rc: int, what: str = "") -> None:
    if rc != EXL3_OK:
        raise RuntimeError(last_error() or f"{what} failed with status {rc}")


def dtype_code(t: torch.Tensor) -> int:
    try:
        return _DTYPE_CODE[t.dtype]
    except KeyError:
        raise RuntimeError(f"unsupported dtype {t.dtype}") from None


def ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def stream_of(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


# torch's current stream of a device (by index) as a raw handle, and the current device
raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)
current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device


def require_cuda(*tensors: torch.Tensor | None, who: str) -> None:
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise RuntimeError(f"{who} requires CUDA tensors (the B200 path has no CPU fallback)")


def require_one_device(*tensors: torch.Tensor | None, who: str) -> None:
    """A kernel that is given another GPU's memory faults: every tensor must be on the first one's GPU."""
    require_cuda(*tensors, who=who)
    where = [t.device for t in tensors if t is not None]
    if any(d != where[0] for d in where):
        raise ValueError(f"{who}: tensors on different GPUs ({', '.join(sorted({str(d) for d in where}))})")


class _NoBackward(torch.autograd.Function):
    @staticmethod
    def forward(ctx, who, result, source):
        ctx.who = who
        return result.view_as(result)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(f"{ctx.who} is for inference: it has no backward pass")


def inference_only(who: str, result: torch.Tensor, source: torch.Tensor) -> torch.Tensor:
    """``result``; where autograd records and ``source`` wants a gradient, in a
    form whose backward pass raises instead of leaving the gradient out."""
    if torch.is_grad_enabled() and source.requires_grad:
        return _NoBackward.apply(who, result, source)
    return result


def profile_enable(on: bool, delay_cycles: int = 0) -> None:
    check(load().exl3_profile_enable(int(bool(on)), int(delay_cycles)))


def profile_read(max_phases: int = 8) -> list[float]:
    """Milliseconds of each kernel phase of the last profiled call."""
    buf = (F32 * max_phases)()
    n = I32(0)
    check(load().exl3_profile_read(buf, max_phases, ctypes.byref(n)))
    return [float(buf[i]) for i in range(n.value)]


_ws_cache: dict[tuple, torch.Tensor] = {}
# Every workspace ever handed out stays referenced for the life of the
# process: a CUDA graph captured with one keeps its address, so freeing it
# when a larger call replaces it would let the next replay write into memory
# that other tensors own.  Growth is geometric, so what is retained is bounded
# by about twice the largest workspace of each (device, stream).
_ws_retired: list[torch.Tensor] = []


def workspace(device: torch.device, nbytes: int, stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """A cached uint8 workspace of at least ``nbytes`` for ``stream`` (torch's
    current stream of ``device`` when None).

    One workspace per (device, stream): calls on one stream run in order, so
    they may share it; calls on different streams never do.  A workspace that
    is too small is replaced by one at least twice as large, and the old one
    is kept alive (see ``_ws_retired``), so graphs captured earlier stay
    valid.  Sizes come from the library's ``*_workspace_size`` queries; call
    each shape once outside capture (a warm-up) so capture finds the
    workspace already large enough.
    """
    if stream is None:
        stream = torch.cuda.current_stream(device)
    key = (device.type, device.index, int(stream.cuda_stream))
    buf = _ws_cache.get(key)
    if buf is None or buf.numel() < nbytes:
        size = max(int(nbytes), 1 << 20)
        if buf is not None:
            size = max(size, 2 * buf.numel())
            _ws_retired.append(buf)
        with torch.cuda.stream(stream):
            buf = torch.empty(size, dtype=torch.uint8, device=device)
            buf[:256].zero_()  # the device status word starts clean
        _ws_cache[key] = buf
    return buf


_serve_ws: dict[tuple[int, int], tuple[int, int]] = {}
_serve_buffers: list[torch.Tensor] = []  # every serving workspace, current and retained


def serve_workspace(index: int, stream: int, nbytes: int = 0, capture: int | None = None) -> tuple[int, int]:
    """(address, bytes) of the workspace of the cache and log-probability
    entries for the raw ``stream`` of device ``index``.  It is kept apart from
    :func:`workspace` because those entries need its counters zero and leave
    them zero.  Grows and is retained in the same way.  ``capture`` is
    ``exl3_capture_id(stream)``, asked here when not given: a call under
    capture gets a workspace of its graph's own."""
    if capture is None:
        capture = load().exl3_capture_id(stream)
    if capture:
        return _captured_workspace(index, stream, capture, nbytes)
    have = _serve_ws.get((index, stream))
    if have is None or have[1] < nbytes:
        key = ("cuda", index, stream, "serve")
        size = max(int(nbytes), 1 << 20)
        old = _ws_cache.get(key)
        if old is not None:
            size = max(size, 2 * old.numel())
            _ws_retired.append(old)
        buf = torch.zeros(size, dtype=torch.uint8, device=torch.device("cuda", index))
        _ws_cache[key] = buf
        _serve_buffers.append(buf)
        have = _serve_ws[(index, stream)] = (buf.data_ptr(), size)
    return have


# A graph's launches run on any stream, beside eager calls and other graphs, so
# what a capture records must not share counters with them: every (capture,
# stream) gets a workspace that belongs to its graph until the graph is gone,
# and then to a later capture.  It is allocated outside the graph's memory and
# zeroed on the device before the capture goes on: a fill recorded in the graph
# would run at each replay, and not before the first.
_captured: dict[tuple[int, int, int], tuple[int, int]] = {}     # (device, stream, capture) -> (address, bytes)
_captured_held: list[tuple[int, tuple[int, int, int], torch.Tensor]] = []  # (token of the graph, key, buffer)
_captured_spare: list[torch.Tensor] = []                        # of graphs that are gone
_captured_lock = threading.Lock()


def _captured_workspace(index: int, stream: int, capture: int, nbytes: int) -> tuple[int, int]:
    key = (index, stream, capture)
    have = _captured.get(key)
    if have is not None and have[1] >= nbytes:
        return have
    lib = load()
    with _captured_lock:
        for held in list(_captured_held):
            if lib.exl3_capture_gone(held[0]):
                _captured_held.remove(held)
                _captured.pop(held[1], None)
                _captured_spare.append(held[2])
        fits = [b for b in _captured_spare if b.device.index == index and b.numel() >= nbytes]
        buf = min(fits, key=torch.Tensor.numel, default=None)
        if buf is not None:
            _captured_spare[:] = [b for b in _captured_spare if b is not buf]
        # The work below is not the graph's: it runs, now, on a stream that is not captured
        before = lib.exl3_capture_mode(2)
        try:
            with torch.cuda.device(index):
                side = next((s for s in (torch.cuda.Stream() for _ in range(64))
                             if s.cuda_stream != stream and not lib.exl3_capture_id(s.cuda_stream)), None)
                if side is None:
                    raise RuntimeError("no stream outside the capture to set up a workspace on")
                with torch.cuda.stream(side):
                    if buf is None:
                        buf = torch.zeros(max(int(nbytes), 1 << 20), dtype=torch.uint8, device=f"cuda:{index}")
                        _serve_buffers.append(buf)
                    else:
                        buf[256:].zero_()  # a status that was recorded in it stays
                side.synchronize()
        finally:
            if before >= 0:
                lib.exl3_capture_mode(before)
        token = P()
        rc = lib.exl3_capture_hold(stream, ctypes.byref(token))
        if rc:
            _captured_spare.append(buf)
            check(rc, "serve_workspace")
        _captured_held.append((token.value, key, buf))
        have = _captured[key] = (buf.data_ptr(), buf.numel())
    return have


def device_workspaces(device: torch.device) -> list[torch.Tensor]:
    """Every workspace handed out on ``device`` (current and retained)."""
    out = [b for k, b in _ws_cache.items() if k[0] == device.type and k[1] == device.index]
    kept = _ws_retired + [held[2] for held in _captured_held] + _captured_spare
    return out + [b for b in kept if b.device == device]


DEV_WAIT_TIMEOUT = 4


def renew_serve_workspace(workspace: torch.Tensor) -> None:
    """Zeroes the counters of a serving workspace in which a wait ran out (on
    the current stream, with none of its calls in flight): items that were
    given up have left theirs behind, and the next call starts from zero."""
    if any(b.data_ptr() == workspace.data_ptr() for b in _serve_buffers):
        workspace[256:].zero_()

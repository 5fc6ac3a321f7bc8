"""ctypes binding of libmfd_b200.so (include/mfd_b200.h).

The library is the only compute path: if it is missing it is built in-tree with nvcc, and if that fails,
or no CUDA device is present, every call raises.  There is no CPU fallback.
"""

from __future__ import annotations

import ctypes
import os
import struct
import threading

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libmfd_b200.so")

_lock = threading.Lock()
_lib = None

c_i64 = ctypes.c_int64
c_int = ctypes.c_int
c_f32 = ctypes.c_float
c_size = ctypes.c_size_t
c_vp = ctypes.c_void_p

# name -> (restype, argtypes)
_SIGS = {
    "mfd_last_error": (ctypes.c_char_p, []),
    "mfd_abi_version": (c_int, []),
    "mfd_topk_logz_workspace": (c_size, [c_i64, c_i64, c_i64]),
    "mfd_topk_logz": (c_int, [c_vp, c_int, c_i64, c_i64, c_i64, c_i64, c_vp, c_vp, c_int, c_vp, c_vp, c_size, c_vp,
                              c_i64, c_vp]),
    "mfd_topk_logz_static": (c_int, [c_vp, c_int, c_i64, c_i64, c_i64, c_i64, c_vp, c_vp, c_int, c_vp, c_vp]),
    "mfd_build_trees": (c_int, [c_vp, c_vp, c_int, c_vp, c_i64, c_i64, c_i64, c_i64, c_i64, c_int, c_vp, c_vp, c_vp,
                                c_vp, c_vp, c_vp]),
    "mfd_accept_workspace": (c_size, [c_i64, c_i64]),
    "mfd_accept_tickets": (c_i64, [c_i64, c_i64]),
    "mfd_accept": (c_int, [c_vp, c_i64, c_i64, c_i64, c_i64, c_vp, c_i64, c_vp, c_i64, c_f32, c_vp, c_i64, c_vp, c_vp,
                           c_i64, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_size, c_vp, c_i64,
                           c_vp]),
    "mfd_sample_tokens_workspace": (c_size, [c_i64]),
    "mfd_sample_tokens": (c_int, [c_vp, c_i64, c_i64, c_i64, c_f32, c_vp, c_vp, c_vp, c_size, c_vp, c_i64, c_vp]),
    "mfd_follow": (c_int, [c_vp, c_vp, c_i64, c_vp, c_i64, c_i64, c_i64, c_i64, c_vp, c_vp, c_i64, c_vp, c_vp, c_vp,
                           c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp]),
    "mfd_verify_inputs": (c_int, [c_vp, c_vp, c_vp, c_vp, c_vp, c_i64, c_vp, c_i64, c_i64, c_i64, c_vp, c_vp, c_vp,
                                  c_vp]),
    "mfd_compile_tree": (c_int, [c_vp, c_vp, c_vp, c_i64, c_vp, c_i64, c_i64, c_i64, c_i64, c_i64, c_vp, c_vp, c_vp,
                                 c_i64, c_i64, c_i64, c_i64, ctypes.c_uint32, c_vp, c_i64, c_vp]),
    "mfd_tree_attention_workspace": (c_size, [c_i64, c_i64, c_i64, c_i64, c_i64]),
    "mfd_tree_attention_tickets": (c_i64, [c_i64, c_i64, c_i64, c_i64]),
    "mfd_tree_attention": (c_int, [c_vp, c_i64, c_i64, c_i64, c_vp, c_i64, c_i64, c_i64, c_vp, c_i64, c_i64, c_i64,
                                   c_i64, c_vp, c_i64, c_vp, c_i64, c_i64, c_i64, c_i64, c_i64, c_i64, c_f32, c_i64,
                                   c_vp, c_i64, c_i64, c_i64, c_vp, c_size, c_vp, c_i64, c_vp]),
    "mfd_paged_mode_attention": (c_int, [c_vp, c_i64, c_i64, c_vp, c_i64, c_i64, c_vp, c_i64, c_i64, c_vp, c_i64,
                                         c_i64, c_vp, c_i64, c_i64, c_i64, c_vp, c_i64, c_i64, c_i64, c_vp, c_vp,
                                         c_vp, c_i64, c_i64, c_i64, c_i64, c_i64, c_i64, c_i64, c_f32, c_i64, c_vp,
                                         c_i64, c_i64, c_vp, c_size, c_vp, c_i64, c_vp]),
    "mfd_tree_gdn": (c_int, [c_vp, c_i64, c_vp, c_i64, c_vp, c_i64, c_vp, c_i64, c_vp, c_i64, c_vp, c_vp, c_i64,
                             c_i64, c_i64, c_i64, c_i64, c_i64, c_vp, c_vp, c_vp, c_vp, c_vp]),
    "mfd_tree_gates": (c_int, [c_vp, c_i64, c_vp, c_i64, c_int, c_vp, c_vp, c_vp, c_i64, c_i64, c_vp, c_vp, c_vp,
                               c_vp]),
    "mfd_tree_prep": (c_int, [c_vp, c_vp, c_vp, c_vp, c_i64, c_i64, c_i64, c_i64, c_i64, c_i64, c_f32, c_vp, c_vp,
                              c_vp, c_vp]),
    "mfd_commit_kv_moves": (c_int, [c_vp, c_i64, c_i64, c_i64, c_vp, c_vp, c_i64, c_i64, c_i64, c_vp, c_vp]),
    "mfd_compact_tail": (c_int, [c_vp, c_i64, c_i64, c_i64, c_i64, c_i64, c_i64, c_i64, c_i64, c_vp, c_i64, c_vp,
                                 c_vp]),
    "mfd_gdn_commit": (c_int, [c_vp, c_int, c_vp, c_vp, c_vp, c_i64, c_vp, c_i64, c_i64, c_i64, c_i64, c_i64, c_i64,
                               c_vp]),
    "mfd_kv8_append": (c_int, [c_vp, c_vp, c_i64, c_i64, c_i64, c_int, c_vp, c_vp, c_i64, c_i64, c_vp, c_i64, c_i64,
                               c_vp, c_vp, c_vp, c_i64, c_i64, c_i64, c_i64, c_vp, c_i64, c_i64, c_vp, c_i64, c_i64,
                               c_i64, c_vp, c_vp, c_vp]),
    "mfd_capture_id": (c_int, [c_vp, c_vp]),
    "mfd_kv8_attention_status": (c_int, [c_vp, c_vp]),
    "mfd_kv8_attention_workspace": (c_size, [c_i64, c_i64, c_i64, c_i64]),
    "mfd_kv8_attention_tickets": (c_i64, [c_i64, c_i64, c_i64, c_i64]),
    "mfd_kv8_attention": (c_int, [c_vp, c_i64, c_i64, c_i64, c_vp, c_vp, c_i64, c_i64, c_i64, c_int, c_vp, c_vp, c_i64,
                                  c_i64, c_vp, c_i64, c_i64, c_vp, c_vp, c_vp, c_i64, c_i64, c_i64, c_vp, c_i64, c_i64,
                                  c_i64, c_i64, c_i64, c_i64, c_f32, c_vp, c_i64, c_i64, c_i64, c_vp, c_vp, c_size,
                                  c_vp, c_i64, c_vp]),
    "mfd_kv8_page_weights_workspace": (c_size, [c_i64, c_i64, c_i64, c_i64]),
    "mfd_kv8_page_weights": (c_int, [c_vp, c_i64, c_i64, c_i64, c_vp, c_vp, c_i64, c_i64, c_i64, c_int, c_vp, c_i64,
                                     c_i64, c_vp, c_i64, c_i64, c_vp, c_vp, c_i64, c_i64, c_vp, c_i64, c_i64, c_i64,
                                     c_i64, c_i64, c_f32, c_f32, c_vp, c_vp, c_i64, c_vp, c_size, c_vp, c_i64, c_vp]),
    "mfd_kv8_evict": (c_int, [c_vp, c_vp, c_vp, c_i64, c_i64, c_i64, c_i64, c_i64, c_i64, c_vp, c_vp, c_vp, c_vp,
                              c_vp, c_vp]),
    "mfd_kv8_call": (c_int, [c_int, ctypes.c_char_p, c_i64]),
    "mfd_conv_commit": (c_int, [c_vp, c_vp, c_i64, c_i64, c_i64, c_i64, c_vp, c_vp]),
}

MFD_F32, MFD_BF16, MFD_I32, MFD_I64, MFD_I8, MFD_E4M3 = 0, 1, 2, 3, 4, 5


def exported_symbols() -> list[str]:
    return list(_SIGS)


def load(build_if_missing: bool = True):
    """Load (building if needed) the library and bind its entry points.  Needs no GPU."""
    global _lib
    with _lock:
        if _lib is not None:
            return _lib
        if not os.path.exists(LIB_PATH):
            if not build_if_missing:
                raise RuntimeError(f"{LIB_PATH} is not built; run python -m mfd_b200.build")
            from . import build as _build

            _build.build()
        lib = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in _SIGS.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _lib = lib
        return lib


def lib():
    return _lib if _lib is not None else load()


def check(rc: int, what: str) -> None:
    if rc != 0:
        msg = lib().mfd_last_error().decode(errors="replace")
        raise RuntimeError(f"{what} failed (status {rc}): {msg}")


def require_cuda(*tensors: torch.Tensor) -> torch.device:
    if not torch.cuda.is_available():
        raise RuntimeError("mfd_b200 needs a CUDA device (no CPU fallback)")
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("mfd_b200: expected CUDA tensors")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise RuntimeError("mfd_b200: tensors on different devices")
    return dev if dev is not None else torch.device("cuda", torch.cuda.current_device())


def stream_ptr(device: torch.device | None = None) -> int:
    return torch.cuda.current_stream(device).cuda_stream


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def device_index(first: torch.Tensor, *rest: torch.Tensor | None) -> int:
    """require_cuda for calls whose host time matters: the CUDA device index all the tensors share, without the
    runtime queries (a CUDA tensor implies a device).  It has to be the current device, on which the kernel runs."""
    idx = first.get_device()
    if idx < 0:
        require_cuda(first)
    for t in rest:
        if t is not None and t.get_device() != idx:
            require_cuda(first, t)
    current = _current_device()
    if idx != current:
        raise RuntimeError(f"mfd_b200: tensors on cuda:{idx} while cuda:{current} is the current device")
    return idx


def raw_stream(idx: int) -> int:
    """The current stream of CUDA device `idx` as an integer."""
    return _raw_stream(idx) if _raw_stream is not None else torch.cuda.current_stream(idx).cuda_stream


_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", torch.cuda.is_current_stream_capturing)


def _recording() -> bool:
    return torch.cuda.is_initialized() and _capturing()


def capture_id(stream: int) -> int:
    """The number of the CUDA graph capture that the current stream (`stream`) records into; 0 when it records none."""
    if not _capturing():
        return 0
    number = ctypes.c_uint64()
    check(lib().mfd_capture_id(stream, ctypes.byref(number)), "mfd_capture_id")
    return number.value


def ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def address(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


def packed(name: str, op: int):
    """Entry point `name` as a function of its arguments through mfd_kv8_call, which takes them as one array (null
    pointers as 0): with 47 arguments a call costs the host 4 us less than their conversion one by one."""
    args = _SIGS[name][1]
    pack, count = struct.Struct("".join("d" if a is c_f32 else "q" for a in args)).pack, len(args)

    def call(*words) -> int:
        return lib().mfd_kv8_call(op, pack(*words), count)

    return call


class Workspace:
    """Per-device, per-purpose scratch, grown on demand, plus one per-device ticket buffer.  Tickets live only in
    the ticket buffer, which starts zeroed and which every ticketed kernel leaves zeroed; scratch needs no
    initialisation.  Calls that share them must be ordered on one stream (as the current-stream launches are).  A buffer
    that was outgrown stays allocated, since a CUDA graph may hold its address (each is at least twice the one before, so
    all of them take less than the last).  One that is made while a graph is captured is zeroed by that graph's replays
    alone, and is left to it."""

    _cache: dict = {}
    _outgrown: list = []

    @classmethod
    def tickets(cls, device: torch.device, n: int) -> torch.Tensor:
        return cls._buffer(device, "__tickets__", int(n), 1024, torch.int32)

    @classmethod
    def get(cls, device: torch.device, purpose: str, nbytes: int) -> torch.Tensor:
        return cls._buffer(device, purpose, int(nbytes), 256, torch.uint8)

    @classmethod
    def _buffer(cls, device: torch.device, purpose, n: int, least: int, dtype: torch.dtype) -> torch.Tensor:
        key = (device.index if device.index is not None else torch.cuda.current_device(), purpose)
        buf = cls._cache.get(key)
        if buf is not None and buf.numel() >= n:
            return buf
        if _recording():
            return torch.zeros(max(n, least), dtype=dtype, device=device)
        size = max(n, least)
        if buf is not None:
            size = max(size, 2 * buf.numel())
            cls._outgrown.append(buf)
        buf = cls._cache[key] = torch.zeros(size, dtype=dtype, device=device)
        return buf


class CaptureScratch:
    """Scratch of calls that are recorded into a CUDA graph: its own for each capture, purpose and stream.

    The workspace is allocated while the graph is captured, so it belongs to the graph's memory pool and lives as long as
    the graph.  The tickets, which have to be zero, are words of a buffer that an earlier plain call zeroed and that is never
    given back (each capture keeps its words); where there is none, or it is used up, a node of the graph zeroes some in
    front of the first call (2 us of a replay).  So a replay depends on no other call, and graphs share no scratch.  (Workspaces
    captured into one pool may overlap: PyTorch wants such graphs replayed in order.)"""

    SPARE = 1 << 22  # bytes of zeroed tickets a device
    _held: dict = {}  # (device index, purpose, stream) -> (capture id, workspace, its bytes, tickets, their bytes)
    _spare: dict = {}  # device index -> (zeroed buffer, bytes taken)

    @classmethod
    def prepare(cls, device: torch.device) -> None:
        """Zero the spare tickets of a device, once; not while capturing.  They are zero when this returns."""
        if device.index not in cls._spare:
            cls._spare[device.index] = torch.zeros(cls.SPARE, dtype=torch.uint8, device=device), 0
            if device.type == "cuda":
                torch.cuda.current_stream(device).synchronize()

    @classmethod
    def _zeroed(cls, device: torch.device, nbytes: int) -> torch.Tensor:
        spare, taken = cls._spare.get(device.index, (None, 0))
        if spare is None or taken + nbytes > spare.numel():
            return torch.zeros(nbytes, dtype=torch.uint8, device=device)
        cls._spare[device.index] = spare, taken + nbytes
        return spare[taken:taken + nbytes]

    @classmethod
    def get(cls, device: torch.device, purpose: str, stream: int, capture: int, nbytes: int, words: int):
        """(workspace, its bytes, tickets, their words), as addresses."""
        key = (device.index, purpose, stream)
        held = cls._held.get(key)
        if held is not None and held[0] != capture:  # (an ended capture's memory stays with its graph)
            del cls._held[key]
            held = None
        if held is None or held[2] < nbytes or held[4] < 4 * words:
            _, ws, had, tk, had_tk = held if held is not None else (0, None, 0, None, 0)
            if had_tk < 4 * words:
                had_tk = -(-4 * words // 256) * 256
                tk = cls._zeroed(device, had_tk)
            if had < nbytes:
                ws, had = torch.empty(nbytes, dtype=torch.uint8, device=device), nbytes
            held = cls._held[key] = capture, ws, had, tk, had_tk
        return held[1].data_ptr(), held[2], held[3].data_ptr(), held[4] // 4

"""ctypes binding of ``libdelrec_b200.so`` (the C-ABI declared in include/delrec_b200.h).

The library is loaded from this directory; nothing here falls back to a CPU or
PyTorch implementation: a missing library, a non-CUDA tensor or a nonzero status
raises.  Scratch memory for the kernels comes from a per-(device, stream) workspace
tensor owned by this module and grown on demand through torch's caching allocator.
"""

from __future__ import annotations

import ctypes
import os

import torch
from torch.autograd import forward_ad

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libdelrec_b200.so")

OK = 0
ERRORS = {1: "invalid argument", 2: "CUDA error", 3: "workspace too small or misaligned",
          4: "unsupported shape"}
AXONAL, SYNAPTIC, HYBRID = 0, 1, 2
HARD_STE, HARD_APPROX = 1, 2     # delrec_axonal_backward_hard modes
SURR_TRIANGLE, SURR_ATAN = 0, 1


class LIF(ctypes.Structure):
    _fields_ = [("tau", ctypes.c_float), ("v_threshold", ctypes.c_float),
                ("v_reset", ctypes.c_float), ("soft_reset", ctypes.c_int32),
                ("detach_reset", ctypes.c_int32), ("surrogate", ctypes.c_int32),
                ("gamma", ctypes.c_float), ("alpha", ctypes.c_float)]


class Layer(ctypes.Structure):
    _fields_ = [("kind", ctypes.c_int32), ("T", ctypes.c_int32), ("B", ctypes.c_int32),
                ("N", ctypes.c_int32), ("L", ctypes.c_int32), ("K", ctypes.c_int32),
                ("has_bias", ctypes.c_int32), ("has_keep", ctypes.c_int32),
                ("s_max", ctypes.c_float), ("d_min", ctypes.c_float)]


class Grads(ctypes.Structure):
    _fields_ = [("dx", ctypes.c_void_p), ("dW", ctypes.c_void_p), ("dbias", ctypes.c_void_p),
                ("dd", ctypes.c_void_p), ("ds", ctypes.c_void_p)]


def _i64(*names):
    return [(n, ctypes.c_int64) for n in names]


class Scan(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in ("T", "B", "N", "G", "dtype", "decay_input", "lengths_wide",
                                              "reserved")] \
        + _i64("z_t", "z_b", "f_t", "f_b", "h_t", "h_b", "gh_t", "gh_b", "dz_t", "dz_b", "df_t", "df_b")


class Block(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in ("T", "B", "N", "dtype", "gate", "lengths_wide")] \
        + [("eps", ctypes.c_float), ("reserved", ctypes.c_int32)] \
        + _i64("x_t", "x_b", "y_t", "y_b", "u_t", "u_b", "o_t", "o_b", "n_t", "n_b", "gx_t", "gx_b", "gn_t",
               "gn_b", "dx_t", "dx_b", "dy_t", "dy_b", "du_t", "du_b")


class Conv(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in ("T", "B", "N", "K", "dtype", "act", "lengths_kind", "reserved")] \
        + _i64("x_t", "x_b", "y_t", "y_b", "gy_t", "gy_b", "dx_t", "dx_b")


class Selective(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in ("T", "B", "N", "S", "G", "dtype", "softplus", "lengths_wide", "ragged",
                                              "no_bc")] \
        + _i64("x_t", "x_b", "dt_t", "dt_b", "u_t", "u_b", "y_t", "y_b", "bm_t", "bm_b", "cm_t", "cm_b", "gy_t",
               "gy_b", "dx_t", "dx_b", "ddt_t", "ddt_b", "du_t", "du_b")


class Vocab(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in ("T", "B", "D", "V", "K", "dtype", "distill", "reduction", "lengths_wide",
                                              "index_wide", "teacher_dtype", "w_aligned")] \
        + [("temperature", ctypes.c_float), ("split", ctypes.c_int32)] + _i64("ignore_index", "x_t", "x_b")


_P = ctypes.c_void_p
_I = ctypes.c_int
_F = ctypes.c_float
_S = ctypes.c_size_t
_SIGS = {
    "delrec_build_mask": (_I, [_I, _I, _P, _P, _I, _P, _P]),
    "delrec_axonal_forward_workspace": (_S, [_P]),
    "delrec_synaptic_forward_workspace": (_S, [_P]),
    "delrec_hybrid_forward_workspace": (_S, [_P]),
    "delrec_axonal_backward_workspace": (_S, [_P]),
    "delrec_synaptic_backward_workspace": (_S, [_P]),
    "delrec_hybrid_backward_workspace": (_S, [_P]),
    "delrec_axonal_forward": (_I, [_P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _S, _P]),
    "delrec_axonal_forward_noalloc": (_I, [_P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P]),
    "delrec_synaptic_forward": (_I, [_P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _S, _P]),
    "delrec_hybrid_forward": (_I, [_P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _S, _P]),
    "delrec_axonal_backward": (_I, [_P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _S, _P]),
    "delrec_axonal_backward_hard_workspace": (_S, [_P]),
    "delrec_axonal_backward_hard": (_I, [_P, _P, _I, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _S, _P]),
    "delrec_synaptic_backward": (_I, [_P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _S, _P]),
    "delrec_hybrid_backward": (_I, [_P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _S, _P]),
    "delrec_hybrid_delay_grad": (_I, [_I, _I, _P, _P, _P, _F, _P, _P]),
    "delrec_lif_forward": (_I, [_I, _I, _P, _P, _P, _P, _P]),
    "delrec_lif_backward": (_I, [_I, _I, _P, _P, _P, _P, _P]),
    "delrec_dcls_forward": (_I, [_I, _I, _I, _I, _I, _I, _I, _P, _P, _P, _P, _P, _P, _P, _P]),
    "delrec_dcls_backward_workspace": (_S, [_I, _I, _I, _I, _I, _I]),
    "delrec_dcls_backward": (_I, [_I, _I, _I, _I, _I, _I, _I, _P, _P, _P, _P, _P, _P, _P, _P,
                                  _P, _P, _P, _S, _P]),
    "delrec_linear_forward_workspace": (_S, [_I, _I, _I, _I]),
    "delrec_linear_forward": (_I, [_I, _I, _I, _P, _P, _P, _I, _P, _P, _S, _P]),
    "delrec_linear_backward_workspace": (_S, [_I, _I, _I, _I]),
    "delrec_linear_backward": (_I, [_I, _I, _I, _P, _P, _P, _I, _P, _P, _P, _P, _S, _P]),
    "delrec_count_nonbinary": (_I, [_P, _S, _P, _P]),
    "delrec_tc_gemm_workspace": (_S, [_I, _I, _I]),
    "delrec_tc_gemm": (_I, [_I, _I, _I, _I, _I, _P, ctypes.c_longlong, _I, _P, ctypes.c_longlong, _I, _P, _P, _I, _I,
                            _P, ctypes.c_longlong, _I, _P, _S, _P]),
    "delrec_get_status": (_I, [_P]),
    "delrec_clear_status": (_I, []),
    "delrec_version": (ctypes.c_char_p, []),
    "delrec_launch_count": (ctypes.c_ulonglong, []),
    "delrec_scan_timing": (_I, [_I]),
    "delrec_scan_time": (_I, [_P, _P]),
    "delrec_scan_time_part": (_I, [_I, _P, _P]),
    "delrec_set_reverse_scan": (_I, [_I]),
    "delrec_readout_sum_forward": (_I, [_I, _I, _I, _I, _P, _P, _P, _P, _P, _P]),
    "delrec_readout_sum_backward": (_I, [_I, _I, _I, _I, _P, _P, _P, _P, _P, _P, _P]),
    "delrec_exchange_floor_workspace": (_S, [_P]),
    "delrec_exchange_floor": (_I, [_P, _P, _S, _P]),
    "delrec_gated_scan_forward": (_I, [_P] * 15),
    "delrec_gated_scan_backward_workspace": (_S, [_P]),
    "delrec_gated_scan_backward": (_I, [_P] * 17 + [_S, _P]),
    "delrec_gated_step": (_I, [_P] * 8),
    "delrec_block_norm_forward": (_I, [_P] * 13),
    "delrec_block_norm_backward_workspace": (_S, [_P]),
    "delrec_block_norm_backward": (_I, [_P] * 19 + [_S, _P]),
    "delrec_pack8": (_I, [ctypes.c_longlong, _I, _I, _P, _P, _P, _P]),
    "delrec_unpack8": (_I, [ctypes.c_longlong, _I, _I, _P, _P, _P, _P]),
    "delrec_linear_forward8": (_I, [_I, _I, _I, _P, _P, _P, _I, _P, _P, _P, _P, _S, _P]),
    "delrec_linear_backward8_workspace": (_S, [_I, _I, _I]),
    "delrec_short_conv_forward": (_I, [_P] * 10),
    "delrec_short_conv_backward_workspace": (_S, [_P]),
    "delrec_short_conv_backward": (_I, [_P] * 14 + [_S, _P]),
    "delrec_selective_forward_workspace": (_S, [_P]),
    "delrec_selective_forward": (_I, [_P] * 16 + [_S, _P]),
    "delrec_selective_backward_workspace": (_S, [_P]),
    "delrec_selective_backward": (_I, [_P] * 24 + [_S, _P]),
    "delrec_selective_step": (_I, [_P] * 14),
    "delrec_vocab_loss_keep": (_S, [_P]),
    "delrec_vocab_loss_forward_workspace": (_S, [_P]),
    "delrec_vocab_loss_forward": (_I, [_P] * 9 + [_S, _P, _S, _P]),
    "delrec_vocab_loss_backward_workspace": (_S, [_P]),
    "delrec_vocab_loss_backward": (_I, [_P] * 6 + [_S] + [_P] * 4 + [_S, _P]),
    "delrec_linear_backward8": (_I, [_I, _I, _I, _P, _P, _P, _P, _P, _P, _P, _P, _S, _P]),
}

_lib = None


def lib():
    """The loaded library (raises if it was not built)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                f"delrec_b200: CUDA library not found at {LIB_PATH}; build it with "
                "`python -c 'import __graft_entry__ as g; g.build()'` (or `make` in csrc/)")
        handle = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in _SIGS.items():
            fn = getattr(handle, name)
            fn.restype = res
            fn.argtypes = args
        _lib = handle
    return _lib


def exported_symbols():
    return list(_SIGS)


def check(rc: int, what: str):
    if rc != OK:
        raise RuntimeError(f"delrec_b200: {what} failed: {ERRORS.get(rc, rc)} (code {rc})")


def ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def require_cuda(*tensors):
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("delrec_b200 runs on CUDA tensors only (there is no CPU path)")
        if t.dtype != torch.float32:
            raise RuntimeError(f"delrec_b200 expects float32 tensors, got {t.dtype}")
        if not t.is_contiguous():
            raise RuntimeError("delrec_b200 expects contiguous tensors")


def stream_ptr(device=None):
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


# ---- sequence operators (gated, block_norm, checkpoint8) ---------------------------------

SEQ_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def require_sequence(t):
    """The dtype code of t; raises unless it is a CUDA tensor of a type the sequence operators
    take."""
    if not t.is_cuda:
        raise RuntimeError("delrec_b200 runs on CUDA tensors only (there is no CPU path)")
    code = SEQ_DTYPES.get(t.dtype)
    if code is None:
        raise RuntimeError(f"delrec_b200 expects float32, bfloat16 or float16 tensors, got {t.dtype}")
    return code


def require_sizes(*sizes):
    """The library's sizes are 32-bit."""
    for n in sizes:
        if n > 0x7fffffff:
            raise RuntimeError(f"delrec_b200: a dimension of {n} is past the library's 32-bit sizes")


def require_lengths(lengths, B, device):
    if lengths.shape != (B,) or lengths.dtype not in (torch.int32, torch.int64) or lengths.device != device \
            or not lengths.is_contiguous():
        raise RuntimeError(f"delrec_b200: lengths must be contiguous int32 or int64 ({B},) on {device}")


def require_resets(resets, T, B, device):
    if resets is None:
        return None
    if resets.shape != (T, B) or resets.dtype != torch.bool or resets.device != device:
        raise RuntimeError(f"delrec_b200: resets must be bool ({T}, {B}) on {device}")
    return resets.contiguous()


def require_active(active, B, device):
    if active is None:
        return None
    if active.shape != (B,) or active.dtype != torch.bool or active.device != device:
        raise RuntimeError(f"delrec_b200: active must be bool ({B},) on {device}")
    return active.contiguous()


def refuse_tangents(*tensors):
    """Raises where a tensor carries a forward-mode tangent: the operators have no forward-mode
    derivative, and a call outside autograd would drop the tangent.  Called only where a
    dual level is open (``forward_ad._current_level``), which small calls test at next to no cost."""
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError("delrec_b200: the sequence operators have no forward-mode derivative")


def rows(t):
    """t with contiguous channels (the last dimension); a copy where they are strided."""
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def empty_rows(like, dtype=None):
    """An output shaped like ``like`` with contiguous channels: its layout where that is dense."""
    r = torch.empty_like(like) if dtype is None else torch.empty_like(like, dtype=dtype)
    return r if r.stride(-1) == 1 or r.shape[-1] <= 1 else torch.empty(r.shape, dtype=r.dtype, device=r.device)


def addr(t):
    return None if t is None else t.data_ptr()


def launch(what, device, *args):
    """Calls the C entry point ``what`` with args and the current stream of ``device``, which
    is made the current device where it is not."""
    index = device.index
    fn = getattr(_lib or lib(), what)
    stream = torch._C._cuda_getCurrentRawStream     # a torch built without CUDA has none
    if index == torch._C._cuda_getDevice():
        rc = fn(*args, stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, stream(index))
    if rc:
        check(rc, what)


def scratch(nbytes, device):
    """Scratch of one call, from torch's caching allocator (so that captured graphs and
    streams never share it); None for 0 bytes.  Its blocks are 512-byte aligned."""
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


_ws_cache: dict = {}


def workspace(nbytes: int, device) -> torch.Tensor:
    """A uint8 scratch tensor of at least ``nbytes`` (256-byte aligned) for ``device``,
    reused across calls on the current stream."""
    key = (torch.device(device).index, torch.cuda.current_stream(device).cuda_stream)
    buf = _ws_cache.get(key)
    need = max(int(nbytes), 256)
    if buf is None or buf.numel() < need:
        buf = torch.empty(need + 256, dtype=torch.uint8, device=device)
        _ws_cache[key] = buf
    off = (-buf.data_ptr()) % 256
    return buf[off:off + need]


def release_workspaces():
    _ws_cache.clear()


def lif_struct(tau, v_threshold, v_reset, detach_reset, surrogate_id, gamma, alpha) -> LIF:
    soft = v_reset is None
    return LIF(float(tau), float(v_threshold), 0.0 if soft else float(v_reset), int(soft),
               int(bool(detach_reset)), int(surrogate_id), float(gamma), float(alpha))


def launch_count() -> int:
    return int(lib().delrec_launch_count())


def scan_timing(enable: bool):
    check(lib().delrec_scan_timing(int(enable)), "delrec_scan_timing")


def scan_time(part=0):
    """(total milliseconds, launches) of the reverse-scan kernels timed since enabling:
    part 0 every scan, 1 the step launches of the chunked scans, 2 their chunk GEMMs."""
    ms = ctypes.c_double(0.0)
    n = ctypes.c_int(0)
    check(lib().delrec_scan_time_part(int(part), ctypes.byref(ms), ctypes.byref(n)), "delrec_scan_time_part")
    return ms.value, n.value


REVERSE_SCAN_CHUNKED, REVERSE_SCAN_STEPWISE, REVERSE_SCAN_CHUNKED_EXCHANGE = 0, 1, 2


def set_reverse_scan(variant: int):
    """Select the layer backwards' reverse scan for this process: REVERSE_SCAN_CHUNKED
    (default: hybrid layers contract their long-lag synapses once per 8-step chunk on the
    tensor cores) or REVERSE_SCAN_STEPWISE (the step-by-step scans only)."""
    check(lib().delrec_set_reverse_scan(int(variant)), "delrec_set_reverse_scan")


def exchange_floor_ms(T, B, N, K=0, repeats=3, device=None):
    """Milliseconds of the reverse scans' per-step exchange alone over T steps (the latency
    floor of one layer's scan) on the tiling used for a (T, B, N) layer; the median of
    ``repeats`` launches timed with CUDA events on the current stream."""
    import statistics
    layer = Layer(HYBRID, int(T), int(B), int(N), 2, int(K), 0, 0, 1.0, 0.0)
    nbytes = lib().delrec_exchange_floor_workspace(ctypes.byref(layer))
    if nbytes == 0:
        raise RuntimeError("delrec_b200: no exchange-floor tiling for this shape")
    ws = workspace(nbytes, device or torch.cuda.current_device())
    st = stream_ptr(device)
    times = []
    for _ in range(repeats + 1):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        check(lib().delrec_exchange_floor(ctypes.byref(layer), ptr(ws), nbytes, st), "delrec_exchange_floor")
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b))
    return statistics.median(times[1:])


def status() -> int:
    out = ctypes.c_int(0)
    check(lib().delrec_get_status(ctypes.byref(out)), "delrec_get_status")
    return out.value

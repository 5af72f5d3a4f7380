"""``_C`` -- the drop-in for the reference's compiled module ``kivi_sycl._C``.

Same twelve functions, keyword names, argument meaning and error behaviour as
the reference binding (src/csrc/bindings/pybind_module.cpp:9-82): the caller
allocates every output, the ops write in place, the blocking ops return
``None`` after the device work has finished and the ``*_async`` ops return a
:class:`KiviEvent`.  Validation follows src/csrc/ops/kv_cache_ops.cpp:19-171
message for message and raises ``RuntimeError`` (what ``TORCH_CHECK`` raises
in Python); the device check expects ROCm-torch's ``cuda`` device type where
the reference expected ``xpu`` (src/csrc/include/kivi/common.hpp:64-75).

Work is launched on ``torch.cuda.current_stream()`` of the tensors' device,
through the C ABI of ``libkivi_hip.so``; nothing here computes on the host.
"""

from __future__ import annotations

import ctypes
import functools
import threading

import torch
from torch.autograd import forward_ad

from . import _native
from ._device import device_index, is_current, on_device, stream_handle

_lib = _native.load()

__all__ = [
    "KiviEvent",
    "quantize_keys", "quantize_values", "dequantize_keys", "dequantize_values",
    "quant_dequant_roundtrip_keys", "quant_dequant_roundtrip_values",
    "quantize_keys_async", "quantize_values_async", "dequantize_keys_async",
    "dequantize_values_async", "quant_dequant_roundtrip_keys_async",
    "quant_dequant_roundtrip_values_async", "set_lazy_events",
]

_DEVICE_TYPE = "cuda"   # ROCm torch reports HIP devices as "cuda"

# torch::toString(ScalarType) spellings used in the reference's messages.
_DTYPE_NAMES = {
    torch.float32: "Float", torch.float64: "Double", torch.float16: "Half",
    torch.bfloat16: "BFloat16", torch.uint8: "Byte", torch.int8: "Char",
    torch.int16: "Short", torch.int32: "Int", torch.int64: "Long",
    torch.bool: "Bool",
}


def _dtype_name(dt) -> str:
    return _DTYPE_NAMES.get(dt, str(dt).replace("torch.", ""))


def _fail(*parts) -> None:
    raise RuntimeError("".join(str(p) for p in parts))


def _check(cond: bool, *parts) -> None:
    if not cond:
        _fail(*parts)


def _check_int(value, name: str) -> int:
    if isinstance(value, bool) or not isinstance(value, int):
        raise TypeError(f"{name} must be an int, got {type(value).__name__}")
    if not -(1 << 31) <= value < (1 << 31):
        raise TypeError(f"{name} does not fit in a C int: {value}")
    return value


def _check_tensor(t, name: str, dtype) -> None:
    """common.hpp:64-75: contiguous, exact dtype, device type."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    _check(t.is_contiguous(), name, " must be contiguous")
    _check(t.dtype == dtype, name, " must be ", _dtype_name(dtype), " but got ",
           _dtype_name(t.dtype))
    _check(t.device.type == _DEVICE_TYPE, name, " must be on ", _DEVICE_TYPE,
           " but got ", t.device.type)


def _check_same_device(*tensors) -> torch.device:
    dev = tensors[0].device
    for t in tensors[1:]:
        _check(t.device == dev, "all tensors must be on the same device, got ",
               dev, " and ", t.device)
    return dev


# --------------------------------------------------------------------------
# Validation: kv_cache_ops.cpp:19-171.  Each returns the count the kernel
# launch needs.
# --------------------------------------------------------------------------
def _validate_quant_keys(input, output, scales, zeros, group_size) -> int:
    _check_tensor(input, "input", torch.float32)
    _check_tensor(output, "output", torch.uint8)
    _check_tensor(scales, "scales", torch.float32)
    _check_tensor(zeros, "zeros", torch.float32)
    _check(group_size > 0 and group_size % 4 == 0,
           "group_size must be positive and divisible by 4, got ", group_size)
    n = scales.numel()
    _check(n > 0, "scales must be non-empty")
    _check(zeros.numel() == n, "zeros size (", zeros.numel(),
           ") must match scales size (", n, ")")
    _check(input.numel() == n * group_size, "input size (", input.numel(),
           ") must equal num_channels(", n, ") * group_size(", group_size, ") = ",
           n * group_size)
    _check(output.numel() == n * (group_size // 4), "output size (", output.numel(),
           ") must equal num_channels(", n, ") * (group_size/4) = ",
           n * (group_size // 4))
    return n


def _validate_quant_values(input, output, scales, zeros, head_dim, group_size) -> int:
    _check_tensor(input, "input", torch.float32)
    _check_tensor(output, "output", torch.uint8)
    _check_tensor(scales, "scales", torch.float32)
    _check_tensor(zeros, "zeros", torch.float32)
    _check(group_size > 0 and group_size % 4 == 0,
           "group_size must be positive and divisible by 4")
    _check(head_dim > 0 and head_dim % group_size == 0,
           "head_dim must be positive and divisible by group_size")
    _check(input.numel() % head_dim == 0, "input.numel() (", input.numel(),
           ") must be divisible by head_dim (", head_dim,
           ") — refusing to silently truncate trailing elements")
    n_tok = input.numel() // head_dim
    gpt = head_dim // group_size
    _check(n_tok > 0, "input must be non-empty")
    _check(scales.numel() == n_tok * gpt, "scales size (", scales.numel(),
           ") must equal num_tokens(", n_tok, ") * groups_per_token(", gpt, ")")
    _check(zeros.numel() == scales.numel(), "zeros size (", zeros.numel(),
           ") must match scales size (", scales.numel(), ")")
    _check(output.numel() == n_tok * (head_dim // 4), "output size (", output.numel(),
           ") must equal num_tokens(", n_tok, ") * (head_dim/4) = ",
           n_tok * (head_dim // 4))
    return n_tok


def _validate_dequant_keys(input, scales, zeros, output, group_size) -> int:
    _check_tensor(input, "input", torch.uint8)
    _check_tensor(scales, "scales", torch.float32)
    _check_tensor(zeros, "zeros", torch.float32)
    _check_tensor(output, "output", torch.float32)
    _check(group_size > 0 and group_size % 4 == 0,
           "group_size must be positive and divisible by 4, got ", group_size)
    n = scales.numel()
    _check(n > 0, "scales must be non-empty")
    _check(zeros.numel() == n, "zeros size (", zeros.numel(),
           ") must match scales size (", n, ")")
    _check(input.numel() == n * (group_size // 4), "input (packed) size (", input.numel(),
           ") must equal num_channels(", n, ") * (group_size/4) = ", n * (group_size // 4))
    _check(output.numel() == n * group_size, "output size (", output.numel(),
           ") must equal num_channels(", n, ") * group_size = ", n * group_size)
    return n


def _validate_dequant_values(input, scales, zeros, output, head_dim, group_size) -> int:
    _check_tensor(input, "input", torch.uint8)
    _check_tensor(scales, "scales", torch.float32)
    _check_tensor(zeros, "zeros", torch.float32)
    _check_tensor(output, "output", torch.float32)
    _check(group_size > 0 and group_size % 4 == 0,
           "group_size must be positive and divisible by 4, got ", group_size)
    _check(head_dim > 0 and head_dim % group_size == 0,
           "head_dim must be positive and divisible by group_size")
    n = scales.numel()
    _check(n > 0, "scales must be non-empty")
    _check(zeros.numel() == n, "zeros size (", zeros.numel(),
           ") must match scales size (", n, ")")
    _check(input.numel() == n * (group_size // 4), "input (packed) size (", input.numel(),
           ") must equal num_groups(", n, ") * (group_size/4) = ", n * (group_size // 4))
    _check(output.numel() == n * group_size, "output size (", output.numel(),
           ") must equal num_groups(", n, ") * group_size = ", n * group_size)
    return n


def _validate_roundtrip_keys(input, output, group_size) -> int:
    _check_tensor(input, "input", torch.float32)
    _check_tensor(output, "output", torch.float32)
    _check(group_size > 0 and group_size % 4 == 0,
           "group_size must be positive and divisible by 4, got ", group_size)
    _check(input.numel() % group_size == 0, "input.numel() (", input.numel(),
           ") must be divisible by group_size (", group_size, ")")
    _check(output.numel() == input.numel(), "output size (", output.numel(),
           ") must equal input size (", input.numel(),
           ") — round-trip is shape-preserving")
    n = input.numel() // group_size
    _check(n > 0, "input must be non-empty")
    return n


def _validate_roundtrip_values(input, output, head_dim, group_size) -> int:
    _check_tensor(input, "input", torch.float32)
    _check_tensor(output, "output", torch.float32)
    _check(group_size > 0 and group_size % 4 == 0,
           "group_size must be positive and divisible by 4")
    _check(head_dim > 0 and head_dim % group_size == 0,
           "head_dim must be positive and divisible by group_size")
    _check(input.numel() % head_dim == 0, "input.numel() (", input.numel(),
           ") must be divisible by head_dim (", head_dim, ")")
    _check(output.numel() == input.numel(), "output size (", output.numel(),
           ") must equal input size (", input.numel(),
           ") — round-trip is shape-preserving")
    n = input.numel() // head_dim
    _check(n > 0, "input must be non-empty")
    return n


# --------------------------------------------------------------------------
# Launch plumbing.
# --------------------------------------------------------------------------
def _stream_of(device: torch.device) -> int:
    return stream_handle(device)


def _ptr(t: torch.Tensor) -> int:
    return t.data_ptr()


class KiviEvent:
    """Handle for work submitted by a ``*_async`` op (event.hpp:16-31).

    ``wait()`` blocks until the work completes and raises ``RuntimeError`` on
    a device-side error; ``query()`` tells, without blocking, whether it has.
    As in the reference, where the event wraps the submitted kernel's own
    ``sycl::event`` (kv_cache_ops.cpp:245-303), the HIP event is the
    completion event of the op's own kernel launch (hipExtLaunchKernel), so
    ``wait()`` and ``query()`` cover that op alone, whatever is queued behind
    it later, and no marker sits between it and the next kernel.

    Lazy recording is opt-in (:func:`set_lazy_events`): the event is then
    recorded (as a marker) at the first ``wait()`` or ``query()``, which
    covers the op and any work queued on the same stream after it.  The op's
    tensors and its stream are kept alive until the event is released."""

    __slots__ = ("_device", "_stream", "_ev", "_keep", "_done")

    def __init__(self, device: torch.device, stream: "torch.cuda.Stream", keep=()):
        self._device = device
        self._stream = stream
        self._ev = None
        self._keep = keep
        self._done = False

    def _record(self) -> None:
        if self._ev is None:
            ev = ctypes.c_void_p()
            with torch.cuda.device(self._device):
                _native.check(_lib.kivi_event_record(ctypes.c_void_p(self._stream.cuda_stream),
                                                     ctypes.byref(ev)), "kivi_event_record")
            self._ev = ev

    def _release(self) -> None:
        ev, self._ev = self._ev, None
        if ev is not None:
            _lib.kivi_event_destroy(ev)
        self._keep = ()
        self._stream = None
        self._done = True

    def wait(self) -> None:
        if self._done:
            return
        self._record()
        try:
            _native.check(_lib.kivi_event_wait(self._ev), "KiviEvent.wait")
        finally:
            self._release()

    def query(self) -> bool:
        """True once the work has completed (non-blocking)."""
        if self._done:
            return True
        self._record()
        rc = _lib.kivi_event_query(self._ev)
        if rc < 0:
            _native.check(-rc, "KiviEvent.query")
        if rc == 1:
            self._release()
            return True
        return False

    def __del__(self):
        ev = getattr(self, "_ev", None)
        if ev is not None and _lib is not None:
            try:
                _lib.kivi_event_destroy(ev)
            except Exception:   # interpreter shutdown
                pass


def _run(device: torch.device, blocking: bool, what: str, fn, *args, keep=()):
    """Runs the C-ABI op ``fn`` on the device's current stream.  Blocking:
    synchronise the stream.  Async (per-op events): the op's ``_ev`` entry
    point, whose event is the completion event of the op's own kernel launch
    (no marker queued behind it).  Async with lazy events: the plain entry
    point, the event recorded at first use."""
    with torch.cuda.device(device):
        stream = torch.cuda.current_stream(device)
        sp = ctypes.c_void_p(stream.cuda_stream)
        if not blocking and not _lazy_events:
            handle = ctypes.c_void_p()
            _native.check(getattr(_lib, fn.__name__ + "_ev")(*args, sp, ctypes.byref(handle)),
                          what)
            ev = KiviEvent(device, stream, keep)
            ev._ev = handle
            return ev
        _native.check(fn(*args, sp), what)
        if blocking:
            _native.check(_lib.kivi_stream_synchronize(sp), what)
            return None
        return KiviEvent(device, stream, keep)


_lazy_events = False


def set_lazy_events(lazy: bool) -> bool:
    """Chooses the ``*_async`` ops' :class:`KiviEvent`: the completion event
    of the op's own kernel launch (the default, the reference's per-op
    semantics) or, with ``lazy=True``, a marker recorded at the event's first
    ``wait()``/``query()``.  Returns the previous setting.  Not part of the
    reference's API."""
    global _lazy_events
    prev, _lazy_events = _lazy_events, bool(lazy)
    return prev


# --------------------------------------------------------------------------
# The twelve ops (pybind_module.cpp:18-81).
# --------------------------------------------------------------------------
def _quantize_keys(input, output, scales, zeros, group_size, blocking):
    group_size = _check_int(group_size, "group_size")
    n = _validate_quant_keys(input, output, scales, zeros, group_size)
    dev = _check_same_device(input, output, scales, zeros)
    return _run(dev, blocking, "quantize_keys", _lib.kivi_quantize_keys_per_channel,
                _ptr(input), _ptr(output), _ptr(scales), _ptr(zeros), n, group_size,
                keep=(input, output, scales, zeros))


def _quantize_values(input, output, scales, zeros, head_dim, group_size, blocking):
    head_dim = _check_int(head_dim, "head_dim")
    group_size = _check_int(group_size, "group_size")
    n_tok = _validate_quant_values(input, output, scales, zeros, head_dim, group_size)
    dev = _check_same_device(input, output, scales, zeros)
    return _run(dev, blocking, "quantize_values", _lib.kivi_quantize_values_per_token,
                _ptr(input), _ptr(output), _ptr(scales), _ptr(zeros), n_tok, head_dim,
                group_size, keep=(input, output, scales, zeros))


def _dequantize_keys(input, scales, zeros, output, group_size, blocking):
    group_size = _check_int(group_size, "group_size")
    n = _validate_dequant_keys(input, scales, zeros, output, group_size)
    dev = _check_same_device(input, scales, zeros, output)
    return _run(dev, blocking, "dequantize_keys", _lib.kivi_dequantize_keys_per_channel,
                _ptr(input), _ptr(scales), _ptr(zeros), _ptr(output), n, group_size,
                keep=(input, scales, zeros, output))


def _dequantize_values(input, scales, zeros, output, head_dim, group_size, blocking):
    head_dim = _check_int(head_dim, "head_dim")
    group_size = _check_int(group_size, "group_size")
    n = _validate_dequant_values(input, scales, zeros, output, head_dim, group_size)
    dev = _check_same_device(input, scales, zeros, output)
    return _run(dev, blocking, "dequantize_values", _lib.kivi_dequantize_values_per_token,
                _ptr(input), _ptr(scales), _ptr(zeros), _ptr(output), n, group_size,
                keep=(input, scales, zeros, output))


def _roundtrip_keys(input, output, group_size, blocking):
    group_size = _check_int(group_size, "group_size")
    n = _validate_roundtrip_keys(input, output, group_size)
    dev = _check_same_device(input, output)
    return _run(dev, blocking, "quant_dequant_roundtrip_keys",
                _lib.kivi_quant_dequant_roundtrip_keys, _ptr(input), _ptr(output), n,
                group_size, keep=(input, output))


def _roundtrip_values(input, output, head_dim, group_size, blocking):
    head_dim = _check_int(head_dim, "head_dim")
    group_size = _check_int(group_size, "group_size")
    n_tok = _validate_roundtrip_values(input, output, head_dim, group_size)
    dev = _check_same_device(input, output)
    return _run(dev, blocking, "quant_dequant_roundtrip_values",
                _lib.kivi_quant_dequant_roundtrip_values, _ptr(input), _ptr(output),
                n_tok, head_dim, group_size, keep=(input, output))


def quantize_keys(input, output, scales, zeros, group_size):
    """Asymmetric 2-bit key quantization (per-channel)."""
    return _quantize_keys(input, output, scales, zeros, group_size, True)


def quantize_values(input, output, scales, zeros, head_dim, group_size):
    """Asymmetric 2-bit value quantization (per-token)."""
    return _quantize_values(input, output, scales, zeros, head_dim, group_size, True)


def dequantize_keys(input, scales, zeros, output, group_size):
    """Asymmetric 2-bit key dequantization (per-channel)."""
    return _dequantize_keys(input, scales, zeros, output, group_size, True)


def dequantize_values(input, scales, zeros, output, head_dim, group_size):
    """Asymmetric 2-bit value dequantization (per-token)."""
    return _dequantize_values(input, scales, zeros, output, head_dim, group_size, True)


def quant_dequant_roundtrip_keys(input, output, group_size):
    """Fused quantize->dequantize round-trip (per-channel); output is
    bit-identical to quantize_keys followed by dequantize_keys."""
    return _roundtrip_keys(input, output, group_size, True)


def quant_dequant_roundtrip_values(input, output, head_dim, group_size):
    """Fused quantize->dequantize round-trip (per-token)."""
    return _roundtrip_values(input, output, head_dim, group_size, True)


def quantize_keys_async(input, output, scales, zeros, group_size):
    """Non-blocking quantize_keys -- returns a KiviEvent, does not wait."""
    return _quantize_keys(input, output, scales, zeros, group_size, False)


def quantize_values_async(input, output, scales, zeros, head_dim, group_size):
    """Non-blocking quantize_values -- returns a KiviEvent, does not wait."""
    return _quantize_values(input, output, scales, zeros, head_dim, group_size, False)


def dequantize_keys_async(input, scales, zeros, output, group_size):
    """Non-blocking dequantize_keys -- returns a KiviEvent, does not wait."""
    return _dequantize_keys(input, scales, zeros, output, group_size, False)


def dequantize_values_async(input, scales, zeros, output, head_dim, group_size):
    """Non-blocking dequantize_values -- returns a KiviEvent, does not wait."""
    return _dequantize_values(input, scales, zeros, output, head_dim, group_size, False)


def quant_dequant_roundtrip_keys_async(input, output, group_size):
    """Non-blocking quant_dequant_roundtrip_keys -- returns a KiviEvent."""
    return _roundtrip_keys(input, output, group_size, False)


def quant_dequant_roundtrip_values_async(input, output, head_dim, group_size):
    """Non-blocking quant_dequant_roundtrip_values -- returns a KiviEvent."""
    return _roundtrip_values(input, output, head_dim, group_size, False)


# --------------------------------------------------------------------------
# Fused packed-KV decode attention (no reference counterpart; see
# include/kivi_hip.h).  Not part of the reference's twelve ops.
# --------------------------------------------------------------------------
_ws_cache = {}
_WS_KEPT = 16 << 20      # largest workspace kept per stream (a decode step's take a few MB)


def _workspace(device, nbytes: int):
    if nbytes == 0:
        return None
    if nbytes > _WS_KEPT:
        # (many query rows over several splits; torch's allocator reuses the
        # block in stream order)
        return torch.empty(nbytes, dtype=torch.uint8, device=device)
    key = (device_index(device), stream_handle(device))
    buf = _ws_cache.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
        _ws_cache[key] = buf
    return buf


def packed_decode_attention(q, store, softmax_scale=None, out=None, num_splits=0,
                            workspace=None):
    """o = softmax(q . [K_hat; K_res]^T * scale) . [V_hat; V_res] for one query
    token per sequence, straight from a :class:`PackedKVStore`.

    q: [B, Hq, D] or [B, Hq, 1, D] fp32 on the store's device.  Returns
    ``out`` ([B, Hq, D] fp32), launched on the current stream (asynchronous).

    A decode step makes this call once per layer, so the checks are ordered
    for the common case: one combined test each, the detailed messages only
    on failure."""
    if not (isinstance(q, torch.Tensor) and q.is_cuda and q.dtype is torch.float32
            and q.is_contiguous()):
        _check_tensor(q, "q", torch.float32)
    B, D = store.B, store.D
    shp = q.shape
    nd = len(shp)
    if not ((nd == 3 or (nd == 4 and shp[2] == 1)) and shp[0] == B and shp[-1] == D):
        _fail("q must be [B, Hq, D] or [B, Hq, 1, D] matching the store, got ", tuple(shp))
    Hq = shp[1]
    dev = q.get_device()
    _check(dev == device_index(store.device), "q must be on the store's device")
    if out is None:
        out = q.new_empty((B, Hq, D))
    else:
        _check_tensor(out, "out", torch.float32)
        _check(out.numel() == B * Hq * D, "out must hold B*Hq*D elements")
    scale = D ** -0.5 if softmax_scale is None else float(softmax_scale)
    need = store.workspace_bytes(Hq, num_splits)
    if workspace is None:
        workspace = _workspace(dev, need)
    elif need:
        _check(workspace.is_contiguous() and workspace.numel() * workspace.element_size() >= need,
               "workspace must be contiguous and hold ", need, " bytes")
    ws_bytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
    res_dt = store.res_dtype_code
    pend = getattr(store, "_pending", None)
    if pend is not None:
        # the staged token goes into the ring within this launch
        kn, vn = pend
        # (plain ints for the pointers: the entry points' argtypes convert them)
        with on_device(dev):
            _native.check(_lib.kivi_packed_decode_attention_append(
                q.data_ptr(), kn.data_ptr(), vn.data_ptr(), kn.stride(0), kn.stride(1),
                store.k_codes.data_ptr(), store.k_scale.data_ptr(), store.k_zero.data_ptr(),
                store.v_codes.data_ptr(), store.v_scale.data_ptr(), store.v_zero.data_ptr(),
                store.k_res.data_ptr(), store.v_res.data_ptr(), res_dt, out.data_ptr(),
                workspace.data_ptr() if workspace is not None else 0, ws_bytes,
                B, Hq, store.H, D, store.G, store.Gv, store.capacity, store.n_chunks, store.R,
                store.res_start, store.res_len, scale, int(num_splits),
                stream_handle(dev)), "packed_decode_attention")
        store._pending = None
        return out
    with on_device(dev):
        _native.check(_lib.kivi_packed_decode_attention(
            q.data_ptr(), store.k_codes.data_ptr(), store.k_scale.data_ptr(),
            store.k_zero.data_ptr(), store.v_codes.data_ptr(), store.v_scale.data_ptr(),
            store.v_zero.data_ptr(), store.k_res.data_ptr(), store.v_res.data_ptr(), res_dt,
            out.data_ptr(), workspace.data_ptr() if workspace is not None else 0, ws_bytes,
            B, Hq, store.H, D, store.G, store.Gv, store.capacity, store.n_chunks, store.R,
            store.res_start, store.res_len, scale, int(num_splits),
            stream_handle(dev)), "packed_decode_attention")
    return out


def hidden_positions(key_mask, device=None):
    """The hidden-position words of kivi_packed_attention_masked from a
    key-padding mask ``[B, T]`` (HF's 2-D ``attention_mask`` convention:
    nonzero / True = the position is attended): ``[B, ceil(T / 32)]`` int32,
    bit ``p % 32`` of word ``p // 32`` of row b set when position p of
    sequence b is hidden.  Computed on ``device`` (default: the mask's)."""
    _check(torch.is_tensor(key_mask) and key_mask.dim() == 2,
           "key_mask must be a [B, T] tensor")
    dev = key_mask.device if device is None else torch.device(device)
    vis = key_mask.to(dev) != 0
    B, T = vis.shape
    W = (T + 31) // 32
    bits = torch.zeros(B, W * 32, dtype=torch.int64, device=dev)
    bits[:, :T] = (~vis).to(torch.int64)
    words = (bits.view(B, W, 32) << torch.arange(32, device=dev)).sum(-1)    # < 2^32
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


def packed_attention(q, store, causal=True, softmax_scale=None, out=None, num_splits=0,
                     workspace=None, kv_start=None, key_mask=None, hidden=None):
    """Attention of ``L`` query tokens per sequence over a
    :class:`PackedKVStore`, ``q [B, Hq, L, D]`` fp32 (the layout HF attention
    functions receive); returns ``[B, L, Hq, D]`` fp32 (the layout they
    return).  ``causal``: the L queries are the residual window's last L
    tokens and token i attends to the cache up to itself (a multi-token
    forward on a non-empty cache); otherwise every query sees the whole
    context (one query token sees it either way).  ``kv_start`` (B ints, a
    list or an int32 tensor): sequence b's first visible context position,
    for a left-padded batch; positions before it take no weight.  Checked
    against the context length when given on the host.  ``key_mask``
    ``[B, T]`` over the whole context (T = quantised + window tokens; nonzero
    = attended, HF's 2-D padding mask), or ``hidden`` (its words,
    :func:`hidden_positions`, computed once for many calls): any other
    padding pattern (right padding, holes), hidden from every query token;
    a query row that sees no position gets zeros.  Launched on the current
    stream."""
    _check(q.dtype == torch.float32, "q must be float32, got ", _dtype_name(q.dtype))
    _check(q.dim() == 4 and q.shape[0] == store.B and q.shape[3] == store.D,
           "q must be [B, Hq, L, D] matching the store, got ", tuple(q.shape))
    _check(q.device == store.device, "q must be on the store's device")
    B, Hq, L, D = q.shape
    store._commit()
    if causal and L > 1:
        _check(L <= store.res_len, "causal attention of ", L, " query tokens needs them in "
               "the residual window (", store.res_len, " tokens)")
    ks_ptr = 0
    if kv_start is not None:
        if not (torch.is_tensor(kv_start) and kv_start.device == q.device):
            starts = [int(x) for x in (kv_start.tolist() if torch.is_tensor(kv_start)
                                       else kv_start)]
            T = store.quantized_tokens + store.res_len
            last = T - L if causal else T - 1
            _check(len(starts) == B and all(0 <= x <= last for x in starts),
                   "kv_start must hold ", B, " positions in [0, ", last, "], got ", starts)
            kv_start = torch.tensor(starts, dtype=torch.int32).to(q.device)
        _check(kv_start.dtype == torch.int32 and kv_start.numel() == B and
               kv_start.is_contiguous(), "kv_start must be a contiguous int32 tensor of ", B,
               " positions")
        ks_ptr = kv_start.data_ptr()
    if key_mask is not None:
        _check(hidden is None, "pass key_mask or hidden, not both")
        T = store.quantized_tokens + store.res_len
        _check(tuple(key_mask.shape) == (B, T), "key_mask must be [B=", B, ", T=", T,
               "] over the whole context, got ", tuple(key_mask.shape))
        hidden = hidden_positions(key_mask, q.device)
    if hidden is not None:
        W = (store.quantized_tokens + store.res_len + 31) // 32
        _check(hidden.dtype == torch.int32 and hidden.dim() == 2 and hidden.shape[0] == B and
               hidden.shape[1] >= W and hidden.stride(1) == 1 and hidden.device == q.device,
               "hidden must be an int32 [B, >=", W, "] tensor with contiguous rows on the "
               "query's device")
    qk = q.transpose(1, 2).contiguous()                                  # [B, L, Hq, D]
    if out is None:
        out = torch.empty(B, L, Hq, D, dtype=torch.float32, device=q.device)
    else:
        _check_tensor(out, "out", torch.float32)
        _check(out.numel() == B * L * Hq * D, "out must hold B*L*Hq*D elements")
    scale = D ** -0.5 if softmax_scale is None else float(softmax_scale)
    need = int(_lib.kivi_packed_attention_workspace_size(
        B, L, Hq, store.H, D, store.G, store.Gv, store.n_chunks, store.res_len, num_splits))
    if workspace is None:
        workspace = _workspace(q.device, need)
    elif need:
        _check(workspace.is_contiguous() and workspace.numel() * workspace.element_size() >= need,
               "workspace must be contiguous and hold ", need, " bytes")
    ws_bytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
    if hidden is not None:
        entry = functools.partial(_lib.kivi_packed_attention_masked,
                                  ctypes.c_void_p(qk.data_ptr()), L, 1 if causal else 0,
                                  ctypes.c_void_p(ks_ptr), ctypes.c_void_p(hidden.data_ptr()),
                                  hidden.stride(0))
    else:
        entry = functools.partial(_lib.kivi_packed_attention, ctypes.c_void_p(qk.data_ptr()),
                                  L, 1 if causal else 0, ctypes.c_void_p(ks_ptr))
    with on_device(q.device):
        _native.check(entry(
            ctypes.c_void_p(store.k_codes.data_ptr()),
            ctypes.c_void_p(store.k_scale.data_ptr()), ctypes.c_void_p(store.k_zero.data_ptr()),
            ctypes.c_void_p(store.v_codes.data_ptr()), ctypes.c_void_p(store.v_scale.data_ptr()),
            ctypes.c_void_p(store.v_zero.data_ptr()), ctypes.c_void_p(store.k_res.data_ptr()),
            ctypes.c_void_p(store.v_res.data_ptr()), store.res_dtype_code,
            ctypes.c_void_p(out.data_ptr()),
            ctypes.c_void_p(workspace.data_ptr() if workspace is not None else 0), ws_bytes,
            B, Hq, store.H, D, store.G, store.Gv, store.capacity, store.n_chunks, store.R,
            store.res_start, store.res_len, scale, int(num_splits),
            ctypes.c_void_p(_stream_of(q.device))), "packed_attention")
    return out


_IO_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def takes_typed_queries(q, store):
    """Whether :func:`packed_attention_typed` takes these queries: more than 8
    query rows per kv head of several tokens on a matrix-core store, on the
    store's device, channels contiguous and aligned for 4-element loads."""
    return (q.dim() == 4 and q.shape[2] > 1 and q.dtype in _IO_DTYPES and q.is_cuda
            and store.code_layout != 0 and q.device == store.device
            and q.shape[0] == store.B and q.shape[3] == store.D and q.numel() > 0
            and q.shape[1] % store.H == 0 and q.shape[2] * (q.shape[1] // store.H) > 8
            and q.stride(3) == 1 and q.data_ptr() % 16 == 0
            and not any(s % 4 for s in q.stride()[:3]))


def packed_attention_typed(q, store, softmax_scale=None, kv_start=None, hidden=None):
    """:func:`packed_attention` (causal) of queries ``q [B, Hq, L, D]`` in the
    model's own type and strides, returning ``[B, L, Hq, D]`` of that type: the
    bits of the fp32 call on converted tensors, without the conversions.  Only
    where :func:`takes_typed_queries`.  ``kv_start`` and ``hidden``: tensors on
    the store's device."""
    _check(takes_typed_queries(q, store), "these queries need packed_attention")
    B, Hq, L, D = q.shape
    store._commit()
    _check(L <= store.res_len, "causal attention of ", L, " query tokens needs them in "
           "the residual window (", store.res_len, " tokens)")
    if kv_start is not None:
        _check(kv_start.dtype == torch.int32 and kv_start.numel() == B and
               kv_start.is_contiguous() and kv_start.device == q.device,
               "kv_start must be a contiguous int32 tensor of ", B, " positions")
    if hidden is not None:
        W = (store.quantized_tokens + store.res_len + 31) // 32
        _check(hidden.dtype == torch.int32 and hidden.dim() == 2 and hidden.shape[0] == B and
               hidden.shape[1] >= W and hidden.stride(1) == 1 and hidden.device == q.device,
               "hidden must be an int32 [B, >=", W, "] tensor with contiguous rows on the "
               "query's device")
    out = torch.empty(B, L, Hq, D, dtype=q.dtype, device=q.device)
    need = int(_lib.kivi_packed_attention_workspace_size(
        B, L, Hq, store.H, D, store.G, store.Gv, store.n_chunks, store.res_len, 0))
    ws = _workspace(q.device, need)
    with on_device(q.device):
        _native.check(_lib.kivi_packed_attention_typed(
            q.data_ptr(), _IO_DTYPES[q.dtype], q.stride(0), q.stride(2), q.stride(1), L, 1,
            0 if kv_start is None else kv_start.data_ptr(),
            0 if hidden is None else hidden.data_ptr(),
            0 if hidden is None else hidden.stride(0),
            store.k_codes.data_ptr(), store.k_scale.data_ptr(), store.k_zero.data_ptr(),
            store.v_codes.data_ptr(), store.v_scale.data_ptr(), store.v_zero.data_ptr(),
            store.k_res.data_ptr(), store.v_res.data_ptr(), store.res_dtype_code, out.data_ptr(),
            0 if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel(),
            B, Hq, store.H, D, store.G, store.Gv, store.capacity, store.n_chunks, store.R,
            store.res_start, store.res_len,
            D ** -0.5 if softmax_scale is None else float(softmax_scale), 0,
            _stream_of(q.device)), "packed_attention")
    return out


# --------------------------------------------------------------------------
# Paged cache (no reference counterpart; see include/kivi_hip.h): sequences of
# unequal lengths on pages of one pool.
# --------------------------------------------------------------------------
def _check_inference(*tensors) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                _fail("inference only: a tensor requires a gradient; call it under "
                      "torch.no_grad()")
    if forward_ad._current_level >= 0:                   # (inside a dual_level())
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                _fail("inference only: a tensor has a forward-mode tangent")


def _host_ints(values, name: str) -> torch.Tensor:
    """Counts as a contiguous int32 host tensor."""
    t = torch.as_tensor(values)
    if t.numel() == 0:
        t = t.to(torch.int64)
    _check(t.dim() == 1 and t.device.type == "cpu" and t.dtype in (torch.int32, torch.int64),
           name, " must hold one int for each sequence, on the host")
    if t.dtype is torch.int64:
        _check(t.numel() == 0 or (int(t.min()) >= 0 and int(t.max()) < 1 << 31), name,
               " must lie in [0, 2^31)")
        t = t.to(torch.int32)
    return t.contiguous()


class PagedPlan:
    """One step over a paged cache (:func:`paged_plan`): which sequences bring
    how many new tokens, and where these lie, as one device array that every
    layer's :func:`paged_append` and :func:`paged_attention` read.  It belongs to
    pools of ``num_pages`` pages and to the geometry it was made for."""

    __slots__ = ("device", "tokens", "context", "num_pages", "page_size", "q_heads", "kv_heads",
                 "head_dim", "dtype", "cache_dtype", "_code", "_index", "_pool", "_scales", "_buf",
                 "_ptr", "_info",
                 "_info_ptr", "_workspace", "_stream", "_event", "_settled")

    def wait(self) -> None:
        """Waits until the plan is on the device.  Needed only before a graph is
        captured with it (which reads the plan's memory at every replay: keep the
        plan as long as the graph); other calls order themselves behind its copy."""
        self._event.synchronize()
        self._settled = True

    def _enter(self, device: int) -> int:
        """The current stream's handle, ordered behind the plan's copy."""
        handle = stream_handle(device)
        if not self._settled:
            # (before a capture on the plan's own stream too: a replay may come on another)
            _check(not torch.cuda.is_current_stream_capturing(),
                   "call the plan's wait() before capturing a graph with it")
            self._settled = self._event.query()
        if handle != self._stream and not torch.cuda.is_current_stream_capturing():
            stream = torch.cuda.current_stream(device)
            if not self._settled:
                stream.wait_event(self._event)
            # (its memory is not given away while this stream may read it)
            self._buf.record_stream(stream)
        return handle


_PLAN_ITEMS = 1 << 13        # int32s of a plan's items that a first buffer has room for


def paged_plan(page_table, context_lens, new_lens, *, page_size, num_pages, q_heads, kv_heads,
               head_dim, dtype=torch.bfloat16, device="cuda", cache_dtype=None) -> PagedPlan:
    """The plan of a step in which sequence s, ``context_lens[s]`` tokens long
    with them, brings its last ``new_lens[s]`` tokens (0: it sits this step out).
    ``page_table`` (int32 host tensor ``[sequences, pages]``): its pages, position
    p on entry ``p // page_size``; entries behind its last position are not read.
    Tokens are numbered sequence by sequence.  ``cache_dtype``: the pages' type,
    ``dtype`` or int8 (no block of 16 positions may then get new tokens of two
    sequences).  Host work and one copy to ``device``, once per step for all
    layers."""
    _check(isinstance(page_table, torch.Tensor) and page_table.dim() == 2
           and page_table.dtype is torch.int32 and page_table.device.type == "cpu",
           "page_table must be an int32 [sequences, pages] tensor on the host")
    _check(dtype in _IO_DTYPES, "dtype must be float32, bfloat16 or float16, got ",
           _dtype_name(dtype))
    eight = cache_dtype is torch.int8
    _check(eight or cache_dtype is None or cache_dtype is dtype, "cache_dtype must be ",
           _dtype_name(dtype), " or int8, got ", _dtype_name(cache_dtype))
    make = _lib.kivi_paged8_plan if eight else _lib.kivi_paged_plan
    dev = torch.device(device)
    _check(dev.type == _DEVICE_TYPE, "device must be on ", _DEVICE_TYPE, " but got ", dev.type)
    page_size, q_heads, kv_heads, head_dim = (
        _check_int(x, n) for x, n in ((page_size, "page_size"), (q_heads, "q_heads"),
                                      (kv_heads, "kv_heads"), (head_dim, "head_dim")))
    num_pages = _check_int(num_pages, "num_pages")
    table = page_table.contiguous()
    ctx, new = _host_ints(context_lens, "context_lens"), _host_ints(new_lens, "new_lens")
    n_seqs = table.shape[0]
    _check(ctx.numel() == n_seqs and new.numel() == n_seqs,
           "context_lens and new_lens must hold one entry for each of the table's ", n_seqs,
           " sequences")
    p = PagedPlan()
    info = (ctypes.c_int64 * 20)()
    p._info, p._info_ptr = info, ctypes.addressof(info)
    args = (n_seqs, new.data_ptr(), ctx.data_ptr(), table.data_ptr(), table.shape[1],
            table.shape[1], page_size, num_pages, _IO_DTYPES[dtype], q_heads, kv_heads, head_dim)
    # (one call where a buffer of the usual size will do; on a host that has not used
    # its GPU yet the arguments are checked first)
    host = None
    if torch.cuda.is_initialized():
        _check(not torch.cuda.is_current_stream_capturing(),
               "a plan is made outside of a graph's capture")
        host = torch.empty(table.numel() + 2 * min(max(int(new.sum()), 0), 1 << 20) + _PLAN_ITEMS,
                           dtype=torch.int32, pin_memory=True)
    rc = make(*args, None if host is None else host.data_ptr(),
              0 if host is None else host.numel(), p._info_ptr)
    if rc and (host is None or info[0] <= host.numel()):
        _native.check(rc, "paged_plan")
    p.device = torch.device(_DEVICE_TYPE, device_index(dev))
    p.tokens, p.context = info[1], info[12]
    p.num_pages, p.page_size, p.dtype, p._code = num_pages, page_size, dtype, _IO_DTYPES[dtype]
    p.q_heads, p.kv_heads, p.head_dim = q_heads, kv_heads, head_dim
    p._index = p.device.index
    p._pool = torch.Size((num_pages, kv_heads, page_size, head_dim))
    p.cache_dtype = torch.int8 if eight else dtype
    p._scales = torch.Size((num_pages, kv_heads, page_size // 16)) if eight else None
    if host is None or info[0] > host.numel():
        host = torch.empty(max(info[0], 1), dtype=torch.int32, pin_memory=True)
        _native.check(make(*args, host.data_ptr(), host.numel(), p._info_ptr), "paged_plan")
    with on_device(p.device):
        p._buf = host[:max(info[0], 1)].to(p.device, non_blocking=True)
        p._event = torch.cuda.Event()
        p._event.record()
        p._stream = stream_handle(p.device)
    p._settled = False
    p._ptr = p._buf.data_ptr()
    p._workspace = int(_lib.kivi_paged_attention_workspace_size(p._info_ptr, kv_heads, head_dim))
    return p


# The calls below are made once per layer of a step, so their checks are ordered
# for the common case: one combined test each, the detailed messages (or the less
# common ways to be right) only where it fails.
def _check_pages(plan, k_pages, v_pages):
    kp, vp = k_pages.data_ptr(), v_pages.data_ptr()
    pool, dt, dev = plan._pool, plan.cache_dtype, plan._index
    if not (k_pages.shape == pool and v_pages.shape == pool and k_pages.dtype is dt
            and v_pages.dtype is dt and k_pages.is_contiguous() and v_pages.is_contiguous()
            and k_pages.get_device() == dev and v_pages.get_device() == dev
            and not (kp | vp) & 15):
        for t, name in ((k_pages, "k_pages"), (v_pages, "v_pages")):
            _check(t.shape == pool and t.dtype is dt and t.is_contiguous()
                   and t.get_device() == dev and not t.data_ptr() & 15,
                   name, " must be a contiguous, 16-byte aligned ", list(pool), " tensor of ",
                   _dtype_name(dt), " on ", plan.device, ", got ", list(t.shape), " of ",
                   _dtype_name(t.dtype), " on ", t.device)
    return kp, vp


def _check_scales(plan, k_scales, v_scales):
    """The scales of pages of 8 bits (none for others): their addresses."""
    shape, dev = plan._scales, plan._index
    if shape is None:
        _check(k_scales is None and v_scales is None,
               "k_scales and v_scales belong to pages of int8, the plan is for ",
               _dtype_name(plan.dtype))
        return 0, 0
    _check(k_scales is not None and v_scales is not None,
           "pages of int8 need k_scales and v_scales")
    if not (k_scales.shape == shape and v_scales.shape == shape
            and k_scales.dtype is torch.float32 and v_scales.dtype is torch.float32
            and k_scales.is_contiguous() and v_scales.is_contiguous()
            and k_scales.get_device() == dev and v_scales.get_device() == dev):
        for t, name in ((k_scales, "k_scales"), (v_scales, "v_scales")):
            _check(t.shape == shape and t.dtype is torch.float32 and t.is_contiguous()
                   and t.get_device() == dev, name, " must be a contiguous ", list(shape),
                   " tensor of Float on ", plan.device, ", got ", list(t.shape), " of ",
                   _dtype_name(t.dtype), " on ", t.device)
    return k_scales.data_ptr(), v_scales.data_ptr()


def _check_tokens(t, name: str, plan, heads: int):
    """A step's rows ``[>= tokens, heads, head_dim]``, any strides of whole rows;
    the strides."""
    sh, st = t.shape, t.stride()
    if not (len(sh) == 3 and sh[0] >= plan.tokens and sh[1] == heads and sh[2] == plan.head_dim
            and st[2] == 1 and t.dtype is plan.dtype and t.get_device() == plan._index):
        _check(len(sh) == 3 and sh[0] >= plan.tokens and sh[1] == heads
               and sh[2] == plan.head_dim and t.dtype is plan.dtype and t.device == plan.device,
               name, " must be [>= ", plan.tokens, ", ", heads, ", ", plan.head_dim, "] of ",
               _dtype_name(plan.dtype), " on ", plan.device, ", got ", list(sh), " of ",
               _dtype_name(t.dtype), " on ", t.device)
        _fail(name, "'s channels must be contiguous")
    return st


def _new_rows(t, plan):
    """An output beside a step's rows ``t``; rows behind the step's tokens, which
    no kernel writes, are zeros."""
    if t.shape[0] > plan.tokens:
        return torch.zeros(t.shape, dtype=t.dtype, device=t.device)
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _check_out(out, name: str, like) -> None:
    _check(out.shape == like.shape and out.dtype is like.dtype and out.device == like.device
           and out.is_contiguous() and out.data_ptr() % 16 == 0, name,
           " must be a contiguous, 16-byte aligned ", list(like.shape), " tensor of ",
           _dtype_name(like.dtype), " on ", like.device)


def paged_append(k, v, k_pages, v_pages, plan, q=None, q_out=None, cos=None, sin=None,
                 interleaved=False, q_norm=None, k_norm=None, eps=1e-6, k_scales=None,
                 v_scales=None):
    """Write a step's new keys and values ``[tokens, Hkv, D]`` to their pages,
    normed and rotated on the way, and return its queries ``q`` ``[tokens, Hq, D]``
    normed and rotated likewise (None without ``q``): one launch.

    ``q_norm``, ``k_norm`` ``[D]``: weights of an RMS norm over each head's
    channels (``eps`` inside the root).  ``cos``, ``sin`` ``[positions, r / 2]``
    fp32 (:func:`rotary_tables`): the first r channels are rotated by the angles of
    the token's position in its sequence, channel i with i + r/2, or 2i with 2i + 1
    if ``interleaved``.  Both in fp32, rounded once.  Values are copied.  Rows may
    have any strides, as slices of one projection have; rows behind the plan's
    tokens are not read, and stay as they are in ``q_out``, which may be ``q``.

    Pages of int8 (a plan with ``cache_dtype=torch.int8``) have ``k_scales`` and
    ``v_scales`` ``[num_pages, Hkv, page_size / 16]`` fp32 beside them, one for each
    block of 16 positions of a page and head: the least power of two from 2^-126 on
    whose 127-fold reaches every value appended to the block since its first position
    was (tokens taken back among them); an element is code * scale, its code the
    quotient rounded to nearest even.  A block's older codes are rounded again
    where new tokens need a larger scale.  What a block's first position finds there
    is not read.  A value that is not finite makes its block's scale NaN."""
    dev = plan._index
    if not is_current(dev):
        with on_device(dev):
            return paged_append(k, v, k_pages, v_pages, plan, q, q_out, cos, sin, interleaved,
                                q_norm, k_norm, eps, k_scales, v_scales)
    _check_inference(k, v, k_pages, v_pages, q, q_out, cos, sin, q_norm, k_norm, k_scales,
                     v_scales)
    kp, vp = _check_pages(plan, k_pages, v_pages)
    _check(kp != vp or plan.tokens == 0, "k_pages and v_pages must be two pools")
    ksp, vsp = _check_scales(plan, k_scales, v_scales)
    _check(ksp != vsp or not ksp or plan.tokens == 0, "k_scales and v_scales must be two tensors")
    ks = _check_tokens(k, "k", plan, plan.kv_heads)
    vs = _check_tokens(v, "v", plan, plan.kv_heads)
    rot = cos_ptr = sin_ptr = 0
    if cos is not None or sin is not None:
        _check(cos is not None and sin is not None, "rotation needs cos and sin")
        sh = cos.shape
        cos_ptr, sin_ptr = cos.data_ptr(), sin.data_ptr()
        _check(len(sh) == 2 and sin.shape == sh and cos.dtype is torch.float32
               and sin.dtype is torch.float32 and cos.is_contiguous() and sin.is_contiguous()
               and cos.get_device() == dev and sin.get_device() == dev
               and not (cos_ptr | sin_ptr) & 15,
               "cos and sin must be contiguous, 16-byte aligned [positions, rotated / 2] float32 "
               "tensors on ", plan.device)
        _check(sh[0] >= plan.context, "cos and sin reach ", sh[0],
               " positions, the step's longest sequence has ", plan.context)
        rot = 2 * sh[1]
    norm_dt = None
    if q_norm is not None or k_norm is not None:
        for t, name in ((q_norm, "q_norm"), (k_norm, "k_norm")):
            if t is None:
                continue
            if not (t.shape == (plan.head_dim,) and t.dtype in _IO_DTYPES and t.is_contiguous()
                    and t.get_device() == dev):
                _fail(name, " must be a contiguous [", plan.head_dim,
                      "] tensor of a float type on ", plan.device)
            _check(norm_dt is None or norm_dt is t.dtype, "q_norm and k_norm must have one type")
            norm_dt = t.dtype
    q_ptr = q_st = q_sh = out_ptr = 0
    if q is not None:
        st = _check_tokens(q, "q", plan, plan.q_heads)
        if q_out is None:
            q_out = _new_rows(q, plan)
        else:
            _check_out(q_out, "q_out", q)
        q_ptr, q_st, q_sh, out_ptr = q.data_ptr(), st[0], st[1], q_out.data_ptr()
    else:
        _check(q_out is None and q_norm is None, "q_out and q_norm need q")
    rows = (q_ptr, q_st, q_sh, k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1],
            plan._code, out_ptr, kp, vp)
    geometry = (plan.num_pages, plan.page_size, plan.q_heads, plan.kv_heads, plan.head_dim,
                plan._ptr)
    way = (cos_ptr, sin_ptr, rot, 1 if interleaved else 0,
           0 if q_norm is None else q_norm.data_ptr(), 0 if k_norm is None else k_norm.data_ptr(),
           0 if norm_dt is None else _IO_DTYPES[norm_dt], eps, plan._enter(dev))
    if ksp:
        rc = _lib.kivi_paged8_append(*rows, ksp, vsp, *geometry, plan._info_ptr, *way)
    else:
        rc = _lib.kivi_paged_append(*rows, *geometry, plan.tokens, *way)
    if rc:
        _native.check(rc, "paged_append")
    return q_out


def rotary_tables(positions, rotary_dim, base=10000.0, inv_freq=None, device="cuda"):
    """cos and sin ``[positions, rotary_dim / 2]`` fp32 of position x frequency,
    the angles formed in fp64.  Frequencies: ``inv_freq`` (a model's own, scaled
    as it scales them), else ``base ** (-2 i / rotary_dim)``."""
    _check(rotary_dim > 0 and rotary_dim % 16 == 0,
           "rotary_dim must be a positive multiple of 16, got ", rotary_dim)
    if inv_freq is None:
        inv_freq = base ** (-torch.arange(rotary_dim // 2, dtype=torch.float64)
                            / (rotary_dim // 2))
    f = inv_freq.detach().to("cpu", torch.float64)
    _check(f.dim() == 1 and f.shape[0] == rotary_dim // 2, "inv_freq must hold ",
           rotary_dim // 2, " frequencies, got ", list(f.shape))
    ang = torch.arange(positions, dtype=torch.float64)[:, None] * f[None, :]
    return ang.cos().float().to(device), ang.sin().float().to(device)


_call_ws = threading.local()


def _call_workspace(device: int, nbytes: int):
    """Device memory for one call: kept for the next of the same host thread and
    stream (two threads' launches on one stream may alternate).  A call that is
    captured has memory of its own: two graphs may run at once."""
    if nbytes == 0:
        return None
    if nbytes > _WS_KEPT or torch.cuda.is_current_stream_capturing():
        return torch.empty(nbytes, dtype=torch.uint8, device=torch.device(_DEVICE_TYPE, device))
    kept, key = _call_ws.__dict__, (device, stream_handle(device))
    buf = kept.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = kept[key] = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8,
                                      device=torch.device(_DEVICE_TYPE, device))
    return buf


def paged_attention(q, k_pages, v_pages, plan, softmax_scale=None, out=None, workspace=None,
                    k_scales=None, v_scales=None):
    """Attention of a step's new tokens ``q [tokens, Hq, D]`` over their
    sequences' pages, their own keys and values included (:func:`paged_append`
    first): token i of n new ones in a context of c sees positions 0 .. c - n + i.
    Returns ``[tokens, Hq, D]`` in q's type.  Chunks of prompts, verification
    passes and single tokens may share a call.  Rows behind the plan's tokens are
    not read, and stay as they are in ``out``.  ``k_scales``, ``v_scales``: the scales
    of pages of int8, as :func:`paged_append` leaves them.  Launched on the current
    stream."""
    dev = plan._index
    if not is_current(dev):
        with on_device(dev):
            return paged_attention(q, k_pages, v_pages, plan, softmax_scale, out, workspace,
                                   k_scales, v_scales)
    _check_inference(q, k_pages, v_pages, out, k_scales, v_scales)
    kp, vp = _check_pages(plan, k_pages, v_pages)
    ksp, vsp = _check_scales(plan, k_scales, v_scales)
    st = _check_tokens(q, "q", plan, plan.q_heads)
    q_ptr = q.data_ptr()
    if q_ptr & 15 or (st[0] | st[1]) * q.element_size() & 15:
        q = q.clone(memory_format=torch.contiguous_format)
        q_ptr, st = q.data_ptr(), q.stride()
    if out is None:
        out = _new_rows(q, plan)
    else:
        _check_out(out, "out", q)
    need = plan._workspace
    ws_ptr = ws_bytes = 0
    if need and workspace is None:
        workspace = _call_workspace(dev, need)         # (held until both launches are made)
        ws_ptr, ws_bytes = workspace.data_ptr(), need
    elif need:
        ws_ptr, ws_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
        _check(workspace.is_contiguous() and workspace.get_device() == dev
               and not ws_ptr & 15 and ws_bytes >= need,
               "workspace must be a contiguous, 16-byte aligned tensor of ", need,
               " bytes on ", plan.device)
    geometry = (plan.num_pages, plan.page_size, plan.q_heads, plan.kv_heads, plan.head_dim,
                plan._ptr, plan._info_ptr,
                plan.head_dim ** -0.5 if softmax_scale is None else float(softmax_scale),
                out.data_ptr(), ws_ptr, ws_bytes, plan._enter(dev))
    if ksp:
        rc = _lib.kivi_paged8_attention(q_ptr, st[0], st[1], plan._code, kp, vp, ksp, vsp,
                                        *geometry)
    else:
        rc = _lib.kivi_paged_attention(q_ptr, st[0], st[1], plan._code, kp, vp, *geometry)
    if rc:
        _native.check(rc, "paged_attention")
    return out


# --------------------------------------------------------------------------
# Sampling (sampling.py:10-25 in the reference, with top-p, min-p and given
# random numbers; see include/kivi_hip.h).
# --------------------------------------------------------------------------
def _setting(value, name: str, rows: int, dtype, dev):
    """A setting as (pointer of a per-row tensor or 0, scalar)."""
    if isinstance(value, torch.Tensor):
        _check(value.dtype is dtype and value.dim() == 1 and value.shape[0] == rows
               and value.is_contiguous() and value.device == dev, name,
               " must be a number or a contiguous [", rows, "] tensor of ", _dtype_name(dtype),
               " on ", dev)
        return value.data_ptr(), 0
    return 0, value


def allowed_tokens(mask):
    """The words that :func:`adjust_logits` takes from a mask ``[rows, vocab]`` (nonzero
    or True: the token is allowed): ``[rows, ceil(vocab / 32)]`` int32, bit ``v % 32``
    of word ``v // 32`` for token v."""
    return ~hidden_positions(mask)


def _row_list(t, name: str, rows: int, dtypes, dev):
    """A list for each row, ``[rows, n]``, or one for all, ``[n]``: rows any distance
    apart.  Its stride."""
    if isinstance(t, torch.Tensor) and t.dtype in dtypes and t.get_device() == dev:
        sh, st = t.shape, t.stride()
        if len(sh) == 2 and sh[0] == rows and (st[1] == 1 or sh[1] <= 1):
            return st[0]
        if len(sh) == 1 and (st[0] == 1 or sh[0] <= 1):
            return 0
    _fail(name, " must be a [", rows, ", n] or [n] tensor of ",
          " or ".join(_dtype_name(d) for d in dtypes), " with contiguous rows on ", _DEVICE_TYPE,
          ":", dev)


def _row_setting(value, name: str, rows: int, dtype, dev):
    """:func:`_setting` of a device's index."""
    if isinstance(value, torch.Tensor):
        if not (value.dtype is dtype and value.shape == (rows,) and value.is_contiguous()
                and value.get_device() == dev):
            _fail(name, " must be a number or a contiguous [", rows, "] tensor of ",
                  _dtype_name(dtype), " on ", _DEVICE_TYPE, ":", dev)
        return value.data_ptr(), 0
    return 0, value


_ID_DTYPES = (torch.int32, torch.int64)


def adjust_logits(logits, tokens=None, lengths=None, prompt_lengths=0, repetition_penalty=1.0,
                  presence_penalty=0.0, frequency_penalty=0.0, bias_ids=None, bias=None,
                  allowed=None, out=None):
    """``logits [rows, vocab]`` (fp32, bf16 or fp16) changed before :func:`sample`:
    penalties for repeated tokens, then biases, then a mask, each where it is given, in
    fp32 with one rounding at the end; launched on the current stream.

    ``tokens [rows, n]`` (int32 or int64): each row's tokens so far, of which the first
    ``lengths`` count (None: all), and of these the first ``prompt_lengths`` are its
    prompt; ids outside the vocabulary are passed over.  A logit x of a token among them
    becomes x / repetition_penalty above 0 and x * repetition_penalty otherwise; of one
    that is k > 0 times behind the prompt, x - (frequency_penalty * k +
    presence_penalty).  ``bias_ids`` (int32 or int64) and ``bias`` (fp32), ``[rows, n]``
    or ``[n]`` for all rows: x plus the sum, in the list's order, of the biases that are
    listed for the token.  ``allowed`` (int32, ``[rows, words]`` or ``[words]``,
    :func:`allowed_tokens`): logits of tokens whose bit is 0 become -infinity.

    Penalties and lengths are numbers or tensors with one value per row (float32;
    lengths int32).  ``out``: where the result goes, ``logits`` itself, or another tensor
    of its type or fp32 (None: a new one of its type).  A logit that nothing concerns
    keeps its bits."""
    if not (isinstance(logits, torch.Tensor) and logits.dim() == 2
            and logits.dtype in _IO_DTYPES and logits.is_cuda):
        _fail("logits must be a [rows, vocab] tensor of a float type on ", _DEVICE_TYPE)
    rows, vocab = logits.shape
    _check(vocab > 0, "a row must have logits")
    stride = logits.stride()
    _check(stride[1] == 1 or vocab == 1, "a row's logits must be contiguous")
    dev = logits.get_device()
    if not is_current(dev):
        with on_device(dev):
            return adjust_logits(logits, tokens, lengths, prompt_lengths, repetition_penalty,
                                 presence_penalty, frequency_penalty, bias_ids, bias, allowed,
                                 out)
    _check_inference(logits, bias, out)
    tok = length = 0, 0, 0, 0
    rp, r = _row_setting(repetition_penalty, "repetition_penalty", rows, torch.float32, dev)
    sp, s = _row_setting(presence_penalty, "presence_penalty", rows, torch.float32, dev)
    fp, f = _row_setting(frequency_penalty, "frequency_penalty", rows, torch.float32, dev)
    if rp or sp or fp:
        _check_inference(*(x for x in (repetition_penalty, presence_penalty, frequency_penalty)
                           if isinstance(x, torch.Tensor)))
    if not (rp or r > 0.0):
        _fail("repetition_penalty must be positive, got ", r)
    if tokens is not None:
        if not (isinstance(tokens, torch.Tensor) and len(tokens.shape) == 2):
            _fail("tokens must be a [", rows, ", n] tensor")
        st, n = _row_list(tokens, "tokens", rows, _ID_DTYPES, dev), tokens.shape[1]
        tok = tokens.data_ptr(), 1 if tokens.dtype is torch.int64 else 0, st, n
        lp, length = _row_setting(n if lengths is None else lengths, "lengths", rows, torch.int32,
                                  dev)
        pp, prompt = _row_setting(prompt_lengths, "prompt_lengths", rows, torch.int32, dev)
        length, prompt = _check_int(length, "lengths"), _check_int(prompt, "prompt_lengths")
        if not 0 <= length <= n:
            _fail("lengths must lie in [0, ", n, "], got ", length)
        if prompt < 0:
            _fail("prompt_lengths must not be negative, got ", prompt)
        length = lp, length, pp, prompt
    elif rp or sp or fp or r != 1.0 or s != 0.0 or f != 0.0 or lengths is not None:
        _fail("penalties need tokens")
    ids = 0, 0, 0, 0, 0, 0
    if bias_ids is not None or bias is not None:
        _check(bias_ids is not None and bias is not None, "biases need bias_ids and bias")
        ist = _row_list(bias_ids, "bias_ids", rows, _ID_DTYPES, dev)
        bst, n = _row_list(bias, "bias", rows, (torch.float32,), dev), bias.shape[-1]
        if bias_ids.shape[-1] != n:
            _fail("bias_ids name ", bias_ids.shape[-1], " tokens, bias has ", n, " values")
        ids = (bias_ids.data_ptr(), 1 if bias_ids.dtype is torch.int64 else 0, ist,
               bias.data_ptr(), bst, n)
    words = 0, 0
    if allowed is not None:
        st = _row_list(allowed, "allowed", rows, (torch.int32,), dev)
        if allowed.shape[-1] * 32 < vocab:
            _fail("allowed has ", allowed.shape[-1], " words for ", vocab, " tokens")
        words = allowed.data_ptr(), st
    code = _IO_DTYPES[logits.dtype]
    if out is None:
        out = logits.new_empty((rows, vocab))
        out_code, out_stride = code, vocab
    else:
        out_stride = out.stride(0) if len(out.shape) == 2 else 0
        if not (out.dtype in (logits.dtype, torch.float32) and out.shape == logits.shape
                and (out.stride(1) == 1 or vocab == 1) and out.get_device() == dev):
            _fail("out must be a [", rows, ", ", vocab, "] tensor of ", _dtype_name(logits.dtype),
                  " or Float with contiguous rows on ", logits.device)
        out_code = _IO_DTYPES[out.dtype]
    rc = _lib.kivi_adjust_logits(
        logits.data_ptr(), code, stride[0], rows, vocab, *tok, *length, rp, r, sp, s, fp, f, *ids,
        *words, out.data_ptr(), out_code, out_stride, stream_handle(dev))
    if rc:
        _native.check(rc, "adjust_logits")
    return out


def sample(logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, out=None):
    """Next tokens ``[rows]`` (int64) from ``logits [rows, vocab]`` (fp32, bf16 or
    fp16) and ``uniforms [rows]`` in [0, 1) (fp32 or fp64), launched on the current
    stream.

    In the order (logit descending, index ascending) with weights
    ``exp((x - max) / temperature)``: the first ``top_k`` tokens (0: all), of these
    the shortest prefix with ``top_p`` of their mass (1: all), of these the ones of
    weight ``min_p`` or more (0: all), the first one always; the result is the
    first whose running mass exceeds ``u`` times the kept mass.  ``temperature``
    0: the largest logit.  Each setting is a number or a tensor with one value per
    row (float32; top_k int32).  NaN logits are never taken; a row without any
    logit above -infinity gives -1."""
    if not (isinstance(logits, torch.Tensor) and logits.dim() == 2
            and logits.dtype in _IO_DTYPES and logits.is_cuda):
        _fail("logits must be a [rows, vocab] tensor of a float type on ", _DEVICE_TYPE)
    _check(logits.stride(1) == 1 or logits.shape[1] == 1, "a row's logits must be contiguous")
    rows, vocab = logits.shape
    dev = logits.device
    _check(isinstance(uniforms, torch.Tensor)
           and uniforms.dtype in (torch.float32, torch.float64) and uniforms.dim() == 1
           and uniforms.shape[0] == rows and uniforms.is_contiguous() and uniforms.device == dev,
           "uniforms must be a contiguous [", rows, "] float32 or float64 tensor on ", dev)
    tp, t = _setting(temperature, "temperature", rows, torch.float32, dev)
    kp, k = _setting(top_k, "top_k", rows, torch.int32, dev)
    pp, p = _setting(top_p, "top_p", rows, torch.float32, dev)
    mp, m = _setting(min_p, "min_p", rows, torch.float32, dev)
    _check(t >= 0.0, "temperature must not be negative, got ", t)
    _check(p >= 0.0, "top_p must not be negative, got ", p)
    _check(0.0 <= m <= 1.0, "min_p must lie in [0, 1], got ", m)
    k = min(_check_int(k, "top_k"), vocab)
    _check(k >= 0, "top_k must not be negative, got ", k)
    if out is None:
        out = torch.empty(rows, dtype=torch.int64, device=dev)
    else:
        _check(out.dtype is torch.int64 and out.shape == (rows,) and out.is_contiguous()
               and out.device == dev, "out must be a contiguous [", rows, "] int64 tensor on ",
               dev)
    index = dev.index
    with on_device(index):
        need = _lib.kivi_sample_workspace_size(rows, vocab)
        workspace = _call_workspace(index, need)
        _native.check(_lib.kivi_sample(
            logits.data_ptr(), _IO_DTYPES[logits.dtype], logits.stride(0), rows, vocab,
            uniforms.data_ptr(), 1 if uniforms.dtype is torch.float64 else 0, tp, t, kp, k, pp, p,
            mp, m, out.data_ptr(), 0 if workspace is None else workspace.data_ptr(), need,
            stream_handle(index)), "sample")
    return out

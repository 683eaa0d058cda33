"""oco_amd: MI355X (gfx950) quantized-weight matrix path of oco.

The product is the native library ``liboco_hip.so`` (HIP kernels behind the C
ABI in ``include/oco_hip.h``).  This package loads it with ctypes and mirrors
the reference's operator seam so callers and tests read like oco's own:

- ``WeightFormat`` / ``block_layout``   -> src/tensor.rs:9-38
- ``DeviceBuffer``                      -> src/gpu/buffer.rs (ReadOnly / BufferView)
- ``DenseMatrix`` (apply_row / apply)   -> src/weights/operands.rs:4-9, compute/matrix.rs:63,130
- ``Output``                            -> compute/matrix.rs:519-548 (f32 logits)
- ``ExpertBank`` / ``Router``           -> operands.rs ExpertWeight/Router, feed_forward.rs:107
- ``PagedCache`` / ``CacheBatch``       -> keys and values in 4-bit pages, and the attention over them

There is no CPU fallback: every compute call goes through the HIP library,
and loading fails loudly when the library is missing.
"""
from __future__ import annotations

import ctypes
import enum
import os

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "liboco_hip.so")


class WeightFormat(enum.IntEnum):
    """GGUF format codes (src/tensor.rs:9-20)."""
    F32 = 0
    F16 = 1
    Q4_0 = 2
    Q4_1 = 3
    Q8_0 = 8
    Q4K = 12
    Q5K = 13
    Q6K = 14
    Bf16 = 30
    Mxfp4 = 39


class Knob(enum.IntEnum):
    """oco_knob: kernel-choice overrides (tests and tuning runs)."""
    STREAM_PLAN = 0
    MATVEC_PLAN = 1
    MATVEC_PLAIN = 2
    MX_TILE = 3
    MX_PREFILL_OFF = 4
    MATMUL_TILE = 5
    MOE_MX_TOKENS = 6
    MOE_MFMA_TOKENS = 7
    MOE_Q4_ROWS = 8
    MOE_WG = 9
    MX_EXPERTS_KS = 10
    STREAM_DIRECT = 11
    MATMUL_VENDOR = 12
    FP8 = 13
    ATTENTION = 14


class DType(enum.IntEnum):
    F32 = 0
    BF16 = 1
    F16 = 2


class Activation(enum.IntEnum):
    SWIGLU_CLIPPED = 0
    SWIGLU = 1


class Gate(enum.IntEnum):
    """oco_gate."""
    NONE = 0
    LINEAR = 1
    SIGMOID = 2
    TANH = 3


class Score(enum.IntEnum):
    """oco_score."""
    SOFTMAX = 0
    SIGMOID = 1


class GroupRank(enum.IntEnum):
    """oco_group_rank."""
    MAX = 0
    TOP2 = 1


class DraftValues(enum.IntEnum):
    """oco_draft_values."""
    LOGITS = 0
    PROBABILITIES = 1


class RotationLayout(enum.IntEnum):
    """oco_rotation_layout."""
    HALF = 0
    INTERLEAVED = 1


class Scaling(enum.IntEnum):
    """oco_scaling."""
    NONE = 0
    LINEAR = 1
    YARN = 2
    BANDS = 3


NO_TOKEN = 0xFFFFFFFF  # oco_draft_verify's places without a token

_BLOCKS = {0: (1, 4), 1: (1, 2), 30: (1, 2), 2: (32, 18), 3: (32, 20), 8: (32, 34),
           12: (256, 144), 13: (256, 176), 14: (256, 210), 39: (32, 17)}


def block_layout(fmt: int) -> tuple[int, int]:
    """(elements, bytes) per block (src/tensor.rs:24-38)."""
    return _BLOCKS[int(fmt)]


def row_bytes(fmt: int, k: int) -> int:
    e, b = block_layout(fmt)
    if k % e:
        raise ValueError(f"k={k} is not a multiple of the {WeightFormat(fmt).name} block ({e})")
    return k // e * b


class OcoError(RuntimeError):
    """Raised for a non-zero status from the C ABI (src/error.rs:9-27)."""

    def __init__(self, code: int, message: str):
        super().__init__(f"[{code}] {message}")
        self.code = code


class Matrix(ctypes.Structure):
    """oco_matrix / Matrix (weights.metal:87-89)."""
    _fields_ = [(n, ctypes.c_uint32) for n in
                ("k", "n", "m", "route_major", "routes", "experts", "has_bias")]


def as_matrix(p) -> Matrix:
    """Accept any object with the Matrix fields (e.g. a struct from another module)."""
    if isinstance(p, Matrix):
        return p
    return Matrix(*[int(getattr(p, f)) for f, _ in Matrix._fields_])


class ExpertsDesc(ctypes.Structure):
    """oco_experts."""
    _fields_ = [("format", ctypes.c_uint32), ("hidden", ctypes.c_uint32), ("ffn", ctypes.c_uint32),
                ("experts", ctypes.c_uint32), ("k", ctypes.c_uint32),
                ("activation", ctypes.c_uint32), ("up_bias_one", ctypes.c_uint32),
                ("gate", ctypes.c_void_p), ("up", ctypes.c_void_p), ("down", ctypes.c_void_p),
                ("gate_bias", ctypes.c_void_p), ("up_bias", ctypes.c_void_p),
                ("down_bias", ctypes.c_void_p)]


class Block(ctypes.Structure):
    """oco_block: the step between two blocks of a layer."""
    _fields_ = ([(n, ctypes.c_uint32) for n in ("rows", "n", "x_dtype", "dtype", "gate", "gate_rows", "x_stride",
                                                "y_stride", "gate_stride", "out_stride")] +
                [(n, ctypes.c_float) for n in ("scale", "epsilon", "weight_offset")])


class Routing(ctypes.Structure):
    """oco_routing: how experts are chosen from their scores."""
    _fields_ = [(n, ctypes.c_uint32) for n in ("experts", "k", "score", "groups", "groups_kept", "group_rank",
                                               "renormalize")] + [("scale", ctypes.c_float)]


class Draft(ctypes.Structure):
    """oco_draft: the rows of a verification of drafted tokens."""
    _fields_ = ([(n, ctypes.c_uint32) for n in ("sequences", "drafts", "vocabulary", "target_values", "draft_values",
                                                "target_dtype", "draft_dtype")] +
                [("temperature", ctypes.c_float), ("target_stride", ctypes.c_uint64), ("draft_stride", ctypes.c_uint64)])


class Rotation(ctypes.Structure):
    """oco_rotation: how the pairs of a head turn; frequencies: address of f64 [dim / 2] on the device."""
    _fields_ = [("dim", ctypes.c_uint32), ("layout", ctypes.c_uint32), ("magnitude", ctypes.c_double),
                ("frequencies", ctypes.c_void_p)]


class Frequencies(ctypes.Structure):
    """oco_frequencies."""
    _fields_ = ([(n, ctypes.c_uint32) for n in ("dim", "scaling")] +
                [(n, ctypes.c_double) for n in ("base", "factor", "original", "fast", "slow")] + [("factors", ctypes.c_void_p)])


class Cache(ctypes.Structure):
    """oco_cache: a pool of pages in 4 bits and a batch of rows on it."""
    _fields_ = ([(n, ctypes.c_uint32) for n in ("head_dim", "heads", "kv_heads", "page_size", "pages", "sequences", "rows",
                                                "max_rows", "max_length", "table_stride", "dtype", "window")] +
                [("scale", ctypes.c_float)] +
                [(n, ctypes.c_uint64) for n in ("q_stride", "k_stride", "v_stride", "out_stride")])


class Logits(ctypes.Structure):
    """oco_logits: rows of logits that are adjusted before a token is chosen."""
    _fields_ = ([(n, ctypes.c_uint32) for n in ("rows", "vocabulary", "dtype", "history_stride", "bias_stride", "mask_stride",
                                                "group", "mask_group")] +
                [("stride", ctypes.c_uint64), ("out_stride", ctypes.c_uint64)])


class GgufEntry(ctypes.Structure):
    """oco_gguf_entry (Entry, gguf.rs:24-33)."""
    _fields_ = [("shape", ctypes.c_uint64 * 4), ("rank", ctypes.c_uint32), ("code", ctypes.c_uint32),
                ("offset", ctypes.c_uint64), ("extent", ctypes.c_uint64)]


class GgufTensor(ctypes.Structure):
    """oco_gguf_tensor (Tensor, gguf.rs:17-22)."""
    _fields_ = [("format", ctypes.c_uint32), ("rank", ctypes.c_uint32), ("shape", ctypes.c_uint64 * 4),
                ("offset", ctypes.c_uint64), ("bytes", ctypes.c_uint64)]


# Every symbol include/oco_hip.h declares, with its ctypes signature.
_vp, _u32, _u64, _i32, _sz = ctypes.c_void_p, ctypes.c_uint32, ctypes.c_uint64, ctypes.c_int, ctypes.c_size_t
_MP = ctypes.POINTER(Matrix)
_EP = ctypes.POINTER(ExpertsDesc)
SIGNATURES = {
    "oco_last_error": (ctypes.c_char_p, []),
    "oco_plan_override": (_i32, [_u32, ctypes.POINTER(ctypes.c_int32), _u32]),
    "oco_block_layout": (_i32, [_u32, ctypes.POINTER(_u32), ctypes.POINTER(_u32)]),
    "oco_row_bytes": (_u64, [_u32, _u32]),
    "oco_device_open": (_i32, [_i32, ctypes.POINTER(_i32)]),
    "oco_buffer_alloc": (_i32, [_sz, ctypes.POINTER(_vp)]),
    "oco_buffer_free": (_i32, [_vp]),
    "oco_buffer_upload": (_i32, [_vp, _vp, _sz]),
    "oco_buffer_download": (_i32, [_vp, _vp, _sz]),
    "oco_buffer_copy": (_i32, [_vp, _vp, _sz, _vp]),
    "oco_buffer_fill32": (_i32, [_vp, _u32, _sz, _vp]),
    "oco_buffer_xor32": (_i32, [_vp, _sz, _vp, _vp]),
    "oco_buffer_xor32_geometry": (_i32, [_u64, ctypes.POINTER(_u64), ctypes.POINTER(_u64)]),
    "oco_stream_create": (_i32, [ctypes.POINTER(_vp)]),
    "oco_stream_sync": (_i32, [_vp]),
    "oco_stream_destroy": (_i32, [_vp]),
    "oco_event_create": (_i32, [ctypes.POINTER(_vp)]),
    "oco_event_record": (_i32, [_vp, _vp]),
    "oco_event_elapsed_ms": (_i32, [_vp, _vp, ctypes.POINTER(ctypes.c_float)]),
    "oco_event_destroy": (_i32, [_vp]),
    "oco_graph_begin": (_i32, [_vp]),
    "oco_graph_end": (_i32, [_vp, ctypes.POINTER(_vp)]),
    "oco_graph_launch": (_i32, [_vp, _vp]),
    "oco_graph_destroy": (_i32, [_vp]),
    "oco_dequant": (_i32, [_u32, _vp, _u64, _vp, _vp]),
    "oco_embed": (_i32, [_u32, _vp, _u32, _u32, _vp, _u32, _vp, _u32, _vp, _vp]),
    "oco_matvec": (_i32, [_u32, _vp, _vp, _i32, _vp, _i32, _vp, _vp, _MP, _vp]),
    "oco_matvec_relu_sqr": (_i32, [_u32, _vp, _vp, _i32, _vp, _i32, _vp, _vp, _MP, _vp]),
    "oco_matmul": (_i32, [_u32, _vp, _vp, _i32, _vp, _i32, _vp, _MP, _vp]),
    "oco_matmul_workspace": (_u64, [_u32, _i32, _MP]),
    "oco_matmul_route": (_i32, [_u32, _i32, _i32, _MP, _u64, ctypes.POINTER(_u32)]),
    "oco_matmul_ws": (_i32, [_u32, _vp, _vp, _i32, _vp, _i32, _vp, _MP, _vp, _u64, _vp]),
    "oco_norm_mx_split": (_i32, [_vp, _vp, _vp, _u32, _u32, ctypes.c_float, _i32, _vp, _u64, _vp]),
    "oco_add_norm_mx_split": (_i32, [_vp, _vp, _vp, _vp, _u32, _u32, ctypes.c_float, _i32, _vp, _u64, _vp]),
    "oco_matmul_mx_split": (_i32, [_vp, _vp, _u64, _vp, _i32, _vp, _MP, _vp]),
    "oco_fp8_quantize": (_i32, [_vp, _i32, _u32, _u32, _u64, _vp, _vp, _vp]),
    "oco_fp8_matmul_workspace": (_u64, [_MP]),
    "oco_fp8_matmul": (_i32, [_vp, _vp, _vp, _vp, _vp, _i32, _vp, _MP, _vp, _u64, _vp]),
    "oco_route_scores": (_i32, [_vp, _i32, _vp, _u32, ctypes.POINTER(Routing), _vp, _vp, _vp]),
    "oco_block_norm": (_i32, [_vp] * 9 + [ctypes.POINTER(Block), _vp]),
    "oco_draft_verify_workspace": (_u64, [ctypes.POINTER(Draft)]),
    "oco_draft_verify": (_i32, [_vp] * 8 + [ctypes.POINTER(Draft), _vp, _u64, _vp]),
    "oco_rotation_frequencies": (_i32, [ctypes.POINTER(Frequencies), _vp, _vp]),
    "oco_rotate": (_i32, [_vp, _i32, _u32, _u32, _u32, _u64, _vp, _vp, _u64, ctypes.POINTER(Rotation), _vp]),
    "oco_cache_page_bytes": (_u64, [ctypes.POINTER(Cache)]),
    "oco_cache_append": (_i32, [_vp] * 9 + [ctypes.POINTER(Rotation), ctypes.POINTER(Cache), _vp]),
    "oco_cache_read": (_i32, [_vp] * 6 + [ctypes.POINTER(Cache), _vp]),
    "oco_cache_attention_workspace": (_u64, [ctypes.POINTER(Cache)]),
    "oco_cache_attention": (_i32, [_vp] * 7 + [ctypes.POINTER(Cache), _vp, _u64, _vp]),
    "oco_logits_adjust": (_i32, [_vp] * 9 + [ctypes.POINTER(Logits), _vp]),
    "oco_route_select": (_i32, [_vp, _u32, _u32, _u32, _vp, _vp, _vp]),
    "oco_router": (_i32, [_vp, _i32, _vp, _vp, _u32, _u32, _u32, _u32, _vp, _vp, _vp, _vp]),
    "oco_route_plan_words": (_u64, [_u32, _u32]),
    "oco_route_plan": (_i32, [_vp, _u32, _u32, _u32, _u32, _u32, _vp, _vp]),
    "oco_experts_workspace": (_u64, [_EP, _u32]),
    "oco_experts_apply": (_i32, [_EP, _vp, _i32, _vp, _vp, _u32, _vp, _vp, _vp, _u64, _vp]),
    "oco_experts_forward": (_i32, [_EP, _vp, _vp, _vp, _i32, _u32, _vp, _vp, _vp, _vp, _vp, _u64, _vp]),
    "oco_experts_forward_static": (_i32, [_EP, _vp, _vp, _vp, _i32, _u32, _vp, _vp, _vp, _vp, _vp]),
    "oco_expert_expand": (_i32, [_EP, _vp, _i32, _vp, _vp, _vp, _vp, _vp, _vp]),
    "oco_moe_sum": (_i32, [_vp, _i32, _vp, _vp, _u32, _u32, _u32, _vp]),
    "oco_norm": (_i32, [_vp, _vp, _vp, _u32, _u32, ctypes.c_float, _i32, _vp]),
    "oco_add_norm": (_i32, [_vp, _vp, _vp, _vp, _u32, _u32, ctypes.c_float, _i32, _vp]),
    "oco_matvec_norm": (_i32, [_u32, _vp, _vp, _vp, ctypes.c_float, _i32, _vp, _i32, _vp, _vp, _MP, _vp]),
    "oco_matvec_group": (_i32, [_u32, _u32, _vp, _vp, _i32, _vp, ctypes.c_float, _i32, _vp, _i32, _vp, _MP, _vp]),
    "oco_argmax_f32": (_i32, [_vp, _u32, _vp, _vp]),
    "oco_argmax_workspace": (_u64, [_u32]),
    "oco_argmax_f32_ws": (_i32, [_vp, _u32, _vp, _vp, _u64, _vp]),
    "oco_gguf_open": (_i32, [ctypes.c_char_p, ctypes.POINTER(ctypes.c_char_p), _u32, ctypes.POINTER(_vp)]),
    "oco_gguf_close": (_i32, [_vp]),
    "oco_gguf_has": (_i32, [_vp, ctypes.c_char_p]),
    "oco_gguf_text": (_i32, [_vp, ctypes.c_char_p, ctypes.POINTER(_vp), ctypes.POINTER(_sz)]),
    "oco_gguf_number": (_i32, [_vp, ctypes.c_char_p, ctypes.POINTER(ctypes.c_double)]),
    "oco_gguf_boolean": (_i32, [_vp, ctypes.c_char_p, ctypes.POINTER(_i32)]),
    "oco_gguf_unsigned": (_i32, [_vp, ctypes.c_char_p, ctypes.POINTER(_u64)]),
    "oco_gguf_array": (_i32, [_vp, ctypes.c_char_p, ctypes.POINTER(_u32), ctypes.POINTER(_u64)]),
    "oco_gguf_array_string": (_i32, [_vp, ctypes.c_char_p, _u64, ctypes.POINTER(_vp), ctypes.POINTER(_sz)]),
    "oco_gguf_array_unsigned": (_i32, [_vp, ctypes.c_char_p, _vp, _u64]),
    "oco_gguf_directory": (_i32, [_vp, ctypes.POINTER(_u64)]),
    "oco_gguf_entry_at": (_i32, [_vp, _u64, ctypes.POINTER(ctypes.c_char_p), ctypes.POINTER(GgufEntry)]),
    "oco_gguf_find": (_i32, [_vp, ctypes.c_char_p, ctypes.POINTER(GgufEntry)]),
    "oco_gguf_select": (_i32, [ctypes.POINTER(GgufEntry), ctypes.POINTER(GgufTensor)]),
    "oco_gguf_data": (_vp, [_vp, ctypes.POINTER(GgufTensor)]),
    "oco_gguf_upload": (_i32, [_vp, ctypes.POINTER(GgufTensor), _vp, _vp]),
}

_lib = None


def load_library(path: str = LIB_PATH):
    """Load liboco_hip.so and bind every declared symbol (fails loudly if absent)."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(path):
        raise OSError(f"{path} is missing: run __graft_entry__.build() (hipcc for gfx950) first")
    L = ctypes.CDLL(path)
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(L, name, None)
        if fn is None:  # tests/test_abi.py asserts every declared symbol is exported
            continue
        fn.restype = res
        fn.argtypes = args
    _lib = L
    return L


def _check(rc: int) -> None:
    if rc != 0:
        raise OcoError(rc, load_library().oco_last_error().decode())


_device_open = False


def open_device(ordinal: int = 0) -> int:
    """Gpu::new (src/gpu.rs:41-50): select the device, return its CU count."""
    global _device_open
    cu = ctypes.c_int()
    _check(load_library().oco_device_open(ordinal, ctypes.byref(cu)))
    _device_open = True
    return cu.value


def _ensure_device():
    if not _device_open:
        open_device(0)


def plan_override(knob: int, values=()):
    """Override one kernel-choice table entry (empty `values` clears it)."""
    vals = (ctypes.c_int32 * max(len(values), 1))(*[int(v) for v in values])
    _check(load_library().oco_plan_override(int(knob), vals, len(values)))


class overridden:
    """Context manager: `with overridden(Knob.X, (a, b)):` ... then cleared."""

    def __init__(self, knob: int, values):
        self.knob, self.values = knob, tuple(values)

    def __enter__(self):
        plan_override(self.knob, self.values)
        return self

    def __exit__(self, *a):
        plan_override(self.knob, ())


class Scratch:
    """Device memory that the calls on one stream take in turn.  A buffer that
    is too small gets a successor of at least twice its size and stays, as a
    captured call may use it: together under four times the largest need."""

    def __init__(self):
        self.buffers = []

    def at_least(self, nbytes: int) -> "DeviceBuffer":
        last = self.buffers[-1].nbytes if self.buffers else 0
        if last < nbytes:
            self.buffers.append(DeviceBuffer(max(nbytes, 2 * last)))
        return self.buffers[-1]


class Stream:
    """One HIP stream (the reference's per-session queue, compute.rs:36-55)."""

    def __init__(self):
        _ensure_device()
        h = ctypes.c_void_p()
        _check(load_library().oco_stream_create(ctypes.byref(h)))
        self.handle = h
        self.scratch = Scratch()  # lives as long as the object, which its graphs hold

    def sync(self):
        _check(load_library().oco_stream_sync(self.handle))

    def close(self):
        if self.handle:
            _check(load_library().oco_stream_destroy(self.handle))
            self.handle = None


class Event:
    def __init__(self):
        h = ctypes.c_void_p()
        _check(load_library().oco_event_create(ctypes.byref(h)))
        self.handle = h

    def record(self, stream=None):
        _check(load_library().oco_event_record(self.handle, _stream(stream)))

    def elapsed_ms(self, end: "Event") -> float:
        ms = ctypes.c_float()
        _check(load_library().oco_event_elapsed_ms(self.handle, end.handle, ctypes.byref(ms)))
        return ms.value

    def __del__(self):
        try:
            if self.handle and _lib is not None:
                _lib.oco_event_destroy(self.handle)
        except Exception:
            pass


class Graph:
    """Captured launches replayed natively (stream capture into a HIP graph)."""

    def __init__(self, stream: "Stream", record):
        _check(load_library().oco_graph_begin(stream.handle))
        try:
            record()
        finally:
            h = ctypes.c_void_p()
            rc = load_library().oco_graph_end(stream.handle, ctypes.byref(h))
        _check(rc)
        self.handle = h
        self.stream = stream

    def launch(self):
        _check(load_library().oco_graph_launch(self.handle, self.stream.handle))

    def __del__(self):
        try:
            if self.handle and _lib is not None:
                _lib.oco_graph_destroy(self.handle)
        except Exception:
            pass


def _stream(s):
    if s is None:
        return None
    return s.handle if isinstance(s, Stream) else s


class DeviceBuffer:
    """Device allocation (src/gpu/buffer.rs BufferView / ReadOnly)."""

    def __init__(self, nbytes: int):
        _ensure_device()
        p = ctypes.c_void_p()
        _check(load_library().oco_buffer_alloc(max(int(nbytes), 1), ctypes.byref(p)))
        self.ptr = p.value
        self.nbytes = int(nbytes)

    @classmethod
    def from_array(cls, a: np.ndarray) -> "DeviceBuffer":
        a = np.ascontiguousarray(a)
        b = cls(a.nbytes)
        b.upload(a)
        return b

    def upload(self, a: np.ndarray, offset: int = 0):
        a = np.ascontiguousarray(a)
        if offset + a.nbytes > self.nbytes:
            raise ValueError("upload past the end of the buffer")
        _check(load_library().oco_buffer_upload(self.ptr + offset, a.ctypes.data, a.nbytes))

    def download(self, dtype, count=None, offset: int = 0) -> np.ndarray:
        dtype = np.dtype(dtype)
        if count is None:
            count = (self.nbytes - offset) // dtype.itemsize
        out = np.empty(count, dtype)
        if offset + out.nbytes > self.nbytes:
            raise ValueError("download past the end of the buffer")
        _check(load_library().oco_buffer_download(out.ctypes.data, self.ptr + offset, out.nbytes))
        return out

    def fill32(self, pattern: int, stream=None):
        _check(load_library().oco_buffer_fill32(self.ptr, pattern & 0xFFFFFFFF, self.nbytes // 4,
                                                _stream(stream)))

    def xor32(self, out, stream=None, offset: int = 0, nbytes=None):
        """out[0..1023] (device) XOR to the XOR of the buffer's 32-bit words (oco_buffer_xor32)."""
        n = (self.nbytes - offset) if nbytes is None else nbytes
        _check(load_library().oco_buffer_xor32(self.ptr + offset, n // 4, _addr(out), _stream(stream)))

    def at(self, offset: int) -> int:
        return self.ptr + offset

    def free(self):
        if self.ptr:
            _check(load_library().oco_buffer_free(self.ptr))
            self.ptr = 0

    def __del__(self):
        try:
            if self.ptr and _lib is not None:
                _lib.oco_buffer_free(self.ptr)
        except Exception:
            pass


def _addr(b) -> int | None:
    if type(b) is int or b is None:  # the usual case of a serving loop, first
        return b
    if isinstance(b, DeviceBuffer):
        return b.ptr
    return int(b)


def synchronize(stream=None):
    if stream is None:
        _check(load_library().oco_stream_sync(None))
    else:
        _check(load_library().oco_stream_sync(_stream(stream)))


# ---- operations (thin wrappers over the C ABI) -------------------------------

def dequant(fmt: int, w, count: int, out, stream=None):
    _check(load_library().oco_dequant(int(fmt), _addr(w), count, _addr(out), _stream(stream)))


def embed(fmt: int, w, k: int, vocabulary: int, ids, rows: int, out, features=None, feature_rows: int = 0,
          stream=None):
    """Token rows to bf16 (embed, weights.metal:90-109): ids >= vocabulary take feature rows."""
    _check(load_library().oco_embed(int(fmt), _addr(w), k, vocabulary, _addr(ids), rows, _addr(features),
                                    feature_rows, _addr(out), _stream(stream)))


class Embedding:
    """Embedding operand (src/weights/operands.rs Embedding; Builder::embedding,
    pipelines.rs:180-193): a GGUF tensor [width, vocabulary] and its lookup."""

    def __init__(self, fmt: int, values, width: int, vocabulary: int):
        self.format, self.values, self.width, self.vocabulary = int(fmt), values, width, vocabulary

    def embed(self, ids, rows: int, out, features=None, feature_rows: int = 0, stream=None):
        """Compute::embed (compute/matrix.rs:487-516)."""
        embed(self.format, self.values, self.width, self.vocabulary, ids, rows, out, features, feature_rows, stream)


def matvec(fmt: int, w, x, y, p: Matrix, x_dtype=DType.F32, y_dtype=DType.F32, bias=None,
           ids=None, stream=None, relu_sqr: bool = False):
    """oco_matvec, or oco_matvec_relu_sqr (x -> max(x, 0)^2 on load) when relu_sqr."""
    lib = load_library()
    fn = lib.oco_matvec_relu_sqr if relu_sqr else lib.oco_matvec
    _check(fn(int(fmt), _addr(w), _addr(x), int(x_dtype), _addr(y), int(y_dtype), _addr(bias), _addr(ids),
              ctypes.byref(as_matrix(p)), _stream(stream)))


def matmul(fmt: int, w, x, y, p: Matrix, x_dtype=DType.BF16, y_dtype=DType.F32, bias=None,
           stream=None, workspace=None, workspace_bytes: int = 0):
    """oco_matmul, or oco_matmul_ws when a workspace is given."""
    lib = load_library()
    if workspace is None:
        _check(lib.oco_matmul(int(fmt), _addr(w), _addr(x), int(x_dtype), _addr(y), int(y_dtype),
                              _addr(bias), ctypes.byref(as_matrix(p)), _stream(stream)))
    else:
        _check(lib.oco_matmul_ws(int(fmt), _addr(w), _addr(x), int(x_dtype), _addr(y), int(y_dtype),
                                 _addr(bias), ctypes.byref(as_matrix(p)), _addr(workspace),
                                 int(workspace_bytes), _stream(stream)))


class MatmulKernel(enum.IntEnum):
    """oco_matmul_kernel."""
    VECTOR = 0
    MX = 1
    FEW_ROWS = 2
    TILES = 3
    PANEL = 4
    GEMM = 5


def matmul_route(fmt: int, p: Matrix, x_dtype=DType.BF16, y_dtype=DType.F32, workspace_bytes: int | None = None):
    """oco_matmul_route: (kernel, row tiles, column tiles, K parts); by default with the reported workspace."""
    if workspace_bytes is None:
        workspace_bytes = matmul_workspace(fmt, p, x_dtype)
    out = (_u32 * 4)()
    _check(load_library().oco_matmul_route(int(fmt), int(x_dtype), int(y_dtype), ctypes.byref(as_matrix(p)),
                                           int(workspace_bytes), out))
    return (MatmulKernel(out[0]), *out[1:])


def matmul_workspace(fmt: int, p: Matrix, x_dtype=DType.BF16) -> int:
    return int(load_library().oco_matmul_workspace(int(fmt), int(x_dtype), ctypes.byref(as_matrix(p))))


def norm_mx_split(x, w, y, rows: int, n: int, epsilon: float, full_layer: bool, split, split_bytes: int,
                  stream=None):
    """oco_norm_mx_split: RMS norm rows (y optional) and their MXFP4-prefill split records."""
    _check(load_library().oco_norm_mx_split(_addr(x), _addr(w), _addr(y), rows, n, float(epsilon),
                                            1 if full_layer else 0, _addr(split), int(split_bytes),
                                            _stream(stream)))


def add_norm_mx_split(x, y, w, out, rows: int, n: int, epsilon: float, full_layer: bool, split, split_bytes: int,
                      stream=None):
    """oco_add_norm_mx_split: x = bf16(x + y), then norm_mx_split of x (out optional)."""
    _check(load_library().oco_add_norm_mx_split(_addr(x), _addr(y), _addr(w), _addr(out), rows, n, float(epsilon),
                                                1 if full_layer else 0, _addr(split), int(split_bytes),
                                                _stream(stream)))


def matmul_mx_split(w, split, split_bytes: int, y, p: Matrix, y_dtype=DType.F32, bias=None, stream=None):
    """oco_matmul_mx_split: the MXFP4 prefill from rows split by norm_mx_split."""
    _check(load_library().oco_matmul_mx_split(_addr(w), _addr(split), int(split_bytes), _addr(y), int(y_dtype),
                                              _addr(bias), ctypes.byref(as_matrix(p)), _stream(stream)))


def fp8_quantize(x, rows: int, k: int, codes, scales, x_dtype=DType.BF16, x_stride: int = 0, stream=None):
    """oco_fp8_quantize: rows to e4m3 codes [rows, k] and f32 scales [ceil(k / 128)][rows]."""
    _check(load_library().oco_fp8_quantize(_addr(x), int(x_dtype), rows, k, x_stride, _addr(codes), _addr(scales),
                                           _stream(stream)))


def fp8_matmul_workspace(p: Matrix) -> int:
    return int(load_library().oco_fp8_matmul_workspace(ctypes.byref(as_matrix(p))))


def fp8_matmul(w, w_scales, codes, scales, y, p: Matrix, y_dtype=DType.F32, bias=None, workspace=None,
               workspace_bytes: int = 0, stream=None):
    """oco_fp8_matmul: e4m3 rows times e4m3 weights with a scale per block of 128 x 128."""
    _check(load_library().oco_fp8_matmul(_addr(w), _addr(w_scales), _addr(codes), _addr(scales), _addr(y), int(y_dtype),
                                         _addr(bias), ctypes.byref(as_matrix(p)), _addr(workspace), int(workspace_bytes),
                                         _stream(stream)))


def block_norm(x, y, p: Block, x_out=None, gate=None, post_w=None, pre_w=None, out=None, codes=None, scales=None,
               stream=None):
    """oco_block_norm: x_out (x itself by default) = x + scale gate norm(y), out = norm(x_out)."""
    _check(load_library().oco_block_norm(_addr(x), _addr(y), _addr(x if x_out is None else x_out), _addr(gate),
                                         _addr(post_w), _addr(pre_w), _addr(out), _addr(codes), _addr(scales),
                                         ctypes.byref(p), _stream(stream)))


def route_scores(logits, tokens: int, p: Routing, ids, weights, dtype=DType.F32, bias=None, stream=None):
    """oco_route_scores: experts by softmax or sigmoid scores, a balance bias and groups."""
    _check(load_library().oco_route_scores(_addr(logits), int(dtype), _addr(bias), tokens, ctypes.byref(p), _addr(ids),
                                           _addr(weights), _stream(stream)))


def draft_verify_workspace(p: Draft) -> int:
    return int(load_library().oco_draft_verify_workspace(ctypes.byref(p)))


def draft_verify(target, draft, draft_ids, uniforms, accepted, tokens, p: Draft, lengths=None, probabilities=None,
                 workspace=None, workspace_bytes: int = 0, stream=None):
    """oco_draft_verify: drafted tokens against the target's distribution, from given random numbers."""
    _check(load_library().oco_draft_verify(_addr(target), _addr(draft), _addr(draft_ids), _addr(lengths), _addr(uniforms),
                                           _addr(accepted), _addr(tokens), _addr(probabilities), ctypes.byref(p),
                                           _addr(workspace), int(workspace_bytes), _stream(stream)))


def rotation_frequencies(dim: int, base: float = 10000.0, scaling=Scaling.NONE, factor: float = 1.0, original: float = 0.0,
                         fast: float = 32.0, slow: float = 1.0, factors=None):
    """oco_rotation_frequencies: (f64 [dim / 2] radians per position, magnitude), on the host."""
    extra = None if factors is None else np.ascontiguousarray(factors, np.float32)
    if extra is not None and extra.shape != (dim // 2,):
        raise ValueError(f"factors of {extra.shape} for {dim // 2} pairs")
    out, magnitude = np.empty(dim // 2), ctypes.c_double()
    p = Frequencies(dim, int(scaling), base, factor, original, fast, slow, None if extra is None else extra.ctypes.data)
    _check(load_library().oco_rotation_frequencies(ctypes.byref(p), out.ctypes.data, ctypes.byref(magnitude)))
    return out, magnitude.value


def rotate(x, rows: int, heads: int, head_dim: int, out, rotation: Rotation, positions, dtype=DType.BF16, x_stride: int = 0,
           out_stride: int = 0, stream=None):
    """oco_rotate: rows of heads, turned by their positions (out may be x)."""
    _check(load_library().oco_rotate(_addr(x), int(dtype), rows, heads, head_dim, x_stride, _addr(positions), _addr(out),
                                     out_stride, ctypes.byref(rotation), _stream(stream)))


def cache_page_bytes(p: Cache) -> int:
    return int(load_library().oco_cache_page_bytes(ctypes.byref(p)))


def cache_append(pages, table, lengths, k, v, p: Cache, starts=None, q=None, q_out=None, positions=None, rotation=None,
                 stream=None):
    """oco_cache_append: a batch's keys (turned) and values into the pages, its queries turned into q_out (q by default)."""
    _check(load_library().oco_cache_append(_addr(pages), _addr(table), _addr(starts), _addr(lengths), _addr(positions), _addr(q),
                                           _addr(k), _addr(v), _addr(q if q_out is None else q_out),
                                           None if rotation is None else ctypes.byref(rotation), ctypes.byref(p), _stream(stream)))


def cache_read(pages, table, lengths, k, v, p: Cache, starts=None, stream=None):
    """oco_cache_read: a batch's rows out of the pages, as the values they stand for."""
    _check(load_library().oco_cache_read(_addr(pages), _addr(table), _addr(starts), _addr(lengths), _addr(k), _addr(v),
                                         ctypes.byref(p), _stream(stream)))


def cache_attention_workspace(p: Cache) -> int:
    return int(load_library().oco_cache_attention_workspace(ctypes.byref(p)))


def cache_attention(q, pages, table, lengths, out, p: Cache, starts=None, sinks=None, workspace=None, workspace_bytes: int = 0,
                    stream=None):
    """oco_cache_attention: causal attention of a batch's rows over their sequences' pages."""
    _check(load_library().oco_cache_attention(_addr(q), _addr(pages), _addr(table), _addr(starts), _addr(lengths), _addr(sinks),
                                              _addr(out), ctypes.byref(p), _addr(workspace), int(workspace_bytes),
                                              _stream(stream)))


def logits_adjust(logits, out, p: Logits, history=None, history_lengths=None, penalties=None, bias_ids=None, biases=None,
                  bias_lengths=None, mask=None, stream=None):
    """oco_logits_adjust: penalties for repeated tokens, biases and masks (out may be logits)."""
    _check(load_library().oco_logits_adjust(_addr(logits), _addr(out), _addr(history), _addr(history_lengths), _addr(penalties),
                                            _addr(bias_ids), _addr(biases), _addr(bias_lengths), _addr(mask), ctypes.byref(p),
                                            _stream(stream)))


def route_select(logits, tokens: int, experts: int, k: int, ids, probs, stream=None):
    _check(load_library().oco_route_select(_addr(logits), tokens, experts, k, _addr(ids),
                                           _addr(probs), _stream(stream)))


def router(x, x_dtype, w, bias, tokens, hidden, experts, k, logits, ids, probs, stream=None):
    _check(load_library().oco_router(_addr(x), int(x_dtype), _addr(w), _addr(bias), tokens, hidden,
                                     experts, k, _addr(logits), _addr(ids), _addr(probs),
                                     _stream(stream)))


def route_plan_words(routes: int, experts: int) -> int:
    return int(load_library().oco_route_plan_words(routes, experts))


def route_plan(ids, routes, experts, tile_rows, up_tiles, down_tiles, plan, stream=None):
    _check(load_library().oco_route_plan(_addr(ids), routes, experts, tile_rows, up_tiles,
                                         down_tiles, _addr(plan), _stream(stream)))


def moe_sum(routes, routes_dtype, probs, out, hidden, tokens, k, stream=None):
    _check(load_library().oco_moe_sum(_addr(routes), int(routes_dtype), _addr(probs), _addr(out),
                                      hidden, tokens, k, _stream(stream)))


def norm(x, w, y, rows: int, n: int, epsilon: float, full_layer: bool = True, stream=None):
    """Compute::norm (elementwise.metal:6-28) over bf16 rows."""
    _check(load_library().oco_norm(_addr(x), _addr(w), _addr(y), rows, n, epsilon, int(full_layer),
                                   _stream(stream)))


def add_norm(x, y, w, out, rows: int, n: int, epsilon: float, full_layer: bool = True, stream=None):
    """add_norm (elementwise.metal:32-58): x = bf16(x + y) in place, out = norm(x)."""
    _check(load_library().oco_add_norm(_addr(x), _addr(y), _addr(w), _addr(out), rows, n, epsilon,
                                       int(full_layer), _stream(stream)))


def matvec_norm(fmt: int, w, x, norm_w, epsilon: float, y, p: Matrix, full_layer: bool = True,
                y_dtype=DType.F32, bias=None, ids=None, stream=None):
    """norm -> matvec with the norm fused into the matvec's activation staging."""
    _check(load_library().oco_matvec_norm(int(fmt), _addr(w), _addr(x), _addr(norm_w), epsilon,
                                          int(full_layer), _addr(y), int(y_dtype), _addr(bias), _addr(ids),
                                          ctypes.byref(as_matrix(p)), _stream(stream)))


def matvec_group(fmt: int, ws, x, ys, p: Matrix, x_dtype=DType.BF16, y_dtype=DType.F32, norm_w=None,
                 epsilon: float = 1e-6, full_layer: bool = True, biases=None, stream=None):
    """Several matrices over the same input rows in one grid (the concurrent
    up/gate pair of feed_forward.rs:97-104); norm_w: fused RMS norm of bf16 x."""
    n = len(ws)
    wa = (ctypes.c_void_p * n)(*[_addr(w) for w in ws])
    ya = (ctypes.c_void_p * n)(*[_addr(y) for y in ys])
    ba = (ctypes.c_void_p * n)(*[_addr(b) for b in biases]) if biases is not None else None
    _check(load_library().oco_matvec_group(int(fmt), n, wa, _addr(x), int(x_dtype), _addr(norm_w), epsilon,
                                           int(full_layer), ya, int(y_dtype), ba, ctypes.byref(as_matrix(p)),
                                           _stream(stream)))


def argmax_workspace(n: int) -> int:
    return int(load_library().oco_argmax_workspace(n))


def argmax(logits, n: int, out, stream=None, workspace=None, workspace_bytes: int = 0):
    """Compute::argmax (compute.rs:132-140): greedy token over f32 logits."""
    lib = load_library()
    if workspace is None:
        _check(lib.oco_argmax_f32(_addr(logits), n, _addr(out), _stream(stream)))
    else:
        _check(lib.oco_argmax_f32_ws(_addr(logits), n, _addr(out), _addr(workspace), int(workspace_bytes),
                                     _stream(stream)))


# ---- GGUF checkpoints (src/gguf.rs) ---------------------------------------------

class Gguf:
    """Gguf (gguf.rs:98-348): an open, structurally validated GGUF v3 file."""

    def __init__(self, path: str, keep=()):
        lib = load_library()
        keys = [k.encode() for k in keep]
        arr = (ctypes.c_char_p * max(len(keys), 1))(*keys)
        h = ctypes.c_void_p()
        _check(lib.oco_gguf_open(os.fsencode(path), arr, len(keys), ctypes.byref(h)))
        self.handle = h

    def close(self):
        if self.handle:
            load_library().oco_gguf_close(self.handle)
            self.handle = None

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _bytes(self, fn, key, *extra):
        p, n = ctypes.c_void_p(), ctypes.c_size_t()
        _check(fn(self.handle, key.encode(), *extra, ctypes.byref(p), ctypes.byref(n)))
        return ctypes.string_at(p.value, n.value).decode() if n.value else ""

    def has(self, key: str) -> bool:
        return bool(load_library().oco_gguf_has(self.handle, key.encode()))

    def text(self, key: str) -> str:
        return self._bytes(load_library().oco_gguf_text, key)

    def number(self, key: str) -> float:
        v = ctypes.c_double()
        _check(load_library().oco_gguf_number(self.handle, key.encode(), ctypes.byref(v)))
        return v.value

    def boolean(self, key: str) -> bool:
        v = ctypes.c_int()
        _check(load_library().oco_gguf_boolean(self.handle, key.encode(), ctypes.byref(v)))
        return bool(v.value)

    def optional_unsigned(self, key: str):
        if not self.has(key):
            return None
        v = ctypes.c_uint64()
        _check(load_library().oco_gguf_unsigned(self.handle, key.encode(), ctypes.byref(v)))
        return v.value

    def strings(self, key: str) -> list:
        kind, count = ctypes.c_uint32(), ctypes.c_uint64()
        _check(load_library().oco_gguf_array(self.handle, key.encode(), ctypes.byref(kind), ctypes.byref(count)))
        return [self._bytes(load_library().oco_gguf_array_string, key, ctypes.c_uint64(i)) for i in range(count.value)]

    def unsigned_integers(self, key: str) -> list:
        kind, count = ctypes.c_uint32(), ctypes.c_uint64()
        _check(load_library().oco_gguf_array(self.handle, key.encode(), ctypes.byref(kind), ctypes.byref(count)))
        out = np.zeros(max(count.value, 1), np.uint64)
        _check(load_library().oco_gguf_array_unsigned(self.handle, key.encode(), out.ctypes.data, count.value))
        return [int(v) for v in out[:count.value]]

    def directory(self) -> dict:
        lib = load_library()
        n = ctypes.c_uint64()
        _check(lib.oco_gguf_directory(self.handle, ctypes.byref(n)))
        out = {}
        for i in range(n.value):
            name, e = ctypes.c_char_p(), GgufEntry()
            _check(lib.oco_gguf_entry_at(self.handle, i, ctypes.byref(name), ctypes.byref(e)))
            out[name.value.decode()] = e
        return out

    @staticmethod
    def select(entry: GgufEntry) -> GgufTensor:
        t = GgufTensor()
        _check(load_library().oco_gguf_select(ctypes.byref(entry), ctypes.byref(t)))
        return t

    def data(self, t: GgufTensor) -> np.ndarray:
        p = load_library().oco_gguf_data(self.handle, ctypes.byref(t))
        if not p:
            raise OcoError(5, "tensor outside the mapping")
        return np.ctypeslib.as_array((ctypes.c_uint8 * t.bytes).from_address(p)).copy()

    def upload(self, t: GgufTensor, dst=None, stream=None) -> "DeviceBuffer":
        buf = dst if dst is not None else DeviceBuffer(t.bytes)
        _check(load_library().oco_gguf_upload(self.handle, ctypes.byref(t), _addr(buf), _stream(stream)))
        return buf


# ---- operator mirror -----------------------------------------------------------

class DenseMatrix:
    """A learned linear map with its GGUF storage (operands.rs:4-9).

    ``input``/``output`` follow oco's [input, output] GGUF shape convention
    (load.rs:175-186); ``values`` is the device buffer of GGUF rows.
    """

    def __init__(self, values: DeviceBuffer, fmt: int, input: int, output: int, offset: int = 0):
        self.values, self.format, self.input, self.output = values, int(fmt), input, output
        self.offset = offset
        row_bytes(fmt, input)

    def _w(self):
        return self.values.ptr + self.offset

    def apply_row(self, x, y, x_dtype=DType.F32, y_dtype=DType.F32, bias=None, rows: int = 1,
                  stream=None):
        """Decode path (compute/matrix.rs:63): y[r] = W x[r] for `rows` rows."""
        p = Matrix(self.input, self.output, rows, 0, 1, 1, 1 if bias is not None else 0)
        matvec(self.format, self._w(), x, y, p, x_dtype, y_dtype, bias, None, stream)

    def apply(self, x, y, rows: int, x_dtype=DType.BF16, y_dtype=DType.F32, bias=None,
              stream=None):
        """Prefill path (compute/matrix.rs:130): Y = X W^T on MFMA."""
        p = Matrix(self.input, self.output, rows, 0, 1, 1, 1 if bias is not None else 0)
        matmul(self.format, self._w(), x, y, p, x_dtype, y_dtype, bias, stream)


class Output(DenseMatrix):
    """lm_head scoring in f32 (Bindings::output, compute/matrix.rs:519-548)."""

    def apply_row(self, x, y, x_dtype=DType.F32, y_dtype=DType.F32, bias=None, rows: int = 1,
                  stream=None):
        super().apply_row(x, y, x_dtype, DType.F32, bias, rows, stream)


class Fp8Matrix:
    """A learned linear map in e4m3 with an f32 scale per block of 128 x 128:
    the counterpart of DenseMatrix for rows in 8-bit floating point."""

    def __init__(self, values, scales, input: int, output: int):
        if input % 16:
            raise ValueError(f"input={input} is not whole groups of 16")
        self.values, self.scales, self.input, self.output = values, scales, input, output
        self._scratches = {}  # of streams that are given by their handle

    def apply(self, codes, scales, y, rows: int, y_dtype=DType.F32, bias=None, workspace=None, stream=None):
        """Y = X W^T for rows of oco_fp8_quantize or oco_block_norm.  Without a
        `workspace` (a DeviceBuffer of fp8_matmul_workspace bytes) a Stream
        keeps one for all its matrices, and the matrix one for each stream that
        is given by its handle and for the default one.  Before a capture
        reserve() draws it, and graphs that run on other streams than they were
        captured on bring their own."""
        p = Matrix(self.input, self.output, rows, 0, 1, 1, 1 if bias is not None else 0)
        need = fp8_matmul_workspace(p)
        if need and workspace is None:
            workspace = self._scratch(stream).at_least(need)
        fp8_matmul(self.values, self.scales, codes, scales, y, p, y_dtype, bias, workspace if need else None,
                   workspace.nbytes if need else 0, stream)

    def reserve(self, rows: int, stream=None):
        """The workspace of calls of 1 to `rows` rows on a stream (the need
        does not rise with the rows throughout), which then draw no memory."""
        need = max((fp8_matmul_workspace(Matrix(self.input, self.output, m, 0, 1, 1, 0)) for m in range(1, rows + 1)), default=0)
        if need:
            self._scratch(stream).at_least(need)

    def _scratch(self, stream) -> Scratch:
        if isinstance(stream, Stream):
            return stream.scratch
        return self._scratches.setdefault(getattr(stream, "value", stream), Scratch())


class PagedCache:
    """A pool of pages with keys and values in 4 bits (oco_cache), and the calls on it.

    A batch is described once and kept: ``batch(table, lengths, ...)`` binds the
    sequences' pages and lengths to the pool, and append, read and attention
    take their rows from it."""

    def __init__(self, pages: int, head_dim: int, kv_heads: int, page_size: int = 64, buffer=None):
        self.pages, self.head_dim, self.kv_heads, self.page_size = pages, head_dim, kv_heads, page_size
        page = cache_page_bytes(Cache(head_dim=head_dim, kv_heads=kv_heads, page_size=page_size))
        if page == 0:
            raise ValueError(f"no cache of {kv_heads} heads of {head_dim} in pages of {page_size} tokens")
        if buffer is not None and buffer.nbytes < pages * page:
            raise ValueError(f"{buffer.nbytes} bytes for {pages} pages of {page}")
        self.buffer = DeviceBuffer(pages * page) if buffer is None else buffer

    def batch(self, table, lengths, sequences: int, rows: int, max_rows: int, max_length: int, table_stride: int, heads: int,
              starts=None, dtype=DType.BF16, window: int = 0, scale: float = 0.0) -> "CacheBatch":
        p = Cache(head_dim=self.head_dim, heads=heads, kv_heads=self.kv_heads, page_size=self.page_size, pages=self.pages,
                  sequences=sequences, rows=rows, max_rows=max_rows, max_length=max_length, table_stride=table_stride,
                  dtype=int(dtype), window=window, scale=scale)
        return CacheBatch(self, p, table, starts, lengths)


class CacheBatch:
    """The rows of a step on a PagedCache."""

    def __init__(self, cache: PagedCache, p: Cache, table, starts, lengths):
        self.cache, self.p, self.table, self.starts, self.lengths = cache, p, table, starts, lengths
        self._scratches = {}  # of streams that are given by their handle

    def append(self, k, v, q=None, q_out=None, positions=None, rotation=None, stride: int = 0, stream=None):
        """Keys (turned) and values into the pages, queries turned into q_out (q
        by default).  stride: between the rows of q, k and v where they lie
        together, as one product writes them; q_out's stay head after head,
        unless it is q."""
        p = self.p
        if stride:
            p = Cache.from_buffer_copy(p)
            p.k_stride = p.v_stride = stride
            if q is not None:
                p.q_stride = stride
                if q_out is None or _addr(q_out) == _addr(q):
                    p.out_stride = stride
        cache_append(self.cache.buffer, self.table, self.lengths, k, v, p, self.starts, q, q_out, positions, rotation, stream)

    def read(self, k, v, stream=None):
        """The rows' keys and values as the pages hold them."""
        cache_read(self.cache.buffer, self.table, self.lengths, k, v, self.p, self.starts, stream)

    def attention(self, q, out, sinks=None, workspace=None, stream=None, stride: int = 0):
        """Causal attention of the rows.  Without a `workspace` (a DeviceBuffer
        of workspace_bytes()) a Stream keeps one, and the batch one for each
        stream that is given by its handle and for the default one; reserve()
        draws it before a capture.  stride: between q's rows where they were
        turned in their place among keys and values (out's stay head after
        head, unless it is q)."""
        need = self.workspace_bytes()
        if need and workspace is None:
            workspace = self._scratch(stream).at_least(need)
        p = self.p
        if stride:
            p = Cache.from_buffer_copy(p)
            p.q_stride = stride
            if _addr(out) == _addr(q):
                p.out_stride = stride
        cache_attention(q, self.cache.buffer, self.table, self.lengths, out, p, self.starts, sinks, workspace if need else None,
                        workspace.nbytes if need else 0, stream)

    def workspace_bytes(self) -> int:
        return cache_attention_workspace(self.p)

    def reserve(self, stream=None):
        need = self.workspace_bytes()
        if need:
            self._scratch(stream).at_least(need)

    def _scratch(self, stream) -> Scratch:
        if isinstance(stream, Stream):
            return stream.scratch
        return self._scratches.setdefault(getattr(stream, "value", stream), Scratch())


class ExpertBank:
    """Routed expert weights (gpt_oss/load.rs:20-40; Experts/ExpertPlan, feed_forward.rs:34-77)."""

    def __init__(self, fmt: int, hidden: int, ffn: int, experts: int, k: int, gate, up, down,
                 gate_bias=None, up_bias=None, down_bias=None,
                 activation=Activation.SWIGLU_CLIPPED, up_bias_one: bool = True):
        self.desc = ExpertsDesc(int(fmt), hidden, ffn, experts, k, int(activation),
                                1 if up_bias_one else 0, _addr(gate), _addr(up), _addr(down),
                                _addr(gate_bias), _addr(up_bias), _addr(down_bias))
        self._keep = (gate, up, down, gate_bias, up_bias, down_bias)
        self._workspace = None

    def workspace_bytes(self, tokens: int) -> int:
        return int(load_library().oco_experts_workspace(ctypes.byref(self.desc), tokens))

    def apply(self, x, x_dtype, ids, probs, tokens: int, out, routed=None, workspace=None,
              stream=None):
        """Bindings::experts (feed_forward.rs:107-275) after the router."""
        need = self.workspace_bytes(tokens)
        if workspace is None:
            if self._workspace is None or self._workspace.nbytes < need:
                self._workspace = DeviceBuffer(max(need, 256))
            workspace = self._workspace
        ws_bytes = workspace.nbytes if isinstance(workspace, DeviceBuffer) else need
        _check(load_library().oco_experts_apply(ctypes.byref(self.desc), _addr(x), int(x_dtype),
                                                _addr(ids), _addr(probs), tokens, _addr(out),
                                                _addr(routed), _addr(workspace), ws_bytes,
                                                _stream(stream)))

    def forward(self, router_w, router_bias, x, x_dtype, tokens: int, out, ids, probs, routed=None,
                workspace=None, stream=None):
        """Bindings::experts (feed_forward.rs:107-275) from the router logits on:
        ids/probs [tokens, k] receive the device's expert selection."""
        need = self.workspace_bytes(tokens)
        if workspace is None:
            if self._workspace is None or self._workspace.nbytes < need:
                self._workspace = DeviceBuffer(max(need, 256))
            workspace = self._workspace
        ws_bytes = workspace.nbytes if isinstance(workspace, DeviceBuffer) else need
        _check(load_library().oco_experts_forward(ctypes.byref(self.desc), _addr(router_w), _addr(router_bias),
                                                  _addr(x), int(x_dtype), tokens, _addr(out), _addr(ids),
                                                  _addr(probs), _addr(routed), _addr(workspace), ws_bytes,
                                                  _stream(stream)))

    def expand(self, x, x_dtype, logits, ids, probs, up_out, act_out, stream=None):
        """expert_expand (projections.metal:78-137) for one token."""
        _check(load_library().oco_expert_expand(ctypes.byref(self.desc), _addr(x), int(x_dtype),
                                                _addr(logits), _addr(ids), _addr(probs),
                                                _addr(up_out), _addr(act_out), _stream(stream)))

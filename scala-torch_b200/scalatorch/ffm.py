"""Host-side binding of libstb200.so -- the Python mirror of scala-torch's ffm module.

The reference reaches the GPU through Java FFM downcalls (ffm/src/main/scala/scalatorch/ffm/
CudaDriver.scala:13-19): each call returns an int status and a nonzero status becomes an
exception.  This module binds the same way with ctypes and keeps the reference's error
vocabulary: invalid arguments raise IllegalArgumentException *before* any native call, native
failures raise IllegalStateException("<fn> failed with status <code>: <message>").

`B200Session` is the device FloatBackend (core/.../FloatBackend.scala:7-31, the trait CudaSession
implements, CudaSession.scala:23-24): upload / download / release / shape / reshape / transpose /
embedding / matmul (against resident (out,in) half weights: the hot path) / add / multiply / scale /
fill / sum / expandScalar / silu / rmsNorm / rope / causalAttention / attentionCache, plus the raw
half upload that replaces SafeTensors.readFloat's F32 widening.

There is no fallback: if libstb200.so is missing or fails to load, every entry point raises.
"""
from __future__ import annotations

import ctypes
import functools
import math
import os
from dataclasses import dataclass, field

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(os.path.dirname(HERE), "libstb200.so")

STB_F32, STB_BF16, STB_F16, STB_E4M3 = 0, 1, 2, 3
STB_U8, STB_I32 = 4, 5  # element types of this binding's buffers alone: scale bytes and row indices
ELEMENT_BYTES = {STB_F32: 4, STB_BF16: 2, STB_F16: 2, STB_E4M3: 1, STB_U8: 1, STB_I32: 4}
DTYPE_NAMES = {"F32": STB_F32, "BF16": STB_BF16, "F16": STB_F16}
STATUS = {0: "OK", 1: "INVALID", 2: "BUDGET", 3: "CUDA", 4: "NCCL", 5: "THREAD", 6: "STATE", 7: "UNSUPPORTED"}


class IllegalArgumentException(ValueError):
    """Rejected request (the reference's require(...) failures)."""


class IllegalStateException(RuntimeError):
    """Native failure or misuse of a closed / foreign handle."""

    def __init__(self, fn: str, code: int, message: str):
        super().__init__(f"{fn} failed with status {code} ({STATUS.get(code, '?')}): {message}")
        self.code = code


_lib = None
_p = ctypes.c_void_p
_u64 = ctypes.c_uint64
_i = ctypes.c_int
_i64 = ctypes.c_int64
_pp = ctypes.POINTER(ctypes.c_void_p)


def library() -> ctypes.CDLL:
    """Load libstb200.so (built in-tree by scala-torch_b200/build.py).  Raises if absent."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise IllegalStateException("load", -1, f"{LIB_PATH} is missing; run scala-torch_b200/build.py")
        lib = ctypes.CDLL(LIB_PATH)
        _declare(lib)
        _lib = lib
    return _lib


def _declare(L):
    sig = {
        "stb_version": (_i, []),
        "stb_last_error": (ctypes.c_char_p, []),
        "stb_session_create": (_i, [_i, _u64, _pp]),
        "stb_session_destroy": (_i, [_p]),
        "stb_session_allocated": (_i, [_p, ctypes.POINTER(_u64)]),
        "stb_session_stream": (_i, [_p, _pp]),
        "stb_session_launches": (_i, [_p, ctypes.POINTER(_u64)]),
        "stb_alloc": (_i, [_p, _u64, ctypes.POINTER(_u64)]),
        "stb_release": (_i, [_p, _u64]),
        "stb_upload": (_i, [_p, _p, _u64, _u64]),
        "stb_download": (_i, [_p, _u64, _p, _u64]),
        "stb_copy": (_i, [_p, _u64, _u64, _u64]),
        "stb_sync": (_i, [_p]),
        "stb_host_alloc": (_i, [_u64, _pp]),
        "stb_host_free": (_i, [_p]),
        "stb_linear": (_i, [_p, _u64, _u64, _i, _u64, _u64, _i, _i, _i]),
        "stb_linear_ld": (_i, [_p, _u64, _i, _u64, _i, _u64, _u64, _i, _i, _i, _i]),
        "stb_linear_prefill": (_i, [_p, _u64, _u64, _i, _u64, _u64, _i, _i, _i]),
        "stb_linear_host": (_i, [_p, _p, _u64, _i, _u64, _p, _i, _i, _i]),
        "stb_linear_prefill_static": (_i, [_p, _u64, _u64, _i, _u64, _u64, _i, _i, _i]),
        "stb_linear_adapted": (_i, [_p, _u64, _u64, _i, _u64, _p, _i, _u64, _i, _i, _i]),
        "stb_fill_normal": (_i, [_p, _u64, _i, _u64, _u64, _u64, ctypes.c_double]),
        "stb_fill_value": (_i, [_p, _u64, _i, _u64, ctypes.c_float]),
        "stb_op_add": (_i, [_p, _u64, _u64, _u64, _u64]),
        "stb_op_multiply": (_i, [_p, _u64, _u64, _u64, _u64]),
        "stb_op_scale": (_i, [_p, _u64, _u64, _u64, ctypes.c_float]),
        "stb_op_silu": (_i, [_p, _u64, _u64, _u64]),
        "stb_op_sum": (_i, [_p, _u64, _u64, _u64]),
        "stb_op_expand_scalar": (_i, [_p, _u64, _u64, _u64]),
        "stb_op_rmsnorm": (_i, [_p, _u64, _u64, _u64, _u64, _i, ctypes.c_double]),
        "stb_op_rope": (_i, [_p, _u64, _u64, _i, _i, _i, _i, _i, ctypes.c_double]),
        "stb_op_transpose": (_i, [_p, _u64, _u64, _i, _p, _i, _i]),
        "stb_op_embedding": (_i, [_p, _u64, _i, ctypes.c_int64, _i, _p, _u64, _u64]),
        "stb_op_cache_append": (_i, [_p, _u64, _u64, _i, _i, _i, _i, _i, _i]),
        "stb_op_causal_attention": (_i, [_p, _u64, _u64, _u64, _u64] + [_i] * 9),
        "stb_linear_pool": (_i, [_p, _u64, _u64, _i, _u64, _p, _u64, _u64, _i, _i, _i]),
        "stb_op_qk_norm_rope": (_i, [_p, _u64, _i64, _i, _u64, _i64, _i, _i, _i, _u64, _u64, _u64, ctypes.c_double,
                                     ctypes.c_double, _u64, _i64, _u64, _i64]),
        "stb_op_paged_append": (_i, [_p, _p, _u64, _i64, _i64, _u64, _i64, _i64, _u64, _i, _i, _u64, _u64, _i]),
        "stb_op_paged_read": (_i, [_p, _p, _u64, _i, _i, _u64, _u64, _i, _u64, _i64, _i64, _u64, _i64, _i64]),
        "stb_op_paged_attention": (_i, [_p, _p, _u64, _i64, _i, _u64, _i, _i, _u64, _u64, _i64]),
        "stb_nccl_unique_id": (_i, [_p]),
        "stb_session_init_tp": (_i, [_p, _i, _i, _p]),
        "stb_allreduce_sum_f32": (_i, [_p, _u64, _u64]),
    }
    for name, (res, args) in sig.items():
        fn = getattr(L, name, None)
        if fn is None:
            continue
        fn.restype = res
        fn.argtypes = args


_functions: dict = {}  # bound entry points by name


def call(name: str, *args) -> None:
    """CudaDriver.call idiom: nonzero status -> exception with the library's message."""
    fn = _functions.get(name)
    if fn is None:
        fn = _functions[name] = getattr(library(), name)
    code = fn(*args)
    if code != 0:
        msg = library().stb_last_error().decode(errors="replace")
        if code == 1:
            raise IllegalArgumentException(f"{name}: {msg}")
        raise IllegalStateException(name, code, msg)


def require(cond: bool, message: str) -> None:
    if not cond:
        raise IllegalArgumentException(message)


def _of_tensors(method):
    """An operand that is no tensor at all is rejected like any other that the operator does not take."""
    @functools.wraps(method)
    def checked(*args, **kw):
        try:
            return method(*args, **kw)
        except AttributeError as e:
            raise IllegalArgumentException(f"operands must be tensors of the session: {e}") from e
    return checked


@dataclass(eq=False)
class DeviceTensor:
    """A resident device buffer with a logical shape (CudaTensor, CudaSession.scala:14-20).

    dtype is the element type in HBM.  `transposed_weight` marks a half (out,in) weight used as
    W^T: its logical shape is (in, out) -- what BackendLlama.prepare's upload(p, transposed=true)
    hands to matmul (BackendLlama.scala:161-162) -- but the bytes stay (out,in) and half."""
    session: "B200Session"
    address: int
    shape: tuple
    dtype: int = STB_F32
    nbytes: int = 0
    transposed_weight: bool = False
    owner: bool = True
    _alive: list = field(default_factory=lambda: [True])
    # handles on one allocation (reshape views share it, CudaSession.scala:95-101); freed at zero
    _refs: list = field(default_factory=lambda: [1])
    # elements between entries of axis 0 in a view of some columns (B200Session.columns); 0: packed
    row_stride: int = 0

    @property
    def numel(self) -> int:
        n = 1
        for d in self.shape:
            n *= int(d)
        return n

    def close(self) -> None:
        self.session.release(self)


class StbAdapter(ctypes.Structure):
    """stb_adapter (include/stb200.h)."""
    _fields_ = [("a", ctypes.c_uint64), ("b", ctypes.c_uint64), ("rank", ctypes.c_int), ("scale", ctypes.c_float),
                ("scoped", ctypes.c_int), ("multiplier", ctypes.c_float)]


class StbAdapterPool(ctypes.Structure):
    """stb_adapter_pool (include/stb200.h)."""
    _fields_ = [("a", ctypes.c_uint64), ("b", ctypes.c_uint64), ("ranks", ctypes.c_uint64), ("scales", ctypes.c_uint64),
                ("dtype", ctypes.c_int), ("slots", ctypes.c_int), ("max_rank", ctypes.c_int)]


class StbPagedCache(ctypes.Structure):
    """stb_paged_cache (include/stb200.h)."""
    _fields_ = [("keys", ctypes.c_uint64), ("values", ctypes.c_uint64), ("key_scales", ctypes.c_uint64),
                ("value_scales", ctypes.c_uint64), ("dtype", ctypes.c_int), ("pages", ctypes.c_int),
                ("page_size", ctypes.c_int), ("kv_heads", ctypes.c_int), ("width", ctypes.c_int)]


class LowRankAdapter:
    """nn.LowRankAdapter (nn/src/main/scala/scalatorch/nn/LowRankAdapter.scala:7-27) over resident
    Float32 factors: a [rank, in], b [out, rank]; scale = (alpha / rank) rounded to Float32."""

    def __init__(self, a: "DeviceTensor", b: "DeviceTensor", alpha: float):
        require(len(a.shape) == 2 and len(b.shape) == 2 and a.dtype == STB_F32 and b.dtype == STB_F32,
                "adapter factors must both be Float32 matrices")
        require(min(a.shape + b.shape) > 0 and a.shape[0] == b.shape[1], "invalid adapter factor dimensions")
        value = float(np.float32(alpha / a.shape[0])) if math.isfinite(alpha) and alpha > 0 else float("nan")
        require(math.isfinite(value) and value > 0, "invalid adapter scale")
        self.a, self.b, self.alpha, self.rank, self.scale = a, b, alpha, a.shape[0], value


class B200Session:
    """Thread-confined device session with a byte budget (CudaSession.withDevice)."""

    def __init__(self, device: int = 0, max_bytes: int = 1 << 30):
        require(device >= 0 and max_bytes >= 0, "invalid device or budget")
        h = ctypes.c_void_p()
        call("stb_session_create", device, max_bytes, ctypes.byref(h))
        self.handle = h
        self.device = device
        self.max_bytes = max_bytes
        self._closed = False

    # -- lifetime
    @classmethod
    def with_device(cls, device: int = 0, max_bytes: int = 1 << 30):
        return cls(device, max_bytes)

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def close(self) -> None:
        if not self._closed:
            self._closed = True
            call("stb_session_destroy", self.handle)

    def _check(self):
        if self._closed:
            raise IllegalStateException("session", 6, "session is closed")

    @property
    def allocated_bytes(self) -> int:
        self._check()
        v = ctypes.c_uint64()
        call("stb_session_allocated", self.handle, ctypes.byref(v))
        return v.value

    @property
    def launches(self) -> int:
        v = ctypes.c_uint64()
        call("stb_session_launches", self.handle, ctypes.byref(v))
        return v.value

    @property
    def stream(self) -> int:
        v = ctypes.c_void_p()
        call("stb_session_stream", self.handle, ctypes.byref(v))
        return v.value or 0

    def sync(self) -> None:
        self._check()
        call("stb_sync", self.handle)

    # -- memory
    def allocate(self, shape, dtype: int = STB_F32) -> DeviceTensor:
        self._check()
        shape = tuple(int(d) for d in shape)
        require(all(d >= 0 for d in shape), "negative dimension")
        require(dtype in ELEMENT_BYTES, "unknown element type")
        esz = ELEMENT_BYTES[dtype]
        n = 1
        for d in shape:
            n *= d
        addr = ctypes.c_uint64()
        call("stb_alloc", self.handle, n * esz, ctypes.byref(addr))
        return DeviceTensor(self, addr.value, shape, dtype, n * esz)

    def release(self, t: DeviceTensor) -> None:
        """Idempotent release (CudaSession.scala:852-861)."""
        self._check()
        require(t.session is self, "tensor belongs to another session")
        if t._alive[0]:
            t._alive[0] = False
            t._refs[0] -= 1
            if t.owner and t._refs[0] == 0:
                call("stb_release", self.handle, t.address)

    def _validate(self, t: DeviceTensor) -> None:
        self._check()
        require(isinstance(t, DeviceTensor) and t.session is self, "tensor belongs to another session")
        if not t._alive[0]:
            raise IllegalStateException("validate", 6, "tensor was released")
        require(t.row_stride == 0, "operation takes packed tensors, not a view of columns")

    def shape(self, t: DeviceTensor) -> tuple:
        self._validate(t)
        return t.shape

    def wrap(self, address: int, shape, dtype: int = STB_F32) -> DeviceTensor:
        """A tensor over device memory that the caller owns (another library's buffer, a slice of an arena): never
        freed here and not charged to the budget.  The caller orders its own work on that memory with the
        session's stream and keeps it alive."""
        self._check()
        shape = tuple(int(d) for d in shape)
        require(dtype in ELEMENT_BYTES, "unknown element type")
        require(all(d >= 0 for d in shape), "negative dimension")
        nbytes = math.prod(shape) * ELEMENT_BYTES[dtype]
        require(address % ELEMENT_BYTES[dtype] == 0 and (address != 0 or nbytes == 0), "null or misaligned memory")
        return DeviceTensor(self, address, shape, dtype, nbytes, owner=False)

    def columns(self, t: DeviceTensor, begin: int, shape) -> DeviceTensor:
        """A view of some columns of a matrix: entry r of axis 0 is t[r, begin : begin + prod(shape)] in `shape` --
        the query, key or value heads inside the rows of a fused projection.  Released like a reshape view; taken
        by the operators whose rows may lie apart (qk_norm_rope, a paged cache's append, read and attend)."""
        self._validate(t)
        shape = tuple(int(d) for d in shape)
        require(len(t.shape) == 2 and not t.transposed_weight and all(d > 0 for d in shape), "columns of a matrix")
        require(0 <= begin and begin + math.prod(shape) <= t.shape[1], "columns outside the matrix")
        t._refs[0] += 1
        return DeviceTensor(self, t.address + begin * ELEMENT_BYTES[t.dtype], (t.shape[0],) + shape, t.dtype, 0,
                            owner=t.owner, _refs=t._refs, row_stride=t.shape[1])

    def as_weight(self, t: DeviceTensor) -> DeviceTensor:
        """A view of a resident (out,in) matrix as the weight that matmul and the Linear forms take."""
        require(len(t.shape) == 2 and t.dtype in (STB_F32, STB_BF16, STB_F16) and not t.transposed_weight,
                "Linear weight must have shape (out, in)")
        w = self.reshape(t, t.shape)
        w.shape, w.transposed_weight = (t.shape[1], t.shape[0]), True
        return w

    # -- transfers
    def upload_ints(self, source) -> DeviceTensor:
        """Row indices, positions, lengths or page tables: int32 on the device.  Values outside Int are rejected."""
        a = np.asarray(source)
        require(a.dtype.kind in "iu" or a.size == 0, "indices must be whole numbers")
        require(a.size == 0 or (int(a.min()) >= -(1 << 31) and int(a.max()) < 1 << 31), "index exceeds Int")
        a = np.ascontiguousarray(a, np.int32)
        t = self.allocate(a.shape, STB_I32)
        try:
            if a.size:
                call("stb_upload", self.handle, a.ctypes.data, a.nbytes, t.address)
        except Exception:
            self.release(t)
            raise
        return t

    def upload(self, source: np.ndarray) -> DeviceTensor:
        """FloatBackend.upload of a Float32 tensor (packed row-major)."""
        a = np.ascontiguousarray(source, dtype=np.float32)
        t = self.allocate(a.shape, STB_F32)
        try:
            if a.size:
                call("stb_upload", self.handle, a.ctypes.data, a.nbytes, t.address)
        except Exception:
            self.release(t)
            raise
        return t

    def upload_half(self, bits: np.ndarray, dtype: int, shape=None, transposed_weight: bool = False) -> DeviceTensor:
        """Raw BF16/F16 payload straight into HBM, no F32 expansion (replaces SafeTensors.readFloat
        + upload of the widened weight, SafeTensors.scala:63-77 / BackendLlama.scala:161-168)."""
        require(dtype in (STB_BF16, STB_F16), "half upload requires BF16 or F16")
        raw = np.ascontiguousarray(bits)
        require(raw.dtype.itemsize == 2, "half payload must be 16-bit words")
        shape = tuple(shape) if shape is not None else raw.shape
        n = 1
        for d in shape:
            n *= int(d)
        require(n == raw.size, "shape does not match payload")
        t = self.allocate(shape, dtype)
        try:
            if raw.size:
                call("stb_upload", self.handle, raw.ctypes.data, raw.nbytes, t.address)
        except Exception:
            self.release(t)
            raise
        if transposed_weight:
            t.shape = (shape[1], shape[0])
            t.transposed_weight = True
        return t

    def upload_weight(self, bits: np.ndarray, dtype: int) -> DeviceTensor:
        """An (out,in) half weight used as W^T by matmul (BackendLlama.prepare's transposed upload)."""
        require(np.ndim(bits) == 2, "Linear weight must have shape (out, in)")
        return self.upload_half(bits, dtype, bits.shape, transposed_weight=True)

    def download(self, t: DeviceTensor) -> np.ndarray:
        self._validate(t)
        require(t.dtype == STB_F32, "download returns Float32 tensors")
        out = np.empty(t.shape, np.float32)
        call("stb_download", self.handle, t.address, out.ctypes.data, out.nbytes)
        return out

    def download_raw(self, t: DeviceTensor) -> np.ndarray:
        self._validate(t)
        out = np.empty(t.nbytes, np.uint8)
        call("stb_download", self.handle, t.address, out.ctypes.data, out.nbytes)
        return out

    # -- arithmetic on the hot path
    def matmul(self, a: DeviceTensor, b: DeviceTensor) -> DeviceTensor:
        """FloatBackend.matmul(x, W^T) where b is a resident (out,in) half weight
        (CudaSession.matmul, CudaSession.scala:561-571 -> the B200 decode GEMV)."""
        self._validate(a)
        self._validate(b)
        require(len(a.shape) == 2 and len(b.shape) == 2 and a.shape[1] == b.shape[0], "CUDA GEMM shape mismatch")
        require(a.dtype == STB_F32, "activations must be Float32")
        require(b.transposed_weight, "device matmul takes a resident (out,in) weight uploaded for W^T")
        M, K = a.shape
        N = b.shape[1]
        require(max(M, N, K) <= 0x7fffffff, "CUDA GEMM dimension exceeds Int indexing")
        y = self.allocate((M, N), STB_F32)
        try:
            call("stb_linear", self.handle, a.address, b.address, b.dtype, 0, y.address, M, N, K)
        except Exception:
            self.release(y)
            raise
        return y

    def linear(self, x: DeviceTensor, weight: DeviceTensor, bias: DeviceTensor | None = None,
               prefill: bool = False, lora: LowRankAdapter | None = None,
               scoped: tuple = ()) -> DeviceTensor:
        """nn.Linear.apply (Linear.scala:11-17): y = x.W^T (+ the Linear's own adapter)
        (+ LinearAdapterScope entries, each (LowRankAdapter, multiplier)) (+ bias).  prefill=True takes
        the tcgen05 path (x rounded to half; no adapters)."""
        self._validate(x)
        self._validate(weight)
        require(weight.transposed_weight, "weight must be a resident (out,in) weight")
        M, K = x.shape
        N = weight.shape[1]
        require(weight.shape[0] == K, "Linear shape mismatch")
        if bias is not None:
            self._validate(bias)
            require(bias.shape == (N,), "Linear bias shape mismatch")
        terms = ([(lora, 0, 1.0)] if lora is not None else []) + [(a, 1, float(m)) for a, m in scoped]
        for adapter, _, mult in terms:
            self._validate(adapter.a)
            self._validate(adapter.b)
            require(adapter.a.shape[1] == K and adapter.b.shape[0] == N, "Linear adapter shape mismatch")
            require(math.isfinite(mult), "adapter multiplier must be finite")
        require(not (prefill and terms), "the prefill form takes no adapters")
        y = self.allocate((M, N), STB_F32)
        try:
            if terms:
                arr = (StbAdapter * len(terms))(*[StbAdapter(a.a.address, a.b.address, a.rank, a.scale, sc, m)
                                                  for a, sc, m in terms])
                call("stb_linear_adapted", self.handle, x.address, weight.address, weight.dtype,
                     bias.address if bias is not None else 0, ctypes.cast(arr, ctypes.c_void_p), len(terms),
                     y.address, M, N, K)
            else:
                fn = "stb_linear_prefill" if prefill else "stb_linear"
                call(fn, self.handle, x.address, weight.address, weight.dtype,
                     bias.address if bias is not None else 0, y.address, M, N, K)
        except Exception:
            self.release(y)
            raise
        return y

    def fill_normal(self, t: DeviceTensor, seed: int, stream: int, std: float) -> None:
        self._validate(t)
        call("stb_fill_normal", self.handle, t.address, t.dtype, t.numel, seed, stream, std)

    def upload_weight_f32(self, w: np.ndarray) -> DeviceTensor:
        """A Float32 (out,in) matrix used as W^T by matmul (BackendLlama.prepare uploads adapter factors
        transposed, BackendLlama.scala:169; here the bytes stay (out,in))."""
        require(np.ndim(w) == 2, "weight must have shape (out, in)")
        t = self.upload(np.ascontiguousarray(w, np.float32))
        t.shape = (t.shape[1], t.shape[0])
        t.transposed_weight = True
        return t

    # -- FloatBackend operator set (FloatBackend.scala:7-31); each op is one kernel (csrc/ops.cu)
    def _out(self, shape) -> DeviceTensor:
        n = 1
        for d in shape:
            n *= int(d)
        require(n <= 0x7FFFFFFF, "CUDA tensor exceeds Int indexing")
        return self.allocate(shape, STB_F32)

    def _f32(self, *ts):
        for t in ts:
            self._validate(t)
            require(t.dtype == STB_F32 and not t.transposed_weight, "operation takes Float32 activations")

    def _run(self, out: DeviceTensor, fn: str, *args) -> DeviceTensor:
        try:
            call(fn, self.handle, *args)
        except Exception:
            self.release(out)
            raise
        return out

    def reshape(self, t: DeviceTensor, shape) -> DeviceTensor:
        """A view over the same allocation (CudaSession.reshape, CudaSession.scala:95-101): released
        independently; the memory is freed when the last handle is released."""
        self._validate(t)
        shape = tuple(int(d) for d in shape)
        n = 1
        for d in shape:
            n *= d
        require(n == t.numel, "reshape changes element count")
        t._refs[0] += 1
        return DeviceTensor(self, t.address, shape, t.dtype, t.nbytes, t.transposed_weight, t.owner, _refs=t._refs)

    def transpose(self, t: DeviceTensor, dim0: int, dim1: int) -> DeviceTensor:
        """Packed copy with two axes swapped (CudaSession.transpose, CudaSession.scala:469-485)."""
        self._f32(t)
        rank = len(t.shape)
        require(0 <= dim0 < rank and 0 <= dim1 < rank, "transpose dimension out of range")
        if dim0 == dim1:
            return self.reshape(t, t.shape)
        dims = list(t.shape)
        dims[dim0], dims[dim1] = dims[dim1], dims[dim0]
        out = self._out(dims)
        if out.numel == 0:
            return out
        arr = (ctypes.c_int64 * rank)(*t.shape)
        return self._run(out, "stb_op_transpose", t.address, out.address, rank, ctypes.cast(arr, ctypes.c_void_p),
                         dim0, dim1)

    def embedding(self, table: DeviceTensor, indices) -> DeviceTensor:
        """Rows of `table` for host int64 ids (CpuFloatBackend.embedding, CpuFloatBackend.scala:49-59); the
        output appends the table width.  A half table (the raw safetensors payload) is widened exactly."""
        self._validate(table)
        require(len(table.shape) == 2 and table.shape[1] > 0, "embedding requires a matrix with positive width")
        rows, width = table.shape
        if table.transposed_weight:  # an (out,in) half payload uploaded as a weight: rows = out
            width, rows = table.shape
        ids = np.ascontiguousarray(np.asarray(indices, np.int64))
        require(bool(np.all((ids >= 0) & (ids < rows))), "embedding token ID out of bounds")
        out = self._out(ids.shape + (width,))
        if out.numel == 0:
            return out
        return self._run(out, "stb_op_embedding", table.address, table.dtype, rows, width, ids.ctypes.data, ids.size,
                         out.address)

    def _binary(self, fn, a, b, name):
        self._f32(a, b)
        require(a.shape == b.shape, f"backend {name} requires equal shapes")
        out = self._out(a.shape)
        return self._run(out, fn, a.address, b.address, out.address, a.numel) if a.numel else out

    def add(self, a: DeviceTensor, b: DeviceTensor) -> DeviceTensor:
        return self._binary("stb_op_add", a, b, "add")

    def multiply(self, a: DeviceTensor, b: DeviceTensor) -> DeviceTensor:
        return self._binary("stb_op_multiply", a, b, "multiply")

    def scale(self, t: DeviceTensor, scalar: float) -> DeviceTensor:
        """Elementwise Float32 scalar multiplication, IEEE nonfinite values included."""
        self._f32(t)
        out = self._out(t.shape)
        return self._run(out, "stb_op_scale", t.address, out.address, t.numel, float(np.float32(scalar))) \
            if t.numel else out

    def fill(self, shape, value: float) -> DeviceTensor:
        out = self._out(tuple(int(d) for d in shape))
        return self._run(out, "stb_fill_value", out.address, STB_F32, out.numel, float(np.float32(value))) \
            if out.numel else out

    def sum(self, t: DeviceTensor) -> DeviceTensor:
        """All elements into a rank-zero Float32, accumulated in double."""
        self._f32(t)
        out = self._out(())
        return self._run(out, "stb_op_sum", t.address, t.numel, out.address)

    def expand_scalar(self, t: DeviceTensor, shape) -> DeviceTensor:
        """Repeat a rank-zero device value without a host transfer."""
        self._f32(t)
        require(len(t.shape) == 0, "expandScalar requires rank zero")
        out = self._out(tuple(int(d) for d in shape))
        return self._run(out, "stb_op_expand_scalar", t.address, out.address, out.numel) if out.numel else out

    def silu(self, t: DeviceTensor) -> DeviceTensor:
        self._f32(t)
        out = self._out(t.shape)
        return self._run(out, "stb_op_silu", t.address, out.address, t.numel) if t.numel else out

    def rms_norm(self, t: DeviceTensor, weight: DeviceTensor, epsilon: float = 1e-6) -> DeviceTensor:
        """RMSNorm over the final axis (CpuFloatBackend.rmsNorm, CpuFloatBackend.scala:78-93)."""
        self._f32(t, weight)
        require(math.isfinite(epsilon) and epsilon > 0, "invalid RMSNorm epsilon")
        require(len(t.shape) > 0 and t.shape[-1] > 0 and weight.shape == (t.shape[-1],), "invalid RMSNorm shapes")
        out = self._out(t.shape)
        width = t.shape[-1]
        return self._run(out, "stb_op_rmsnorm", t.address, weight.address, out.address, t.numel // width, width,
                         float(epsilon)) if t.numel else out

    def rope(self, t: DeviceTensor, position_start: int = 0, theta: float = 10000.0) -> DeviceTensor:
        """Rotary embedding of (batch, heads, tokens, width) (CpuAttention.rope, CpuAttention.scala:6-18)."""
        self._f32(t)
        require(len(t.shape) == 4 and t.shape[3] > 0 and t.shape[3] % 2 == 0,
                "RoPE requires rank 4 and positive even width")
        require(position_start >= 0 and math.isfinite(theta) and theta > 0, "invalid rotary position or theta")
        if t.numel == 0:
            return self.reshape(t, t.shape)
        b, h, n, w = t.shape
        out = self._out(t.shape)
        return self._run(out, "stb_op_rope", t.address, out.address, b, h, n, w, position_start, float(theta))

    def causal_attention(self, query: DeviceTensor, key: DeviceTensor, value: DeviceTensor, query_start: int = 0,
                         max_score_elements: int = 16777216) -> DeviceTensor:
        """Causal grouped-query attention (CpuAttention.causal, CpuAttention.scala:20-50) with
        AttentionLayout.validate's rules (AttentionLayout.scala:3-19)."""
        self._f32(query, key, value)
        out_shape, _ = attention_layout(query.shape, key.shape, value.shape, query_start, max_score_elements)
        return self._attend(query, key, value, out_shape, key.shape[2], key.shape[2], query_start)

    def _attend(self, q, k, v, out_shape, keys, key_stride, start):
        out = self._out(out_shape)
        if out.numel == 0:
            return out
        b, h, t, d = q.shape
        return self._run(out, "stb_op_causal_attention", q.address, k.address, v.address, out.address, b, h, t, d,
                         k.shape[1], keys, key_stride, v.shape[3], start)

    def attention_cache(self, batch_size: int, heads: int, capacity: int, key_width: int, value_width: int,
                        max_bytes: int = 268435456) -> "B200AttentionCache":
        self._check()
        return B200AttentionCache(self, batch_size, heads, capacity, key_width, value_width, max_bytes)

    # -- several requests in one batch
    # These calls are a few microseconds on the GPU: their checks are one expression per tensor on the way through, and
    # _refuse names what was wrong with it.
    def _refuse(self, *tensors) -> None:
        """tensors: (tensor, dtype, shape or None), of which one at least is not what the operator takes."""
        self._check()
        for t, dtype, shape in tensors:
            require(isinstance(t, DeviceTensor) and t.session is self, "tensor belongs to another session")
            if not t._alive[0]:
                raise IllegalStateException("validate", 6, "tensor was released")
            require(t.dtype == dtype and not t.transposed_weight, "operation takes Float32 rows and int32 indices")
            require(shape is None or t.shape == shape, f"shape mismatch: {t.shape} where {shape} is needed")
            require(t.row_stride == 0 or dtype == STB_F32 and len(t.shape) > 1,
                    "operation takes packed indices, weights and biases, not a view of columns")
        raise IllegalArgumentException("operands do not fit together")

    def _outs(self, *shapes):
        """Float32 outputs of an operator that has several; none is left behind where one does not fit."""
        made = []
        try:
            for shape in shapes:
                made.append(self._out(shape))
        except Exception:
            for t in made:
                self.release(t)
            raise
        return tuple(made)

    @_of_tensors
    def qk_norm_rope(self, query: DeviceTensor, key: DeviceTensor, query_weight: DeviceTensor | None,
                     key_weight: DeviceTensor | None, positions: DeviceTensor, epsilon: float = 1e-6,
                     theta: float = 10000.0, out=None):
        """RMSNorm of each query and key head (no norm where the weight is None) and rotary embedding of its row's
        own position, in one pass: query (rows, heads, width), key (rows, kv_heads, width), positions int32 (rows,).
        query and key may be columns of a fused projection.  Returns (query, key); out = (query, key) tensors to
        write, which may be the inputs themselves.  A row with a negative position is padding and left as it is."""
        qs, ks = getattr(query, "shape", ()), getattr(key, "shape", ())
        if len(qs) != 3 or len(ks) != 3 or qs[0] != ks[0] or qs[2] != ks[2]:
            raise IllegalArgumentException("query and key heads must have shapes (rows, heads, width)")
        rows, heads, width = qs
        made = out is None
        if made:
            self._check()
            out = self._outs(qs, ks)
        yq, yk = out
        qw, kw = query_weight, key_weight
        try:
            if not (not self._closed and query.session is self and query._alive[0] and query.dtype == STB_F32 and not query.transposed_weight
                    and key.session is self and key._alive[0] and key.dtype == STB_F32 and not key.transposed_weight
                    and positions.session is self and positions._alive[0] and positions.dtype == STB_I32
                    and positions.shape == (rows,) and positions.row_stride == 0
                    and yq.session is self and yq._alive[0] and yq.dtype == STB_F32 and yq.shape == qs and not yq.transposed_weight
                    and yk.session is self and yk._alive[0] and yk.dtype == STB_F32 and yk.shape == ks and not yk.transposed_weight
                    and (qw is None or qw.session is self and qw._alive[0] and qw.dtype == STB_F32 and qw.shape == (width,) and qw.row_stride == 0)
                    and (kw is None or kw.session is self and kw._alive[0] and kw.dtype == STB_F32 and kw.shape == (width,) and kw.row_stride == 0)):
                self._refuse((query, STB_F32, None), (key, STB_F32, None), (positions, STB_I32, (rows,)), (yq, STB_F32, qs), (yk, STB_F32, ks),
                             *[(w, STB_F32, (width,)) for w in (qw, kw) if w is not None])
            kv_heads = ks[1]
            call("stb_op_qk_norm_rope", self.handle, query.address, query.row_stride or heads * width, heads, key.address,
                 key.row_stride or kv_heads * width, kv_heads, width, rows, 0 if qw is None else qw.address,
                 0 if kw is None else kw.address, positions.address, epsilon, theta, yq.address, yq.row_stride or heads * width,
                 yk.address, yk.row_stride or kv_heads * width)
        except Exception:
            if made:
                self.release(yq)
                self.release(yk)
            raise
        return out

    def paged_cache(self, keys: DeviceTensor, values: DeviceTensor, key_scales: DeviceTensor | None = None,
                    value_scales: DeviceTensor | None = None) -> "B200PagedCache":
        """A paged cache over buffers of the caller: keys and values (pages, kv_heads, page_size, width) in Float32,
        BF16, F16 or E4M3, the last with a scale byte per (page, head, slot)."""
        return B200PagedCache(self, keys, values, key_scales, value_scales)

    def adapter_pool(self, a: DeviceTensor, b: DeviceTensor, ranks: DeviceTensor, scales: DeviceTensor) -> "AdapterPool":
        """Low-rank adapters that the rows of one call choose from (linear_adapted): a (slots, max_rank, in),
        b (slots, out, max_rank), ranks int32 (slots,), scales Float32 (slots,)."""
        return AdapterPool(self, a, b, ranks, scales)

    @_of_tensors
    def linear_adapted(self, x: DeviceTensor, weight: DeviceTensor, pool: "AdapterPool", rows: DeviceTensor,
                       bias: DeviceTensor | None = None, out: DeviceTensor | None = None) -> DeviceTensor:
        """x.W^T + scale (x.A^T).B^T + bias with row m's adapter rows[m] of the pool (int32; negative: none).  out may not
        overlap x.  A capture needs a call of this size before it."""
        require(isinstance(pool, AdapterPool) and pool.session is self, "adapter pool belongs to another session")
        M, K, N = x.shape[0] if len(x.shape) == 2 else -1, pool.inner, pool.out
        if not (not self._closed and x.session is self and x._alive[0] and x.dtype == STB_F32 and x.shape == (M, K) and not x.transposed_weight
                and x.row_stride == 0 and weight.session is self and weight._alive[0] and weight.transposed_weight
                and weight.shape == (K, N) and rows.session is self and rows._alive[0] and rows.dtype == STB_I32
                and rows.shape == (M,) and rows.row_stride == 0
                and (bias is None or bias.session is self and bias._alive[0] and bias.dtype == STB_F32 and bias.shape == (N,) and bias.row_stride == 0)):
            self._validate(x)
            self._validate(weight)
            require(weight.transposed_weight, "weight must be a resident (out,in) weight")
            require(x.dtype == STB_F32 and not x.transposed_weight, "activations must be Float32")
            require(weight.shape == (K, N), "Linear adapter shape mismatch")
            self._refuse((x, STB_F32, (M, K)), (rows, STB_I32, (M,)), *([(bias, STB_F32, (N,))] if bias is not None else []))
        pool.check()
        y = self._out((M, N)) if out is None else out
        if not (y.session is self and y._alive[0] and y.dtype == STB_F32 and y.shape == (M, N) and not y.transposed_weight and y.row_stride == 0):
            self._validate(y)
            self._refuse((y, STB_F32, (M, N)))
        try:
            call("stb_linear_pool", self.handle, x.address, weight.address, weight.dtype, 0 if bias is None else bias.address,
                 pool.ref, rows.address, y.address, M, N, K)
        except Exception:
            if out is None:
                self.release(y)
            raise
        return y

    # -- tensor parallel
    @staticmethod
    def nccl_unique_id() -> bytes:
        buf = (ctypes.c_uint8 * 128)()
        call("stb_nccl_unique_id", buf)
        return bytes(buf)

    def init_tp(self, nranks: int, rank: int, unique_id: bytes | None) -> None:
        buf = (ctypes.c_uint8 * 128)(*(unique_id or bytes(128)))
        call("stb_session_init_tp", self.handle, nranks, rank, buf)

    def allreduce_sum(self, t: DeviceTensor) -> None:
        self._validate(t)
        call("stb_allreduce_sum_f32", self.handle, t.address, t.numel)


def attention_layout(q, k, v, start: int, max_scores: int):
    """AttentionLayout.validate (core/src/main/scala/scalatorch/AttentionLayout.scala:3-19): output shape
    and score count, IllegalArgumentException on any violated rule."""
    require(len(q) == 4 and len(k) == 4 and len(v) == 4, "attention expects (batch,heads,tokens,width)")
    require(start >= 0 and max_scores >= 0, "invalid attention offset or workspace limit")
    require(q[0] == k[0] == v[0], "attention batch mismatch")
    require(q[1] > 0 and k[1] > 0 and k[1] == v[1] and q[1] % k[1] == 0, "invalid grouped attention heads")
    require(q[3] > 0 and q[3] == k[3] and v[3] > 0 and k[2] == v[2], "attention width/token mismatch")
    out = (q[0], q[1], q[2], v[3])
    require(out[0] * out[1] * out[2] * out[3] <= 0x7FFFFFFF, "attention output exceeds Int indexing")
    if q[0] * q[1] * q[2] * q[3] == 0:
        return out, 0
    require(k[2] > 0, "nonempty queries require keys")
    scores = q[0] * q[1] * q[2] * k[2]
    require(scores <= max_scores and scores <= 0x7FFFFFFF, "attention score workspace limit exceeded")
    return out, scores


class B200AttentionCache:
    """AttentionCache on the device (CudaSession.attentionCache, CudaSession.scala:397-431; CacheLayout,
    AttentionCache.scala:8-27): Float32 keys (batch, heads, capacity, key_width) and values, appended at
    a written prefix and attended in one call."""

    def __init__(self, session: B200Session, batch: int, heads: int, capacity: int, key_width: int,
                 value_width: int, max_bytes: int):
        require(batch > 0 and heads > 0 and capacity > 0 and key_width > 0 and value_width > 0 and max_bytes >= 0,
                "invalid attention cache dimensions/budget")
        kc, vc = batch * heads * capacity * key_width, batch * heads * capacity * value_width
        require(kc <= 0x7FFFFFFF and vc <= 0x7FFFFFFF and (kc + vc) * 4 <= max_bytes,
                "attention cache allocation budget exceeded")
        self.session, self.batch, self.heads, self.capacity = session, batch, heads, capacity
        self.key_width, self.value_width = key_width, value_width
        self.keys = session.allocate((batch, heads, capacity, key_width))
        try:
            self.values = session.allocate((batch, heads, capacity, value_width))
        except Exception:
            session.release(self.keys)
            raise
        self.written = 0
        self._closed = False

    def attend(self, query: DeviceTensor, key: DeviceTensor, value: DeviceTensor, position: int,
               max_score_elements: int = 16777216) -> DeviceTensor:
        s = self.session
        if self._closed:
            raise IllegalStateException("attend", 6, "attention cache is closed")
        s._f32(query, key, value)
        require(len(key.shape) == 4, "cache key must have rank 4")
        chunk = key.shape[2]
        require(chunk > 0 and key.shape == (self.batch, self.heads, chunk, self.key_width)
                and value.shape == (self.batch, self.heads, chunk, self.value_width), "cache append shape mismatch")
        require(len(query.shape) == 4 and query.shape[2] == chunk, "cache query/chunk mismatch")
        end = position + chunk
        require(0 <= position <= self.written and end <= self.capacity, "cache append gap or capacity exceeded")
        out_shape, _ = attention_layout(query.shape, (self.batch, self.heads, end, self.key_width),
                                        (self.batch, self.heads, end, self.value_width), position, max_score_elements)
        for src, dst, w in ((key, self.keys, self.key_width), (value, self.values, self.value_width)):
            call("stb_op_cache_append", s.handle, src.address, dst.address, self.batch, self.heads, chunk, w,
                 self.capacity, position)
        out = s._attend(query, self.keys, self.values, out_shape, end, self.capacity, position)
        self.written = end
        return out

    def close(self) -> None:
        if not self._closed:
            self._closed = True
            self.session.release(self.keys)
            self.session.release(self.values)


class AdapterPool:
    """Resident factors of several low-rank adapters, one slot each (stb_adapter_pool).  Slots are loaded, replaced
    and unloaded by writing the tensors between calls; a slot uses the first ranks[slot] rows of its factors."""

    def __init__(self, session: B200Session, a: DeviceTensor, b: DeviceTensor, ranks: DeviceTensor, scales: DeviceTensor):
        for t in (a, b, ranks, scales):
            session._validate(t)
        require(a.dtype in (STB_F32, STB_BF16, STB_F16) and a.dtype == b.dtype, "adapter factors must share one type")
        require(len(a.shape) == 3 and len(b.shape) == 3 and min(a.shape + b.shape) > 0 and a.shape[0] == b.shape[0]
                and a.shape[1] == b.shape[2] and a.shape[1] <= 256, "invalid adapter factor dimensions")
        require(ranks.shape == (a.shape[0],) and ranks.dtype == STB_I32, "adapter ranks must be int32 (slots,)")
        require(scales.shape == (a.shape[0],) and scales.dtype == STB_F32, "adapter scales must be Float32 (slots,)")
        self.session, self.tensors = session, (a, b, ranks, scales)
        self.slots, self.max_rank, self.inner = a.shape
        self.out = b.shape[1]
        self._struct = StbAdapterPool(a.address, b.address, ranks.address, scales.address, a.dtype, self.slots, self.max_rank)
        self.ref = ctypes.byref(self._struct)

    def check(self) -> None:
        for t in self.tensors:
            if not t._alive[0]:
                raise IllegalStateException("adapter pool", 6, "tensor was released")


class B200PagedCache:
    """Keys and values of several requests in pages (stb_paged_cache), each request at its own position: the token at
    position p of request r lies in page tables[r, p // page_size].  Beside B200AttentionCache, whose one written
    prefix serves the whole batch in Float32.  The tensors are the caller's; tables (batch, blocks), sequences, positions
    and lengths are int32 device tensors, so that a captured step can be replayed with new ones."""

    def __init__(self, session: B200Session, keys: DeviceTensor, values: DeviceTensor, key_scales=None, value_scales=None):
        scaled = [t for t in (key_scales, value_scales) if t is not None]
        for t in (keys, values, *scaled):
            session._validate(t)
        require(keys.dtype in (STB_F32, STB_BF16, STB_F16, STB_E4M3) and keys.dtype == values.dtype, "paged cache type")
        require(len(keys.shape) == 4 and min(keys.shape) > 0 and keys.shape == values.shape and keys.shape[3] <= 512,
                "invalid paged cache dimensions")
        require(len(scaled) == (2 if keys.dtype == STB_E4M3 else 0), "an E4M3 cache has scales, the other types have none")
        require(all(t.shape == keys.shape[:3] and t.dtype == STB_U8 for t in scaled),
                "paged cache scales must be bytes (pages, kv_heads, page_size)")
        self.session, self.tensors = session, (keys, values, *scaled)
        self.pages, self.kv_heads, self.page_size, self.width = keys.shape
        self.dtype = keys.dtype
        self._struct = StbPagedCache(keys.address, values.address, *([t.address for t in scaled] or [0, 0]), keys.dtype,
                                     self.pages, self.page_size, self.kv_heads, self.width)
        self.ref = ctypes.byref(self._struct)

    def _check(self) -> None:
        self.session._check()
        for t in self.tensors:
            if not t._alive[0]:
                raise IllegalStateException("paged cache", 6, "tensor was released")

    def _open(self, tables, *indices) -> None:
        """Checks the cache, the page tables and row indices of one length."""
        s = self.session
        alive = not s._closed
        for t in self.tensors:
            alive = alive and t._alive[0]
        if not (alive and tables.session is s and tables._alive[0] and tables.dtype == STB_I32 and len(tables.shape) == 2
                and tables.row_stride == 0):
            self._check()
            require(len(getattr(tables, "shape", ())) == 2, "page tables must have shape (batch, blocks)")
            s._refuse((tables, STB_I32, None))
        shape = indices[0].shape
        for t in indices:
            if not (t.session is s and t._alive[0] and t.dtype == STB_I32 and t.shape == shape and len(shape) == 1 and t.row_stride == 0):
                require(len(shape) == 1, "row indices must have shape (rows,)")
                s._refuse((t, STB_I32, shape))

    def _rows(self, t: DeviceTensor, shape) -> int:
        """Checks a Float32 tensor of this shape; elements between its rows."""
        s = self.session
        if not (t.session is s and t._alive[0] and t.dtype == STB_F32 and t.shape == shape and not t.transposed_weight):
            s._refuse((t, STB_F32, shape))
        return t.row_stride or shape[1] * shape[2]

    @_of_tensors
    def append(self, key: DeviceTensor, value: DeviceTensor, tables: DeviceTensor, sequences: DeviceTensor,
               positions: DeviceTensor) -> None:
        """Writes key and value rows (rows, kv_heads, width) at positions[r] of request sequences[r], rounded or quantised
        to the cache's type.  Rows with a negative sequence or position are padding; no two rows may name one token."""
        self._open(tables, sequences, positions)
        rows, w = sequences.shape[0], self.width
        shape = (rows, self.kv_heads, w)
        key_row, value_row = self._rows(key, shape), self._rows(value, shape)
        batch, blocks = tables.shape
        call("stb_op_paged_append", self.session.handle, self.ref, key.address, key_row, w, value.address, value_row, w, tables.address,
             batch, blocks, sequences.address, positions.address, rows)

    @_of_tensors
    def read(self, tables: DeviceTensor, sequences: DeviceTensor, positions: DeviceTensor, out=None,
             heads_first: bool = False):
        """(key, value) of the named tokens in Float32, (rows, kv_heads, width), or (kv_heads, rows, width) with
        heads_first -- causal_attention's layout for one request.  With `out` the two tensors are written, padding
        rows left as they are; without it padding rows come back as zeros."""
        self._open(tables, sequences, positions)
        s, rows, w = self.session, sequences.shape[0], self.width
        batch, blocks = tables.shape
        shape = (self.kv_heads, rows, w) if heads_first else (rows, self.kv_heads, w)
        made = out is None
        if made:
            out = s._outs(shape, shape)
        try:
            if made and out[0].numel:  # padding rows of a fresh output
                for t in out:
                    call("stb_fill_value", s.handle, t.address, STB_F32, t.numel, 0.0)
            k, v = out
            kr, vr = self._rows(k, shape), self._rows(v, shape)
            kh = vh = w
            if heads_first:
                kr, kh, vr, vh = w, kr, w, vr
            call("stb_op_paged_read", s.handle, self.ref, tables.address, batch, blocks, sequences.address, positions.address, rows,
                 k.address, kr, kh, v.address, vr, vh)
        except Exception:
            if made:
                s.release(out[0])
                s.release(out[1])
            raise
        return out

    @_of_tensors
    def attend(self, query: DeviceTensor, tables: DeviceTensor, lengths: DeviceTensor,
               out: DeviceTensor | None = None) -> DeviceTensor:
        """Attention of one new token per request: query (batch, heads, width) against the first lengths[b] tokens of
        tables[b] (the new token's own key among them: append first).  A length of zero gives a row of zeros.  out may
        not overlap the query."""
        self._open(tables, lengths)
        s, shape = self.session, query.shape
        batch, blocks = tables.shape
        require(len(shape) == 3 and shape[0] == batch == lengths.shape[0] and shape[2] == self.width and shape[1] > 0
                and shape[1] % self.kv_heads == 0, "paged attention query must have shape (batch, heads, width)")
        q_row = self._rows(query, shape)
        y = s._out(shape) if out is None else out
        try:
            call("stb_op_paged_attention", s.handle, self.ref, query.address, q_row, shape[1], tables.address, batch, blocks,
                 lengths.address, y.address, self._rows(y, shape))
        except Exception:
            if out is None:
                s.release(y)
            raise
        return y

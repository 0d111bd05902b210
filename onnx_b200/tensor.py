"""Device-resident tensors and per-GPU contexts.

``DeviceTensor`` is the device-storage counterpart of the reference's
``DenseTensor<T>`` (src/Lokad.Onnx.Tensors/DenseTensor.cs:31-278): a dense
row-major buffer plus its dimensions, living in one GPU's HBM.  Reshape is a
zero-copy view over the same buffer (DenseTensor.cs:231-242).
"""
from __future__ import annotations

import ctypes
import threading

import numpy as np

from . import _native as N

# Element types numpy has no name for: one field holding the bits (a host copy
# is read as `a.view(np.uint16)` or `a.view(np.uint8)`).
BFLOAT16 = np.dtype([("bfloat16", "<u2")])
FLOAT8E4M3 = np.dtype([("float8e4m3fn", "u1")])

ONNX_DTYPE = {np.dtype(np.float16): 10, BFLOAT16: 16, FLOAT8E4M3: 17,
              np.dtype(np.float32): 1, np.dtype(np.int64): 7, np.dtype(np.int32): 6,
              np.dtype(np.uint8): 2, np.dtype(np.bool_): 9, np.dtype(np.float64): 11}
NP_DTYPE = {v: k for k, v in ONNX_DTYPE.items()}
# what np.dtype() answers for the usual types, without its cost
_DTYPES = {**{d: d for d in ONNX_DTYPE}, **{d.type: d for d in ONNX_DTYPE if d.type is not np.void}}


class Context:
    """One GPU: device, CUDA stream and caching allocator (lonnx_ctx).  Calls
    leave its device as the thread's current one: a program with tensors of
    another library on several devices names their device, or sets it again."""

    _default = {}
    _lock = threading.Lock()

    def __init__(self, device: int = 0, stream: int | None = None):
        """``stream``: a CUDA stream of the caller's (its handle, 0 the default
        stream) to run on and to be ordered with; None makes one."""
        h = ctypes.c_void_p()
        if stream is None:
            N.check(N.lib.lonnx_ctx_create(device, ctypes.byref(h)))
        else:
            N.check(N.lib.lonnx_ctx_create_on_stream(device, stream, ctypes.byref(h)))
        self.handle = h
        self.device = device

    @classmethod
    def default(cls, device: int = 0) -> "Context":
        with cls._lock:
            if device not in cls._default:
                cls._default[device] = cls(device)
            return cls._default[device]

    def sync(self):
        N.check(N.lib.lonnx_sync(self.handle))

    @property
    def launches(self) -> int:
        return int(N.lib.lonnx_launch_count(self.handle))

    @property
    def stream(self) -> int:
        return int(N.lib.lonnx_ctx_stream(self.handle) or 0)

    def close(self):
        if self.handle:
            N.lib.lonnx_ctx_destroy(self.handle)
            self.handle = None


class _Allocation:
    """Memory of a context's allocator, given back with its last tensor."""

    def __init__(self, ctx: Context, nbytes: int):
        p = ctypes.c_void_p()
        N.check(N.lib.lonnx_malloc(ctx.handle, max(nbytes, 1), ctypes.byref(p)))
        self.ctx, self.ptr = ctx, p.value

    def __del__(self):
        try:
            if self.ptr and self.ctx.handle:
                N.lib.lonnx_free(self.ctx.handle, self.ptr)
        except Exception:
            pass


class DeviceTensor:
    """A dense tensor in device memory (float32 activations, int64 indices)."""

    name = None

    def __init__(self, ctx: Context, shape, dtype, ptr=None, owner=None):
        self.ctx = ctx
        self.shape = tuple(map(int, shape))
        self.dtype = _DTYPES.get(dtype) or np.dtype(dtype)
        if ptr is None:
            owner = _Allocation(ctx, self.nbytes)
            ptr = owner.ptr
        self.ptr = ptr
        self._owner = owner

    @property
    def size(self) -> int:
        return int(np.prod(self.shape)) if self.shape else 1

    @property
    def nbytes(self) -> int:
        return self.size * self.dtype.itemsize

    @property
    def rank(self) -> int:
        return len(self.shape)

    @classmethod
    def from_host(cls, ctx: Context, arr) -> "DeviceTensor":
        a = np.ascontiguousarray(arr)
        t = cls(ctx, a.shape, a.dtype)
        if a.nbytes:
            N.check(N.lib.lonnx_memcpy_h2d(ctx.handle, t.ptr, a.ctypes.data, a.nbytes))
            # pageable source: the copy is staged before returning, but keep the
            # array alive until the stream has consumed it
            t._host_ref = a
        return t

    def to_host(self) -> np.ndarray:
        out = np.empty(self.shape, self.dtype)
        if out.nbytes:
            N.check(N.lib.lonnx_memcpy_d2h(self.ctx.handle, out.ctypes.data, self.ptr, out.nbytes))
        return out

    def reshape(self, *shape) -> "DeviceTensor":
        if len(shape) == 1 and isinstance(shape[0], (tuple, list)):
            shape = tuple(shape[0])
        shape = list(shape)
        if -1 in shape:
            known = int(np.prod([s for s in shape if s != -1]))
            shape[shape.index(-1)] = self.size // known
        if int(np.prod(shape)) != self.size:
            raise ValueError(f"cannot reshape {self.shape} to {tuple(shape)}")
        return DeviceTensor(self.ctx, shape, self.dtype, ptr=self.ptr, owner=self)

    def __repr__(self):
        return f"DeviceTensor(shape={self.shape}, dtype={self.dtype}, device={self.ctx.device})"

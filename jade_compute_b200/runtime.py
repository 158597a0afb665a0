"""Python host mirror of the reference's runtime contract over the C ABI.

The reference's Rust host (src/runtime/mod.rs:45-61 ``trait Runtime``;
src/runtime/corex.rs:335-613 ``impl Runtime for CorexRuntime``) owns buffers,
performs exact transfers, compiles validated KernelSpecs and executes ordered
batches. This module exposes the same operations (``info``, ``alloc``,
``upload``, ``download``, ``compile``, ``execute``) with the same argument
meaning and error behaviour, calling ``libjade_runtime.so`` through ctypes.
There is no CPU fallback: if the CUDA library is missing, importing the
runtime raises.
"""
from __future__ import annotations

import ctypes
import json
import os
import time
import weakref
from array import array
from dataclasses import dataclass, field
from typing import Iterable, Sequence

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
# JADE_RUNTIME_LIBRARY selects another build of this library (e.g. a variant
# compiled with different options); by default the in-tree build.
LIB_PATH = os.environ.get("JADE_RUNTIME_LIBRARY") or os.path.join(HERE, "lib", "libjade_runtime.so")
INCLUDE = os.path.join(os.path.dirname(HERE), "include", "jade_runtime.h")

JR_OK, JR_EINVAL, JR_ECUDA, JR_ENOMEM, JR_ETIMEOUT = 0, 1, 2, 3, 4
JR_EXEC_GRAPH = 1
JR_EXEC_STREAMS = 2
JR_EXEC_DEFER_MS = 4
JR_EXEC_HOLD_MS = 8

DTYPE_SIZE = {"fp32": 4, "tf32": 4, "bf16": 2, "fp16": 2, "u8": 1, "i32": 4}
NP_DTYPE = {"fp32": np.float32, "tf32": np.float32, "bf16": np.uint16, "fp16": np.float16, "u8": np.uint8, "i32": np.int32}


class JadeError(RuntimeError):
    """Error returned by the native runtime; ``code`` is the jr_* error code."""

    def __init__(self, code: int, message: str):
        super().__init__(f"Jade runtime error {code}: {message}")
        self.code = code
        self.message = message


_lib = None


def library_path() -> str:
    return LIB_PATH


def lib() -> ctypes.CDLL:
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise ImportError(f"{LIB_PATH} is missing: build the CUDA extension first (__graft_entry__.build())")
    L = ctypes.CDLL(LIB_PATH, mode=ctypes.RTLD_GLOBAL)
    c_char_p, sz, vp, i32, u32 = ctypes.c_char_p, ctypes.c_size_t, ctypes.c_void_p, ctypes.c_int, ctypes.c_uint32
    u64p = ctypes.POINTER(ctypes.c_uint64)
    L.jr_version.restype = u32
    L.jr2_version.restype = u32
    L.jr_device_count.restype = i32
    L.jr_create.argtypes = [i32, ctypes.POINTER(vp), c_char_p, sz]
    L.jr_destroy.argtypes = [vp]
    L.jr_destroy.restype = None
    L.jr_info.argtypes = [vp, c_char_p, sz, c_char_p, sz]
    L.jr_alloc.argtypes = [vp, sz, ctypes.POINTER(vp), c_char_p, sz]
    L.jr_free.argtypes = [vp, vp]
    L.jr_free.restype = None
    L.jr_upload.argtypes = [vp, vp, vp, sz, c_char_p, sz]
    L.jr_download.argtypes = [vp, vp, vp, sz, c_char_p, sz]
    L.jr_execute.argtypes = [vp, vp, sz, u32, ctypes.POINTER(ctypes.c_double), c_char_p, sz]
    L.jr_spec_validate.argtypes = [c_char_p, c_char_p, sz]
    L.jr_spec_bindings.argtypes = [c_char_p, c_char_p, sz, c_char_p, sz]
    L.jr_spec_validate_bindings.argtypes = [c_char_p, u64p, u64p, sz, c_char_p, sz]
    L.jr_spec_launch.argtypes = [c_char_p, c_char_p, sz, c_char_p, sz]
    L.jr_spec_emit.argtypes = [c_char_p, c_char_p, c_char_p, sz, ctypes.POINTER(sz), c_char_p, sz]
    L.jr_spec_canonical.argtypes = [c_char_p, c_char_p, sz, c_char_p, sz]
    L.jr_compile.argtypes = [vp, c_char_p, ctypes.POINTER(vp), c_char_p, sz]
    L.jr_kernel_release.argtypes = [vp]
    L.jr_kernel_release.restype = None
    L.jr_kernel_info.argtypes = [vp, c_char_p, sz, c_char_p, sz]
    L.jr_execute2.argtypes = [vp, vp, sz, u32, u32, ctypes.POINTER(ctypes.c_double),
                              ctypes.POINTER(ctypes.c_double), c_char_p, sz]
    L.jr_batch_ms.argtypes = [vp, ctypes.POINTER(ctypes.c_double), c_char_p, sz]
    L.jr_held_ms.argtypes = [vp, ctypes.POINTER(ctypes.c_double), c_char_p, sz]
    L.jr_buffer_bytes.argtypes = [vp, vp, ctypes.POINTER(sz)]
    L.jr_host_alloc.argtypes = [vp, sz, ctypes.POINTER(vp), c_char_p, sz]
    L.jr_host_free.argtypes = [vp, vp]
    L.jr_host_free.restype = None
    L.jr_comm_unique_id.argtypes = [ctypes.c_char_p, c_char_p, sz]
    L.jr_comm_init.argtypes = [vp, i32, i32, ctypes.c_char_p, u32, c_char_p, sz]
    L.jr_comm_init_all.argtypes = [ctypes.POINTER(vp), i32, u32, c_char_p, sz]
    L.jr_comm_destroy.argtypes = [vp]
    L.jr_peer_handle.argtypes = [vp, vp, ctypes.c_char_p, c_char_p, sz]
    L.jr_peer_attach.argtypes = [vp, vp, ctypes.c_char_p, i32, i32, c_char_p, sz]
    _lib = L
    return L


def _err():
    return ctypes.create_string_buffer(1024)


def _check(rc: int, err) -> None:
    if rc != JR_OK:
        raise JadeError(rc, err.value.decode(errors="replace"))


def _spec_text(spec) -> bytes:
    if isinstance(spec, (bytes, bytearray)):
        return bytes(spec)
    if isinstance(spec, str):
        return spec.encode()
    return json.dumps(spec).encode()


# ---------------------------------------------------------------- IR front end
def device_count() -> int:
    return lib().jr_device_count()


def spec_validate(spec) -> None:
    e = _err()
    _check(lib().jr_spec_validate(_spec_text(spec), e, len(e)), e)


def spec_bindings(spec) -> list:
    e, out = _err(), ctypes.create_string_buffer(1 << 16)
    _check(lib().jr_spec_bindings(_spec_text(spec), out, len(out), e, len(e)), e)
    return json.loads(out.value)


def spec_validate_bindings(spec, lengths: Sequence[int], ids: Sequence[int]) -> None:
    e = _err()
    n = len(lengths)
    L = (ctypes.c_uint64 * max(n, 1))(*lengths)
    I = (ctypes.c_uint64 * max(len(ids), 1))(*ids)
    if len(ids) != n:
        raise JadeError(JR_EINVAL, "lengths and ids differ in count")
    _check(lib().jr_spec_validate_bindings(_spec_text(spec), L, I, n, e, len(e)), e)


def spec_launch(spec) -> dict:
    e, out = _err(), ctypes.create_string_buffer(4096)
    _check(lib().jr_spec_launch(_spec_text(spec), out, len(out), e, len(e)), e)
    return json.loads(out.value)


def emit(spec, target: str = "corex") -> str:
    e = _err()
    need = ctypes.c_size_t(0)
    out = ctypes.create_string_buffer(1 << 16)
    rc = lib().jr_spec_emit(_spec_text(spec), target.encode(), out, len(out), ctypes.byref(need), e, len(e))
    if rc != JR_OK and need.value > len(out):
        out = ctypes.create_string_buffer(need.value)
        rc = lib().jr_spec_emit(_spec_text(spec), target.encode(), out, len(out), ctypes.byref(need), e, len(e))
    _check(rc, e)
    return out.value.decode()


def canonical(spec) -> str:
    e, out = _err(), ctypes.create_string_buffer(1 << 16)
    _check(lib().jr_spec_canonical(_spec_text(spec), out, len(out), e, len(e)), e)
    return out.value.decode()


# ---------------------------------------------------------------- bf16 helpers
def f32_to_bf16(x) -> np.ndarray:
    """Round-to-nearest-even FP32 -> BF16 bit patterns (uint16)."""
    b = np.ascontiguousarray(x, dtype=np.float32).view(np.uint32)
    nan = (b & 0x7F800000) == 0x7F800000
    nan &= (b & 0x7FFFFF) != 0
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    r[nan] = ((b[nan] >> 16) | 0x40).astype(np.uint16)
    return r


def bf16_to_f32(h) -> np.ndarray:
    return (np.ascontiguousarray(h, dtype=np.uint16).astype(np.uint32) << 16).view(np.float32)


# ---------------------------------------------------------------- objects
@dataclass
class Buffer:
    """Owned device (or pinned host) allocation. ``elements`` counts ``dtype`` items."""
    runtime: "Runtime"
    ptr: int
    nbytes: int
    dtype: str
    host: bool = False
    freed: bool = False

    @property
    def elements(self) -> int:
        return self.nbytes // DTYPE_SIZE[self.dtype]

    def __len__(self) -> int:
        return self.elements

    def free(self) -> None:
        if not self.freed and self.runtime.ctx:
            (lib().jr_host_free if self.host else lib().jr_free)(self.runtime.ctx, self.ptr)
        self.freed = True

    def host_view(self) -> np.ndarray:
        """numpy view of a pinned host buffer."""
        if not self.host:
            raise JadeError(JR_EINVAL, "not a host buffer")
        raw = (ctypes.c_uint8 * self.nbytes).from_address(self.ptr)
        return np.frombuffer(raw, dtype=NP_DTYPE[self.dtype])


@dataclass
class Kernel:
    runtime: "Runtime"
    handle: int
    spec: dict
    info: dict = field(default_factory=dict)

    def release(self) -> None:
        if self.handle:
            lib().jr_kernel_release(self.handle)
            self.handle = 0


@dataclass
class Execution:
    """src/runtime/mod.rs:23-30 plus per-job device times. ``gpu_ms`` of a batch that has
    run is read from the device when it is asked for, or before the runtime's next batch
    at the latest."""
    host_ms: float
    gpu_ms: float | None
    dispatches: int
    repeats: int
    job_ms: list | None = None

    # Runtime.execute leaves gpu_ms unset and adds _runtime, a weak reference
    def __getattr__(self, name):  # of attributes not set: gpu_ms that has not been read
        if name != "gpu_ms" or "_runtime" not in self.__dict__:
            raise AttributeError(name)
        runtime = self._runtime()
        if runtime is None:
            raise JadeError(JR_EINVAL, "the batch's runtime is gone")
        self.gpu_ms = runtime._held_ms()
        return self.gpu_ms

    def __getstate__(self):
        self.gpu_ms
        return {k: v for k, v in self.__dict__.items() if k != "_runtime"}


class _Dispatch(ctypes.Structure):
    """jr_dispatch, for direct calls of jr_execute2 (execute packs the same words)."""
    _fields_ = [("kernel", ctypes.c_void_p), ("buffers", ctypes.POINTER(ctypes.c_void_p)), ("buffer_count", ctypes.c_size_t)]


class Runtime:
    """One device context: a stream, timing events, owned buffers and kernels."""

    def __init__(self, device: int = 0):
        L = lib()
        if L.jr_version() != 1 or L.jr2_version() != 2:
            raise JadeError(JR_EINVAL, "unsupported native runtime ABI")
        e = _err()
        h = ctypes.c_void_p()
        _check(L.jr_create(device, ctypes.byref(h), e, len(e)), e)
        self.ctx = h.value
        self.device = device
        out = ctypes.create_string_buffer(2048)
        _check(L.jr_info(self.ctx, out, len(out), e, len(e)), e)
        self.device_info = out.value.decode()
        self._kernels: list[Kernel] = []
        self._message = _err()  # of execute (a context is used serially)
        self._self = weakref.ref(self)
        self._last = None  # weak reference to the last batch's Execution, and its attributes

    # -- lifetime
    def close(self) -> None:
        if self.ctx:
            try:
                self._settle(closing=True)
            except JadeError:
                pass  # a context that has failed has no time to give
            for k in self._kernels:
                k.release()
            lib().jr_destroy(self.ctx)
            self.ctx = None

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def info(self) -> dict:
        """src/runtime/mod.rs:15-21 RuntimeInfo."""
        return {"backend": "CUDA sm_100a built-in kernels", "device": self.device_info,
                "execution": "ordered launches on one persistent non-blocking stream; optional CUDA-graph replay",
                "limitations": ["synchronous API at the public boundary",
                                "FP32, TF32, BF16 and FP16 buffers only"]}

    # -- memory
    def alloc(self, elements: int, dtype: str = "fp32") -> Buffer:
        if elements <= 0:
            raise JadeError(JR_EINVAL, "buffer allocation must be nonempty")
        return self.alloc_bytes(elements * DTYPE_SIZE[dtype], dtype)

    def alloc_bytes(self, nbytes: int, dtype: str = "u8") -> Buffer:
        e = _err()
        p = ctypes.c_void_p()
        _check(lib().jr_alloc(self.ctx, nbytes, ctypes.byref(p), e, len(e)), e)
        return Buffer(self, p.value, nbytes, dtype)

    def host_alloc(self, elements: int, dtype: str = "fp32") -> Buffer:
        e = _err()
        p = ctypes.c_void_p()
        nbytes = elements * DTYPE_SIZE[dtype]
        _check(lib().jr_host_alloc(self.ctx, nbytes, ctypes.byref(p), e, len(e)), e)
        return Buffer(self, p.value, nbytes, dtype, host=True)

    def _own(self, buf: Buffer) -> None:
        if buf.runtime is not self:
            raise JadeError(JR_EINVAL, "buffer belongs to another runtime/device context")
        if buf.freed:
            raise JadeError(JR_EINVAL, "buffer was freed")

    def upload(self, buf: Buffer, data) -> None:
        """Exact transfer: element count must match the buffer (corex.rs:389-411)."""
        self._own(buf)
        arr = np.ascontiguousarray(data, dtype=NP_DTYPE[buf.dtype]).ravel()
        if arr.size != buf.elements:
            raise JadeError(JR_EINVAL, "upload element count must match buffer exactly")
        e = _err()
        _check(lib().jr_upload(self.ctx, buf.ptr, arr.ctypes.data, buf.nbytes, e, len(e)), e)

    def download(self, buf: Buffer, start: int = 0, count: int | None = None) -> np.ndarray:
        """Elements [start, start+count) of a buffer (all of it by default)."""
        self._own(buf)
        count = buf.elements - start if count is None else count
        if start < 0 or count < 1 or start + count > buf.elements:
            raise ValueError(f"range [{start}, {start + count}) outside a buffer of {buf.elements} elements")
        out = np.empty(count, dtype=NP_DTYPE[buf.dtype])
        size = out.itemsize
        e = _err()
        _check(lib().jr_download(self.ctx, buf.ptr + start * size, out.ctypes.data, count * size, e, len(e)), e)
        return out

    def download_f32(self, buf: Buffer, start: int = 0, count: int | None = None) -> np.ndarray:
        out = self.download(buf, start, count)
        if buf.dtype == "bf16":
            return bf16_to_f32(out)
        return out.astype(np.float32)

    # -- kernels
    def compile(self, spec) -> Kernel:
        e = _err()
        h = ctypes.c_void_p()
        text = _spec_text(spec)
        _check(lib().jr_compile(self.ctx, text, ctypes.byref(h), e, len(e)), e)
        out = ctypes.create_string_buffer(1 << 16)
        lib().jr_kernel_info(h.value, out, len(out), e, len(e))
        k = Kernel(self, h.value, json.loads(text), json.loads(out.value or b"{}"))
        self._kernels.append(k)
        return k

    def execute(self, jobs: Iterable, repeats: int = 1, graph: bool = False, per_job: bool = False,
                streams: bool = False) -> Execution:
        """Ordered batch (corex.rs:544-612): every job is validated before any is
        launched; the sequence is replayed ``repeats`` times; returns host and
        device times. ``jobs`` holds (Kernel, [Buffer, ...]) pairs. ``streams``
        (JR_EXEC_STREAMS) runs transfer jobs on their own streams, ordered only by
        the data dependencies of their bindings."""
        jobs = list(jobs)
        if not jobs or repeats <= 0:
            raise JadeError(JR_EINVAL, "execution requires jobs and positive repeats")
        # jr_dispatch records as machine words (kernel, buffer array, count): ctypes
        # structures and pointer arrays cost several times as much host time per call
        words, arrays = array("Q"), []
        for kernel, bufs in jobs:
            if kernel.runtime is not self:
                raise JadeError(JR_EINVAL, "kernel belongs to another runtime/device context")
            for b in bufs:
                if b.freed or b.runtime is not self:
                    self._own(b)  # raises
            arrays.append(array("Q", [b.ptr for b in bufs]))
            words.extend((kernel.handle, arrays[-1].buffer_info()[0], len(bufs)))
        e = self._message
        gpu = ctypes.c_double(0)
        jm = (ctypes.c_double * len(jobs))() if per_job else None
        flags = (JR_EXEC_GRAPH if graph else 0) | (JR_EXEC_STREAMS if streams else 0) | JR_EXEC_DEFER_MS | JR_EXEC_HOLD_MS
        self._settle()
        t0 = time.perf_counter()
        rc = lib().jr_execute2(self.ctx, words.buffer_info()[0], len(jobs), repeats, flags, ctypes.byref(gpu), jm, e, len(e))
        host_ms = (time.perf_counter() - t0) * 1e3
        if rc != JR_OK:
            _check(rc, e)
        done = Execution.__new__(Execution)
        done.__dict__ = known = {"host_ms": host_ms, "dispatches": len(jobs) * repeats, "repeats": repeats,
                                 "job_ms": list(jm) if per_job else None, "_runtime": self._self}
        self._last = weakref.ref(done), known
        return done

    def _held_ms(self) -> float | None:
        e, ms = _err(), ctypes.c_double(0)
        _check(lib().jr_held_ms(self.ctx, ctypes.byref(ms), e, len(e)), e)
        return ms.value if ms.value > 0 else None

    def _settle(self, closing: bool = False) -> None:
        """Reads the last batch's time if its Execution is still held (when the runtime is
        collected as garbage its weak references are already cleared: read in any case)."""
        if self._last is None:
            return
        (held, attributes), self._last = self._last, None
        if (closing or held() is not None) and "gpu_ms" not in attributes:
            attributes["gpu_ms"] = self._held_ms()

    # -- conveniences used by tests and benches
    def fill(self, buf: Buffer, dist: str, seed: int, stream: int = 0, lo: float = 0.0, hi: float = 1.0,
             offset: int = 0) -> None:
        """Counter-based synthetic input: uniform [lo, hi) or normal(mean=lo, std=hi).
        ``offset``: the generator index of element 0, so that a buffer can hold a
        slice [offset, offset + len) of a larger generated tensor."""
        spec = {"op": "fill", "len": buf.elements, "dist": dist, "seed": seed, "stream": stream, "lo": lo, "hi": hi,
                "dtype": buf.dtype if buf.dtype != "tf32" else "fp32"}
        if offset:
            spec["offset"] = offset
        k = self.compile(spec)
        self.execute([(k, [buf])])
        k.release()
        self._kernels.remove(k)

    # -- peer memory (collectives over NVLink without NCCL)
    def peer_handle(self, buf: Buffer) -> bytes:
        """The 64-byte CUDA IPC handle of a device buffer, for the other ranks."""
        self._own(buf)
        out = ctypes.create_string_buffer(64)
        e = _err()
        _check(lib().jr_peer_handle(self.ctx, buf.ptr, out, e, len(e)), e)
        return out.raw

    def peer_attach(self, buf: Buffer, handles: Sequence[bytes], rank: int) -> None:
        """Maps every other rank's counterpart of `buf` (handles in rank order)."""
        self._own(buf)
        blob = b"".join(handles)
        e = _err()
        _check(lib().jr_peer_attach(self.ctx, buf.ptr, blob, len(handles), rank, e, len(e)), e)

    # -- collectives
    def comm_init(self, nranks: int, rank: int, unique_id: bytes, timeout_ms: int = 60000) -> None:
        e = _err()
        _check(lib().jr_comm_init(self.ctx, nranks, rank, unique_id, timeout_ms, e, len(e)), e)

    def comm_destroy(self) -> None:
        lib().jr_comm_destroy(self.ctx)


def comm_unique_id() -> bytes:
    e = _err()
    buf = ctypes.create_string_buffer(128)
    _check(lib().jr_comm_unique_id(buf, e, len(e)), e)
    return buf.raw


def comm_init_all(runtimes: Sequence[Runtime], timeout_ms: int = 60000) -> None:
    e = _err()
    arr = (ctypes.c_void_p * len(runtimes))(*[r.ctx for r in runtimes])
    _check(lib().jr_comm_init_all(arr, len(runtimes), timeout_ms, e, len(e)), e)

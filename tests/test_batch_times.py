"""Execution as a value, and batch times that are read after later batches of the same context."""
import copy
import ctypes
import dataclasses
import gc
import pickle
import weakref

import pytest

import jade_compute_b200 as jc


def test_execution_is_a_dataclass():
    e = jc.Execution(1.5, 0.25, 6, 3)
    assert e == jc.Execution(1.5, 0.25, 6, 3, None) and e != jc.Execution(1.5, None, 6, 3)
    assert dataclasses.asdict(e) == {"host_ms": 1.5, "gpu_ms": 0.25, "dispatches": 6, "repeats": 3, "job_ms": None}
    assert repr(e) == "Execution(host_ms=1.5, gpu_ms=0.25, dispatches=6, repeats=3, job_ms=None)"
    assert dataclasses.replace(e, gpu_ms=None, job_ms=[1.0]).job_ms == [1.0]
    assert [f.name for f in dataclasses.fields(e)] == ["host_ms", "gpu_ms", "dispatches", "repeats", "job_ms"]
    e.gpu_ms = 2.0
    assert e.gpu_ms == 2.0 and pickle.loads(pickle.dumps(e)) == e
    with pytest.raises(AttributeError):
        e.something


class Batch:
    """A batch whose device time goes with its repeats, and ways to run it through the C ABI."""

    def __init__(self):
        self.rt = jc.Runtime(0)
        self.kernel = self.rt.compile({"op": "l2_flush", "bytes": 1 << 28})
        self.buf = self.rt.alloc_bytes(1 << 28)

    def run(self, repeats):
        return self.rt.execute([(self.kernel, [self.buf])], repeats=repeats)

    def run_c(self, repeats, flags=0):
        from jade_compute_b200.runtime import _Dispatch
        buffers = (ctypes.c_void_p * 1)(self.buf.ptr)
        job = (_Dispatch * 1)()
        job[0].kernel, job[0].buffers, job[0].buffer_count = self.kernel.handle, ctypes.cast(buffers, ctypes.POINTER(ctypes.c_void_p)), 1
        ms, e = ctypes.c_double(0), ctypes.create_string_buffer(512)
        assert jc.lib().jr_execute2(self.rt.ctx, job, 1, repeats, flags, ctypes.byref(ms), None, e, 512) == 0, e.value
        return ms.value

    def last_ms(self):
        ms, e = ctypes.c_double(0), ctypes.create_string_buffer(512)
        rc = jc.lib().jr_batch_ms(self.rt.ctx, ctypes.byref(ms), e, 512)
        return rc, ms.value


@pytest.fixture
def batch():
    b = Batch()
    b.run(2)
    yield b
    b.rt.close()


@pytest.mark.gpu
def test_time_outlives_batches_of_the_c_abi(batch):
    long = batch.run(40)
    short = batch.run_c(1)
    assert short > 0 and long.gpu_ms > 10 * short
    long, other = batch.run(40), batch.run(1)
    for _ in range(3):
        batch.run_c(2)
    assert other.gpu_ms > 0 and long.gpu_ms > 10 * other.gpu_ms


@pytest.mark.gpu
def test_time_outlives_a_launch_function_batch(batch):
    launches = []

    @ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, ctypes.POINTER(ctypes.c_void_p))
    def nothing(stream, buffers):
        launches.append(stream)
        return 0

    class Job(ctypes.Structure):
        _fields_ = [("launch", ctypes.c_void_p), ("buffers", ctypes.POINTER(ctypes.c_void_p)), ("count", ctypes.c_size_t)]

    long = batch.run(40)
    buffers = (ctypes.c_void_p * 1)(batch.buf.ptr)
    job = (Job * 1)(Job(ctypes.cast(nothing, ctypes.c_void_p), ctypes.cast(buffers, ctypes.POINTER(ctypes.c_void_p)), 1))
    ms, e = ctypes.c_double(0), ctypes.create_string_buffer(512)
    L = jc.lib()
    L.jr_execute.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_uint32, ctypes.POINTER(ctypes.c_double), ctypes.c_char_p, ctypes.c_size_t]
    assert L.jr_execute(batch.rt.ctx, job, 1, 1, ctypes.byref(ms), e, 512) == 0, e.value
    assert len(launches) == 1
    rc, last = batch.last_ms()  # the context's last batch is that one
    assert rc == 0 and last == ms.value
    assert long.gpu_ms > 10 * ms.value


@pytest.mark.gpu
def test_time_outlives_deferred_batches_of_the_c_abi(batch):
    from jade_compute_b200.runtime import JR_EXEC_DEFER_MS
    held = batch.run(40)
    for _ in range(100):  # deferred ones that nobody asks for
        assert batch.run_c(1, JR_EXEC_DEFER_MS) == 0.0
    rc, last = batch.last_ms()
    assert rc == 0 and last > 0 and held.gpu_ms > 10 * last


@pytest.mark.gpu
def test_copies_and_pickles_hold_the_time(batch):
    long = batch.run(40)
    again, kept = copy.copy(long), pickle.loads(pickle.dumps(long))
    batch.run(1)
    assert again == long == kept and long.gpu_ms == again.gpu_ms == kept.gpu_ms > 0


@pytest.mark.gpu
def test_unread_execution_does_not_keep_its_runtime():
    b = Batch()
    done, gone = b.run(5), weakref.ref(b.rt)
    del b
    gc.collect()
    assert gone() is None
    assert done.gpu_ms > 0

"""Calls from several threads: those on one stream are issued one behind the other, those on different streams do not wait for each
other's.  The library's entry point is replaced by a function that stays inside until it is told to return, as a launch does whose
stream takes no more work."""
import ctypes
import threading

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture
def entered():
    """Binds a copy_pages of Python; yields (a semaphore it releases on entry, an event it waits for)."""
    from nanovllm_jax_b200 import _lib
    native = _lib.binding()
    inside, leave = threading.Semaphore(0), threading.Event()
    result, args = _lib.SIGNATURES["nvllm_b200_copy_pages"]

    def fake(*_):
        inside.release()
        leave.wait(20)
        return 0

    held = ctypes.CFUNCTYPE(result, *args)(fake)
    table = {name: ctypes.cast(getattr(_lib.load(), name), ctypes.c_void_p).value for name in _lib.SIGNATURES}
    native.bind({**table, "nvllm_b200_copy_pages": ctypes.cast(held, ctypes.c_void_p).value}, _lib.check)
    yield inside, leave
    leave.set()
    native.bind(table, _lib.check)


def start(stream):
    import torch
    from nanovllm_jax_b200 import ops
    cache = torch.zeros((2, 64, 4), device="cuda")
    src, dst = (torch.tensor([i], dtype=torch.int32, device="cuda") for i in (0, 1))

    def run():
        with torch.cuda.stream(stream):
            ops.copy_pages([cache], src, dst, 64)

    t = threading.Thread(target=run, daemon=True)
    t.start()
    return t


def test_a_thread_does_not_wait_for_another_stream(entered):
    import torch
    inside, leave = entered
    threads = [start(torch.cuda.Stream())]
    assert inside.acquire(timeout=10)
    threads.append(start(torch.cuda.Stream()))
    assert inside.acquire(timeout=5), "a call on another stream waits for the one that is inside"
    leave.set()
    for t in threads:
        t.join(10)
        assert not t.is_alive()


def test_calls_on_one_stream_are_issued_one_behind_the_other(entered):
    import torch
    inside, leave = entered
    stream = torch.cuda.Stream()
    threads = [start(stream) for _ in range(2)]
    assert inside.acquire(timeout=10)
    assert not inside.acquire(timeout=1)
    leave.set()
    assert inside.acquire(timeout=10)
    for t in threads:
        t.join(10)
        assert not t.is_alive()

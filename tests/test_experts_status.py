"""The words that the expert operators' kernels report failures to: what is decided on the host (no GPU needed)."""

import threading

import pytest
import torch

from einjax_b200 import _lib as L
from einjax_b200 import sparse


@pytest.fixture
def status(monkeypatch):
    """Status words in pageable memory, and the devices that were waited for."""
    zeros = torch.zeros
    made = []

    def host_zeros(*args, pin_memory=False, **kw):
        made.append(zeros(*args, **kw))
        return made[-1]

    waited = []
    monkeypatch.setattr(sparse.torch, "zeros", host_zeros)
    monkeypatch.setattr(sparse.torch.cuda, "synchronize", waited.append)
    words = sparse._StatusWords()
    words.made, words.waited = made, waited
    return words


def fail(address, code):
    """What a kernel does."""
    import ctypes
    ctypes.c_int32.from_address(address).value = code


def test_first_calls_of_two_threads_share_a_word(status, monkeypatch):
    host_zeros = sparse.torch.zeros
    both = threading.Barrier(2)

    def slow_zeros(*args, **kw):  # lets the other thread come as far, if it can
        try:
            both.wait(0.5)
        except threading.BrokenBarrierError:
            pass
        return host_zeros(*args, **kw)

    monkeypatch.setattr(sparse.torch, "zeros", slow_zeros)
    got = []
    threads = [threading.Thread(target=lambda: got.append(status.address("es_grouped_matmul", 0))) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(got) == 2 and got[0] == got[1] == status.address("es_grouped_matmul", 1)
    fail(got[0], L.ES_ERR_TIMEOUT)
    with pytest.raises(L.EinsparseError, match="es_grouped_matmul"):
        status.flush()


def test_every_failure_is_raised_once(status):
    fail(status.address("es_int8_matmul", 0), L.ES_ERR_TIMEOUT)
    fail(status.address("es_expert_plan", 0), L.ES_ERR_INDEX)
    raised = []
    for _ in range(2):
        with pytest.raises((ValueError, L.EinsparseError)) as e:
            status.flush()
        raised.append(type(e.value))
    assert set(raised) == {ValueError, L.EinsparseError}
    status.flush()


def test_flush_while_threads_call(status):
    """Devices and operators that come up during a flush disturb it in nothing."""
    stop = threading.Event()
    errors = []

    def calls():
        try:
            while not stop.is_set():
                for d in range(64):
                    for fn in ("es_expert_plan", "es_grouped_matmul", "es_grouped_matmul_wgrad", "es_int8_matmul"):
                        status.address(fn, d)
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=calls) for _ in range(2)]
    for t in threads:
        t.start()
    try:
        for _ in range(20):
            status.flush()
    finally:
        stop.set()
        for t in threads:
            t.join()
    assert not errors


def test_devices_are_waited_for_again(status):
    """A replay of a captured call names no device."""
    status.address("es_grouped_matmul", 1)
    status.address("es_expert_plan", 3)
    for _ in range(2):
        status.waited.clear()
        status.flush()
        assert sorted(status.waited) == [1, 3]

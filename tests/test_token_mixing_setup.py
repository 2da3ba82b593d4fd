"""The first token-mixing call of a process: what other threads see while it sets
the binding up, and what is left when that fails."""
import threading

import pytest
import torch

import mcv_b200


def call():
    x = torch.zeros(3, 2, 64).half()
    mcv_b200.mrope(x, torch.zeros(1, 3, dtype=torch.int32), mcv_b200.MRope(64, [32]), torch.zeros_like(x))


@pytest.fixture
def fresh(monkeypatch):
    """The binding as it is before the first call."""
    mcv_b200.lib()
    for name in ("_torch", "_f16_rows", "_dense", "_rows_out"):
        monkeypatch.setattr(mcv_b200, name, None)
    monkeypatch.setattr(mcv_b200, "_fns", {})
    return monkeypatch


def test_set_up_shows_itself_complete(fresh):
    """A second thread makes its call while the first is still asking the library for its functions."""
    real, within, go = mcv_b200.lib, threading.Event(), threading.Event()

    def slow():
        if threading.current_thread().name == "first" and not go.is_set():
            within.set()
            assert go.wait(30)
        return real()

    # host tensors are refused after the set-up and before any function is called; a call that went on with half of
    # it fails otherwise
    seen = []

    def run():
        try:
            call()
        except Exception as e:      # noqa: BLE001
            seen.append((str(e), dict(mcv_b200._fns)))

    spec = mcv_b200.MRope(64, [32])
    fresh.setattr(mcv_b200, "MRope", lambda *a: spec)
    fresh.setattr(mcv_b200, "lib", slow)
    one = threading.Thread(target=run, name="first")
    one.start()
    assert within.wait(30)
    assert mcv_b200._torch is None
    two = threading.Thread(target=run, name="second")
    two.start()
    two.join(30)
    assert not two.is_alive() and len(seen) == 1
    message, functions = seen[0]
    assert "must be on a CUDA device" in message and "mrope" in functions
    go.set()
    one.join(30)
    assert len(seen) == 2 and "must be on a CUDA device" in seen[1][0]


def test_failed_set_up_is_tried_again(fresh):
    """A library that cannot be loaded gives its reason at every call, and calls work once it can."""
    real = mcv_b200.lib
    spec = mcv_b200.MRope(64, [32])
    fresh.setattr(mcv_b200, "MRope", lambda *a: spec)

    def missing():
        raise RuntimeError("libmcv_b200.so not built")

    fresh.setattr(mcv_b200, "lib", missing)
    for _ in range(2):
        with pytest.raises(RuntimeError, match="not built"):
            call()
    fresh.setattr(mcv_b200, "lib", real)
    with pytest.raises(RuntimeError, match="must be on a CUDA device"):
        call()

"""The attention of new rows is two launches that meet in its scratch: no other call on the stream, from
whatever thread, comes between them with the same scratch.  On the CPU: the library and the stream are
stand-ins, a call of the library takes as long as its two launches."""
import contextlib
import threading
import time

import pytest
import torch

import yirage_amd.fused as F
from tests.test_serving_scratch import BF, NB, STREAM, _i32, _logprobs, _select, _sparse
from yirage_amd import _lib


def _tree():
    cache = torch.zeros((4, 16, 2, 64), dtype=BF)
    return F.gqa_tree_paged(torch.zeros((2, 8, 64), dtype=BF), cache, cache, _i32(0, 1, 2), _i32(0, 1), _i32(3, 4))


class Library:
    """Every workspace NB bytes.  Calls that use one while another uses the same one are counted."""

    def __init__(self, wait):
        self.wait, self.users, self.met, self.calls, self.guard = wait, {}, 0, [], threading.Lock()

    def __getattr__(self, name):
        if name.endswith("_workspace"):
            return lambda *a: NB

        def launch(*a):
            assert a[-2:] == (NB, STREAM)
            address = a[-3]
            with self.guard:
                self.calls.append((name, address))
                self.met += self.users.get(address, 0)
                self.users[address] = self.users.get(address, 0) + 1
            time.sleep(self.wait)
            with self.guard:
                self.users[address] -= 1
            return _lib.YR_OK

        return launch


@pytest.fixture
def stand_ins(monkeypatch):
    library = Library(0.002)
    monkeypatch.setattr(F, "lib", lambda: library)
    monkeypatch.setattr(F, "_one_device", lambda *ts: 0)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: STREAM, raising=False)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(F, "_scratch_cache", {})
    return library


def _together(*calls, times=5):
    errors, start = [], threading.Barrier(len(calls))

    def run(call):
        try:
            start.wait()
            for _ in range(times):
                call()
        except Exception as e:  # (a thread's own error)
            errors.append(e)

    threads = [threading.Thread(target=run, args=(c,)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors


def test_two_threads_on_one_stream(stand_ins):
    _tree()  # (the scratch is there)
    _together(_tree, _tree, _tree)
    assert len(stand_ins.calls) == 16 and stand_ins.met == 0


@pytest.mark.parametrize("other", [_select, _sparse, _logprobs])
def test_another_operator_beside_it(stand_ins, other):
    _tree()
    other()
    _together(_tree, other, _tree)
    assert len(stand_ins.calls) == 17 and stand_ins.met == 0


def test_an_error_leaves_the_next_call_free(stand_ins):
    fail = stand_ins.__getattr__("yr_hip_gqa_tree_paged")
    stand_ins.yr_hip_last_error = lambda: b"no"
    stand_ins.yr_hip_gqa_tree_paged = lambda *a: _lib.YR_E_INVALID
    with pytest.raises(Exception):
        _tree()
    stand_ins.yr_hip_gqa_tree_paged = fail
    done = threading.Thread(target=_tree, daemon=True)
    done.start()
    done.join(10)
    assert not done.is_alive()

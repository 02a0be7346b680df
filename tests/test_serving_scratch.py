"""The serving operators' scratch lives until their launch has returned, whatever
another thread does to the cache of workspaces in between.  On the CPU: the library
and the stream are stand-ins."""
import contextlib
import gc
import weakref

import pytest
import torch

import yirage_amd.fused as F
from yirage_amd import _lib

STREAM, NB = 77, 70000
BF = torch.bfloat16


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32)


def _select():
    return F.select_pages(torch.zeros((2, 8, 64), dtype=BF), torch.zeros((4, 2, 2, 64), dtype=BF), _i32(0, 1, 2), _i32(0, 1),
                          _i32(3, 4), page_size=16, top_pages=4, max_kv_len=16)


def _sparse():
    cache = torch.zeros((4, 16, 2, 64), dtype=BF)
    return F.gqa_sparse_paged(torch.zeros((2, 8, 64), dtype=BF), cache, cache, _i32(0, 1, 2), _i32(0, 1), _i32(3, 4),
                              torch.zeros((2, 2, 3), dtype=torch.int32))


def _logprobs():
    return F.token_logprobs(torch.zeros((2, 10)), torch.zeros(2, dtype=torch.int64), top_n=2)


class Library:
    """Every workspace NB bytes; a launch runs `during` with the workspace's address."""

    def __init__(self, during):
        self.during, self.launches = during, 0

    def __getattr__(self, name):
        if name.endswith("_workspace"):
            return lambda *a: NB

        def launch(*a):
            assert a[-2:] == (NB, STREAM)
            self.launches += 1
            self.during(a[-3])
            return _lib.YR_OK

        return launch


@pytest.mark.parametrize("capturing", [False, True], ids=["eager", "captured"])
@pytest.mark.parametrize("call", [_select, _sparse, _logprobs])
def test_scratch_outlives_a_replaced_cache_entry(call, capturing, monkeypatch):
    key = (None, STREAM)  # (a CPU tensor's device has no index)
    made, empty = [], torch.empty

    def allocate(*a, **kw):
        t = empty(*a, **kw)
        if t.dtype is torch.uint8:
            made.append((weakref.ref(t), t.data_ptr()))
        return t

    def during(address):
        # another thread's larger call on the same stream takes the entry over
        F._scratch_cache[key] = torch.zeros(4 * NB, dtype=torch.uint8)
        gc.collect()
        assert [p for _, p in made] == [address]
        assert made[0][0]() is not None, "the scratch was freed before the launch"

    lib = Library(during)
    monkeypatch.setattr(F, "lib", lambda: lib)
    monkeypatch.setattr(F, "_one_device", lambda *ts: 0)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: STREAM, raising=False)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    monkeypatch.setattr(torch, "empty", allocate)
    monkeypatch.setattr(F, "_scratch_cache", {})
    if not capturing:
        F._scratch_cache[key] = torch.empty(NB, dtype=torch.uint8)
    call()
    assert lib.launches == 1


@pytest.mark.parametrize("call", [_select, _sparse, _logprobs])
def test_the_other_operators_workspace_stays(call, monkeypatch):
    """A graph may have its address: a call that needs more takes memory of its own."""
    lib = Library(lambda address: None)
    monkeypatch.setattr(F, "lib", lambda: lib)
    monkeypatch.setattr(F, "_one_device", lambda *ts: 0)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: STREAM, raising=False)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: type("Stream", (), {"cuda_stream": STREAM}))
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    mine = torch.empty(NB - 1, dtype=torch.uint8)
    monkeypatch.setattr(F, "_ws_cache", {(None, STREAM): mine})
    monkeypatch.setattr(F, "_scratch_cache", {}, raising=False)
    call()
    assert lib.launches == 1
    assert F.workspace(NB - 1, "cpu") is mine

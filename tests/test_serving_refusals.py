"""What the operators around a paged cache refuse, through the C ABI and through
the torch wrappers; nothing here reaches a GPU."""
import ctypes

import pytest
import torch

import yirage_amd.fused as F
from yirage_amd import YirageHipError, _lib

FAKE, ODD = ctypes.c_void_p(4096), ctypes.c_void_p(4104)


def _call(name, args, **change):
    vals = dict(args)
    vals.update(change)
    rc = getattr(_lib.lib(), name)(*vals.values())
    return rc, _lib.last_error()


def _strides(*v):
    return (ctypes.c_int64 * 7)(*(v or (6144, 512, 128, 6144, 128, 6144, 128)))


def _append(**change):
    a = dict(q=FAKE, k=FAKE, v=FAKE, q_out=FAKE, kc=FAKE, vc=FAKE, bounds=FAKE, cos=FAKE, sin=FAKE,
             tdt=_lib.DTYPE_F32, npos=64, qn=None, kn=None, eps=1e-6, qo=FAKE, ptr=FAKE, idx=FAKE, nidx=4, lens=FAKE,
             rows=5, batch=2, hq=32, hkv=8, d=128, page=64, pages=4, strides=_strides(), dt=_lib.DTYPE_BF16, stream=None)
    return _call("yr_hip_append_kv_paged", a, **change)


@pytest.mark.parametrize("change,text", [
    (dict(k=None), "null"), (dict(vc=None), "null"), (dict(lens=None), "null"), (dict(idx=None), "null"),
    (dict(strides=None), "null"), (dict(q=None), "together"), (dict(q_out=None), "together"), (dict(cos=None), "together"),
    (dict(tdt=_lib.DTYPE_F16), "tables"), (dict(npos=0), "tables"), (dict(dt=_lib.DTYPE_F32), "dtype"), (dict(d=96), "head_dim"),
    (dict(hq=30), "multiple"), (dict(hkv=0), "multiple"), (dict(hq=0), "positive"), (dict(rows=0), "positive"),
    (dict(batch=-1), "positive"), (dict(page=0), "page size"), (dict(pages=0), "page size"), (dict(nidx=-1), "page size"),
    (dict(qo=None), "one row"), (dict(k=ODD), "aligned"), (dict(bounds=ODD), "aligned"), (dict(sin=ODD), "aligned"),
    (dict(kn=ODD), "aligned"), (dict(strides=_strides(6144, 512, 128, 6144, 100, 6144, 128)), "multiples of 8"),
])
def test_append(change, text):
    rc, msg = _append(**change)
    assert rc == -1 and text in msg, msg


def _select(**change):
    a = dict(q=FAKE, bounds=FAKE, qo=FAKE, ptr=FAKE, idx=FAKE, nidx=4, lens=FAKE, pages=FAKE, rows=5, batch=2, hq=32,
             hkv=8, d=128, page=64, npages=4, maxlen=4096, top=8, first=1, last=1, dt=_lib.DTYPE_F16, ws=FAKE, nb=1 << 30, stream=None)
    return _call("yr_hip_select_pages", a, **change)


@pytest.mark.parametrize("change,text", [
    (dict(q=None), "null"), (dict(pages=None), "null"), (dict(ptr=None), "null"), (dict(d=32), "head_dim"),
    (dict(dt=0), "dtype"), (dict(hq=0), "positive"), (dict(hq=33), "multiple"), (dict(maxlen=0), "max_kv_len"),
    (dict(last=0), "last page"), (dict(first=-1), "last page"), (dict(top=0), "top_pages"),
    (dict(first=8), "top_pages"), (dict(first=2 ** 31 - 1), "top_pages"), (dict(page=1, maxlen=16385), "exceed"),
    (dict(q=ODD), "aligned"), (dict(bounds=ODD), "aligned"), (dict(qo=None), "one row"),
    (dict(rows=2 ** 30), "too many"),
])
def test_select(change, text):
    rc, msg = _select(**change)
    assert rc == -1 and text in msg, msg


def test_select_workspace():
    need = _lib.lib().yr_hip_select_pages_workspace(5, 8, 64, 40000)
    assert need == 65536 + 5 * 8 * 625 * 8
    for change in (dict(nb=need - 1), dict(ws=None)):
        rc, msg = _select(maxlen=40000, **change)
        assert rc == -3 and "workspace" in msg
    assert _lib.lib().yr_hip_select_pages_workspace(2048, 8, 64, 40000) == 0


def _sparse(**change):
    a = dict(q=FAKE, kc=FAKE, vc=FAKE, qo=FAKE, ptr=FAKE, idx=FAKE, nidx=4, lens=FAKE, pages=FAKE, out=FAKE, rows=5,
             batch=2, hq=32, hkv=8, d=128, page=64, npages=4, top=8, dt=_lib.DTYPE_F16, ws=FAKE, nb=1 << 30, stream=None)
    return _call("yr_hip_gqa_sparse_paged", a, **change)


@pytest.mark.parametrize("change,text", [
    (dict(kc=None), "null"), (dict(out=None), "null"), (dict(pages=None), "null"), (dict(lens=None), "null"),
    (dict(d=256), "head_dim"), (dict(dt=_lib.DTYPE_F32), "dtype"), (dict(hq=136), "group size"), (dict(hq=0), "group size"),
    (dict(top=0), "top_pages"), (dict(top=1025), "top_pages"), (dict(page=0), "page size"), (dict(qo=None), "one row"),
    (dict(top=1024, page=2 ** 20 + 1), "page size"), (dict(hq=2 ** 22, hkv=2 ** 20), "too many"), (dict(rows=2 ** 30), "too many"), (dict(vc=ODD), "aligned"),
    (dict(out=ODD), "aligned"),
])
def test_sparse(change, text):
    rc, msg = _sparse(**change)
    assert rc == -1 and text in msg, msg


def test_sparse_workspace():
    need = _lib.lib().yr_hip_gqa_sparse_workspace(5, 2, 1, 32, 8, 128, 64, 8)
    assert need > 65536
    for change in (dict(nb=need - 1), dict(ws=None)):
        rc, msg = _sparse(**change)
        assert rc == -3 and "workspace" in msg
    assert _lib.lib().yr_hip_gqa_sparse_workspace(64, 64, 0, 32, 8, 128, 64, 8) == 0


def _logprobs(**change):
    a = dict(x=FAKE, tok=FAKE, lp=FAKE, h=FAKE, tlp=FAKE, tid=FAKE, rows=3, n=1000, nv=1000, stride=1000, top=5,
             dt=_lib.DTYPE_F32, ws=FAKE, nb=1 << 30, stream=None)
    return _call("yr_hip_token_logprobs", a, **change)


@pytest.mark.parametrize("change,text", [
    (dict(x=None), "null"), (dict(tok=None), "null"), (dict(tlp=None), "null"), (dict(tid=None), "null"),
    (dict(rows=0), "bad shape"), (dict(n=0), "bad shape"), (dict(nv=0), "bad shape"), (dict(nv=1001), "bad shape"),
    (dict(stride=999), "bad shape"), (dict(top=-1), "top_n"), (dict(top=65), "top_n"), (dict(nv=4), "top_n"),
    (dict(dt=_lib.DTYPE_I32), "dtype"), (dict(x=ctypes.c_void_p(4098)), "aligned"), (dict(n=2 ** 30 + 1, stride=2 ** 31), "too many"),
])
def test_logprobs(change, text):
    rc, msg = _logprobs(**change)
    assert rc == -1 and text in msg, msg


def test_logprobs_workspace():
    need = _lib.lib().yr_hip_token_logprobs_workspace(3, 100000, 5, _lib.DTYPE_F32)
    assert need > 65536
    for change in (dict(nb=need - 1), dict(ws=None)):
        rc, msg = _logprobs(n=100000, nv=100000, stride=100000, **change)
        assert rc == -3 and "workspace" in msg
    assert _lib.lib().yr_hip_token_logprobs_workspace(4096, 100000, 5, _lib.DTYPE_F32) == 0


# ------------------------------------------------------------------ wrappers
BF = torch.bfloat16


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32)


def _step(**change):
    t = dict(q=torch.zeros((2, 8, 64), dtype=BF), k=torch.zeros((2, 2, 64), dtype=BF), v=torch.zeros((2, 2, 64), dtype=BF),
             kc=torch.zeros((4, 16, 2, 64), dtype=BF), vc=torch.zeros((4, 16, 2, 64), dtype=BF),
             bounds=torch.zeros((4, 2, 2, 64), dtype=BF), ptr=_i32(0, 1, 2), idx=_i32(0, 1), lens=_i32(3, 4), qo=None,
             cos=torch.zeros((16, 64)), sin=torch.zeros((16, 64)), qn=None, kn=None, out=None,
             pages=torch.zeros((2, 2, 3), dtype=torch.int32))
    t.update(change)
    return t


@pytest.mark.parametrize("change,text", [
    (dict(k=torch.zeros((2, 2, 64))), "dtype"), (dict(k=torch.zeros((2, 2, 64), dtype=torch.float16)), "dtype"),
    (dict(k=torch.zeros((2, 3, 64), dtype=BF)), "k and v"), (dict(vc=torch.zeros((3, 16, 2, 64), dtype=BF)), "k and v"),
    (dict(kc=torch.zeros((4, 16, 1, 64), dtype=BF), vc=torch.zeros((4, 16, 1, 64), dtype=BF)), "cache heads"),
    (dict(idx=torch.zeros(2, dtype=torch.int64)), "int32"), (dict(lens=_i32(3)), "entries"), (dict(ptr=_i32(0, 1)), "entries"),
    (dict(qo=_i32(0, 2)), "entries"), (dict(lens=_i32(3, 4, 5), ptr=_i32(0, 1, 2, 2)), "one row"),
    (dict(bounds=torch.zeros((4, 2, 64), dtype=BF)), "page_bounds"), (dict(kn=torch.zeros(32, dtype=BF)), "norm weights"),
    (dict(sin=None), "together"), (dict(sin=torch.zeros((8, 64))), "cos and sin"), (dict(cos=torch.zeros((16, 32)), sin=torch.zeros((16, 32))), "cos and sin"),
    (dict(cos=torch.zeros((16, 64), dtype=torch.float64), sin=torch.zeros((16, 64), dtype=torch.float64)), "tables"),
    (dict(q=torch.zeros((2, 7, 64), dtype=BF)), "heads"), (dict(q=torch.zeros((2, 3, 4, 64), dtype=BF)), "q must be"),
    (dict(q=None, out=torch.zeros((2, 8, 64), dtype=BF)), "need q"), (dict(out=torch.zeros((2, 8, 32), dtype=BF)), "out must be"),
    (dict(out=torch.zeros((2, 8, 64))), "out must be"), (dict(kc=torch.zeros((4, 2, 16, 64), dtype=BF).transpose(1, 2)), "contiguous"),
    (dict(k=torch.zeros((2, 64, 2), dtype=BF).transpose(1, 2)), "last dim"), ({}, "GPU"),
])
def test_append_wrapper(change, text):
    t = _step(**change)
    with pytest.raises(YirageHipError, match=text):
        F.append_kv_paged(t["k"], t["v"], t["kc"], t["vc"], t["ptr"], t["idx"], t["lens"], q=t["q"], cos=t["cos"],
                          sin=t["sin"], q_norm=t["qn"], k_norm=t["kn"], qo_indptr=t["qo"], page_bounds=t["bounds"], out=t["out"])


@pytest.mark.parametrize("change,text", [
    (dict(q=torch.zeros((2, 8, 64))), "dtype"), (dict(bounds=torch.zeros((4, 2, 3, 64), dtype=BF)), "page_bounds"),
    (dict(q=torch.zeros((2, 8, 128), dtype=BF)), "page_bounds"), (dict(q=torch.zeros((2, 64, 8), dtype=BF).transpose(1, 2)), "contiguous"),
    (dict(lens=_i32(3)), "entries"), (dict(out=torch.zeros((2, 2, 4), dtype=torch.int64)), "out must be"), ({}, "GPU"),
])
def test_select_wrapper(change, text):
    t = _step(**change)
    with pytest.raises(YirageHipError, match=text):
        F.select_pages(t["q"], t["bounds"], t["ptr"], t["idx"], t["lens"], page_size=16, top_pages=4, out=t["out"])


@pytest.mark.parametrize("change,text", [
    (dict(vc=torch.zeros((4, 16, 2, 64))), "dtype"), (dict(pages=torch.zeros((2, 2, 3), dtype=torch.int64)), "int32"),
    (dict(pages=torch.zeros((2, 8, 3), dtype=torch.int32)), "pages must be"), (dict(q=torch.zeros((2, 8, 32), dtype=BF)), "caches"),
    (dict(pages=torch.zeros((2, 3, 2), dtype=torch.int32).transpose(1, 2)), "contiguous"), (dict(qo=_i32(0, 1, 2, 2)), "entries"),
    ({}, "GPU"),
])
def test_sparse_wrapper(change, text):
    t = _step(**change)
    with pytest.raises(YirageHipError, match=text):
        F.gqa_sparse_paged(t["q"], t["kc"], t["vc"], t["ptr"], t["idx"], t["lens"], t["pages"], qo_indptr=t["qo"], out=t["out"])


def test_logprobs_wrapper():
    x, tok = torch.zeros((2, 10)), torch.zeros(2, dtype=torch.int64)
    for bad, text in [((x.double(), tok), "dtype"), ((x[0], tok), "logits must be"), ((x.t().contiguous().t(), tok), "logits must be"),
                      ((x, tok.int()), "tokens"), ((x, tok[:1]), "tokens"), ((x, tok), "GPU")]:
        with pytest.raises(YirageHipError, match=text):
            F.token_logprobs(*bad)

"""What the operators of drafting over a paged cache refuse, through the C ABI and through the
torch wrappers; nothing here reaches a GPU."""
import ctypes

import pytest
import torch

import test_serving_scratch as Scratch
import yirage_amd.fused as F
from test_serving_refusals import FAKE, ODD, _call, _i32, _strides
from yirage_amd import YirageHipError, _lib

E4M3, E8M0, BF = torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.bfloat16


def _append(name="yr_hip_append_kv_paged_fp8", **change):
    a = dict(q=FAKE, k=FAKE, v=FAKE, q_out=FAKE, kc=FAKE, vc=FAKE, ks=FAKE, vs=FAKE, cos=FAKE, sin=FAKE, tdt=_lib.DTYPE_F32,
             npos=64, qn=None, kn=None, eps=1e-6, pos=FAKE, qo=FAKE, ptr=FAKE, idx=FAKE, nidx=4, lens=FAKE, rows=5, batch=2, hq=32,
             hkv=8, d=128, page=64, pages=4, strides=_strides(), dt=_lib.DTYPE_BF16, stream=None)
    return _call(name, a, **change)


@pytest.mark.parametrize("change,text", [
    (dict(k=None), "null"), (dict(vc=None), "null"), (dict(ks=None), "null"), (dict(vs=None), "null"), (dict(lens=None), "null"),
    (dict(strides=None), "null"), (dict(q=None), "together"), (dict(q_out=None), "together"), (dict(cos=None), "together"),
    (dict(cos=None, sin=None), "positions"), (dict(q=None, q_out=None, qn=FAKE), "q_norm"), (dict(tdt=_lib.DTYPE_F16), "tables"),
    (dict(npos=0), "tables"), (dict(dt=_lib.DTYPE_F32), "dtype"), (dict(dt=_lib.DTYPE_E4M3), "dtype"), (dict(d=96), "head_dim"),
    (dict(hq=30), "multiple"), (dict(hkv=0), "multiple"), (dict(hq=0), "positive"), (dict(rows=0), "positive"),
    (dict(page=0), "page size"), (dict(nidx=-1), "page size"), (dict(qo=None), "one row"), (dict(k=ODD), "aligned"),
    (dict(vc=ODD), "aligned"), (dict(kn=ODD), "aligned"), (dict(hq=2 ** 21, hkv=2 ** 20), "too many"),
    (dict(strides=_strides(6144, 512, 128, 6144, 100, 6144, 128)), "multiples of 8"),
])
def test_append(change, text):
    rc, msg = _append(**change)
    assert rc == -1 and text in msg, msg


def test_append_at():
    """The 16-bit append with positions checks what the one without does, and its positions."""
    a = dict(q=FAKE, k=FAKE, v=FAKE, q_out=FAKE, kc=FAKE, vc=FAKE, bounds=FAKE, cos=FAKE, sin=FAKE, tdt=_lib.DTYPE_F32, npos=64, qn=None,
             kn=None, eps=1e-6, pos=FAKE, qo=FAKE, ptr=FAKE, idx=FAKE, nidx=4, lens=FAKE, rows=5, batch=2, hq=32, hkv=8, d=128,
             page=64, pages=4, strides=_strides(), dt=_lib.DTYPE_BF16, stream=None)
    for change, text in [(dict(pos=None), "positions"), (dict(cos=None, sin=None), "positions"), (dict(k=None), "null"),
                         (dict(d=32), "head_dim"), (dict(bounds=ODD), "aligned")]:
        rc, msg = _call("yr_hip_append_kv_paged_at", a, **change)
        assert rc == -1 and text in msg and "paged_at" in msg, msg


def _read(**change):
    a = dict(kc=FAKE, vc=FAKE, ks=FAKE, vs=FAKE, ptr=FAKE, idx=FAKE, nidx=4, lens=FAKE, to=FAKE, k=FAKE, v=FAKE, rows=5, batch=2,
             hkv=8, d=128, page=64, pages=4, dt=_lib.DTYPE_BF16, stream=None)
    return _call("yr_hip_read_kv_paged_fp8", a, **change)


@pytest.mark.parametrize("change,text", [
    (dict(kc=None), "null"), (dict(vs=None), "null"), (dict(to=None), "null"), (dict(v=None), "null"), (dict(idx=None), "null"),
    (dict(d=32), "head_dim"), (dict(dt=_lib.DTYPE_E4M3), "dtype"), (dict(rows=0), "positive"), (dict(hkv=0), "multiple"),
    (dict(pages=0), "page size"), (dict(page=2 ** 20 + 1), "page size"), (dict(vc=ODD), "aligned"), (dict(k=ODD), "aligned"),
    (dict(hkv=2 ** 20 + 1), "too many"),
])
def test_read(change, text):
    rc, msg = _read(**change)
    assert rc == -1 and text in msg, msg


def _tree(**change):
    a = dict(q=FAKE, kc=FAKE, vc=FAKE, ks=FAKE, vs=FAKE, mask=FAKE, mrow=8, mcols=8, qo=FAKE, ptr=FAKE, idx=FAKE, nidx=4, lens=FAKE,
             out=FAKE, rows=5, batch=2, hq=32, hkv=8, d=128, page=64, pages=4, most=4096, cdt=_lib.DTYPE_E4M3, dt=_lib.DTYPE_F16,
             ws=FAKE, nb=1 << 40, stream=None)
    return _call("yr_hip_gqa_tree_paged", a, **change)


@pytest.mark.parametrize("change,text", [
    (dict(q=None), "null"), (dict(kc=None), "null"), (dict(out=None), "null"), (dict(lens=None), "null"), (dict(d=256), "head_dim"),
    (dict(dt=_lib.DTYPE_F32), "dtype"), (dict(cdt=_lib.DTYPE_BF16), "q's type"), (dict(ks=None), "scales"), (dict(vs=None), "scales"),
    (dict(cdt=_lib.DTYPE_F16), "scales"), (dict(hq=136), "group size"), (dict(hq=0), "group size"), (dict(hq=33), "multiple"),
    (dict(mcols=0), "tree_mask"), (dict(mrow=-1), "tree_mask"), (dict(qo=None), "one row"), (dict(kc=ODD), "aligned"),
    (dict(out=ODD), "aligned"), (dict(page=2 ** 20, pages=2 ** 12), "2^32"), (dict(hq=2 ** 21, hkv=2 ** 21), "too many"),
    (dict(rows=2 ** 30), "too many"),
])
def test_tree(change, text):
    rc, msg = _tree(**change)
    assert rc == -1 and text in msg, msg


def test_tree_workspace():
    need = _lib.lib().yr_hip_gqa_tree_workspace(5, 2, 1, 32, 8, 128, 4096, _lib.DTYPE_E4M3)
    assert need > 65536
    for change in (dict(nb=need - 1), dict(ws=None)):
        rc, msg = _tree(**change)
        assert rc == -3 and "workspace" in msg
    # short sequences, and many, are not split
    assert _lib.lib().yr_hip_gqa_tree_workspace(5, 2, 1, 32, 8, 128, 512, _lib.DTYPE_E4M3) == 0
    assert _lib.lib().yr_hip_gqa_tree_workspace(1024, 1024, 0, 32, 8, 128, 4096, _lib.DTYPE_F16) == 0


def test_new_lengths_beside_the_old():
    """Overlapping lengths are refused, neighbouring ones are not."""
    both, t = torch.zeros(8, dtype=torch.int32), _step()
    args = lambda lens: (t["kc"], t["vc"], t["ptr"], t["idx"], lens, t["path"])
    for at, text in ((1, "another"), (2, "GPU"), (0, "another")):
        with pytest.raises(YirageHipError, match=text):
            F.keep_kv_paged(*args(both[:2]), k_scale=t["ks"], v_scale=t["vs"], out=both[at: at + 2])
    for at in (4092, 4096, 4100):  # kv_len is 4096 there, of two sequences
        rc, msg = _keep(out=ctypes.c_void_p(at))
        assert rc == -1 and "place of their own" in msg, (at, msg)


def _keep(**change):
    a = dict(kc=FAKE, vc=FAKE, ks=FAKE, vs=FAKE, bounds=None, path=FAKE, depth=4, qo=FAKE, ptr=FAKE, idx=FAKE, nidx=4, lens=FAKE,
             out=ctypes.c_void_p(8192), batch=2, hkv=8, d=128, page=64, pages=4, dt=_lib.DTYPE_E4M3, stream=None)
    return _call("yr_hip_keep_kv_paged", a, **change)


@pytest.mark.parametrize("change,text", [
    (dict(kc=None), "null"), (dict(path=None), "null"), (dict(out=None), "null"), (dict(lens=None), "null"), (dict(ks=None), "scales"),
    (dict(dt=_lib.DTYPE_F16), "scales"), (dict(bounds=FAKE), "bounds"), (dict(dt=_lib.DTYPE_F32, ks=None, vs=None), "dtype"),
    (dict(depth=0), "entry"), (dict(batch=0), "positive"), (dict(d=96), "head_dim"), (dict(page=0), "page size"),
    (dict(kc=ODD), "aligned"), (dict(out=FAKE), "place of their own"), (dict(hkv=2 ** 20 + 1), "too many"),
])
def test_keep(change, text):
    rc, msg = _keep(**change)
    assert rc == -1 and text in msg, msg


# ------------------------------------------------------------------ wrappers
def _step(**change):
    z = lambda *s, dtype=BF: torch.zeros(s, dtype=dtype)
    t = dict(q=z(2, 8, 64), k=z(2, 2, 64), v=z(2, 2, 64), kc=z(4, 16, 2, 64, dtype=E4M3), vc=z(4, 16, 2, 64, dtype=E4M3),
             ks=z(4, 16, 2, dtype=torch.uint8).view(E8M0), vs=z(4, 16, 2, dtype=torch.uint8).view(E8M0), k16=z(4, 16, 2, 64),
             ptr=_i32(0, 1, 2), idx=_i32(0, 1), lens=_i32(3, 4), qo=None, cos=z(16, 64, dtype=torch.float32),
             sin=z(16, 64, dtype=torch.float32), qn=None, kn=None, out=None, pos=_i32(2, 3), mask=z(2, 4, dtype=torch.bool),
             path=z(2, 3, dtype=torch.int32), bounds=None, to=_i32(0, 1, 2), total=2, dtype=BF)
    t.update(change)
    return t


@pytest.mark.parametrize("change,text", [
    (dict(k=torch.zeros((2, 2, 64))), "dtype"), (dict(v=torch.zeros((2, 2, 64), dtype=torch.float16)), "dtype"),
    (dict(kc=torch.zeros((4, 16, 2, 64), dtype=BF)), "e4m3fn"), (dict(ks=torch.zeros((4, 16, 2))), "e8m0"), (dict(vs=None), "e8m0"),
    (dict(ks=torch.zeros((4, 2, 16), dtype=torch.uint8).view(E8M0)), "scales"), (dict(vc=torch.zeros((4, 8, 2, 64), dtype=E4M3)), "scales"),
    (dict(kc=torch.zeros((4, 2, 16, 64), dtype=torch.uint8).transpose(1, 2).view(E4M3)), "contiguous"),
    (dict(k=torch.zeros((2, 3, 64), dtype=BF)), "k and v"), (dict(k=torch.zeros((2, 1, 64), dtype=BF), v=torch.zeros((2, 1, 64), dtype=BF)), "cache heads"),
    (dict(pos=_i32(1)), "positions"), (dict(pos=torch.zeros(2, dtype=torch.int64)), "positions"), (dict(cos=None, sin=None), "positions"),
    (dict(sin=None), "together"), (dict(cos=torch.zeros((16, 64), dtype=torch.float64), sin=torch.zeros((16, 64), dtype=torch.float64)), "tables"),
    (dict(kn=torch.zeros(32, dtype=BF)), "norm weights"), (dict(lens=_i32(3)), "entries"), (dict(q=torch.zeros((2, 7, 64), dtype=BF)), "heads"),
    (dict(q=None, out=torch.zeros((2, 8, 64), dtype=BF)), "need q"), (dict(out=torch.zeros((2, 8, 32), dtype=BF)), "out must be"),
    (dict(k=torch.zeros((2, 64, 2), dtype=BF).transpose(1, 2)), "last dim"), ({}, "GPU"),
])
def test_append_wrapper(change, text):
    t = _step(**change)
    with pytest.raises(YirageHipError, match=text):
        F.append_kv_paged_fp8(t["k"], t["v"], t["kc"], t["vc"], t["ks"], t["vs"], t["ptr"], t["idx"], t["lens"], q=t["q"], cos=t["cos"],
                              sin=t["sin"], q_norm=t["qn"], k_norm=t["kn"], qo_indptr=t["qo"], positions=t["pos"], out=t["out"])


@pytest.mark.parametrize("change,text", [(dict(pos=_i32(1)), "positions"), (dict(cos=None, sin=None), "positions"), ({}, "GPU")])
def test_append_16_bit_with_positions(change, text):
    t = _step(**change)
    with pytest.raises(YirageHipError, match=text):
        F.append_kv_paged(t["k"], t["v"], t["k16"], t["k16"], t["ptr"], t["idx"], t["lens"], cos=t["cos"], sin=t["sin"], positions=t["pos"])


@pytest.mark.parametrize("change,text", [
    (dict(kc=torch.zeros((4, 16, 2, 64), dtype=BF)), "e4m3fn"), (dict(dtype=torch.float32), "dtype"), (dict(total=-1), "negative"),
    (dict(to=None), "out_indptr"), (dict(to=_i32(0, 2)), "entries"), (dict(lens=_i32(3)), "entries"),
    (dict(out=(torch.zeros((2, 2, 64), dtype=BF), torch.zeros((2, 2, 64)))), "out must be"), ({}, "GPU"),
])
def test_read_wrapper(change, text):
    t = _step(**change)
    with pytest.raises(YirageHipError, match=text):
        F.read_kv_paged_fp8(t["kc"], t["vc"], t["ks"], t["vs"], t["ptr"], t["idx"], t["lens"], t["to"], t["total"], dtype=t["dtype"], out=t["out"])


@pytest.mark.parametrize("change,text", [
    (dict(q=torch.zeros((2, 8, 64))), "dtype"), (dict(ks=None), "e8m0"), (dict(kc=torch.zeros((4, 16, 2, 64), dtype=torch.float16)), "dtype"),
    (dict(kc=torch.zeros((4, 16, 2, 64), dtype=BF), vc=torch.zeros((4, 16, 2, 64), dtype=BF)), "go with"), (dict(vc=torch.zeros((4, 16, 2, 64), dtype=BF)), "e4m3fn"),
    (dict(q=torch.zeros((2, 8, 128), dtype=BF)), "q must be"), (dict(q=torch.zeros((2, 64, 8), dtype=BF).transpose(1, 2)), "contiguous"),
    (dict(mask=torch.zeros((2, 4), dtype=torch.uint8)), "tree_mask"), (dict(mask=torch.zeros((3, 4), dtype=torch.bool)), "tree_mask"),
    (dict(mask=torch.zeros((2, 0), dtype=torch.bool)), "tree_mask"), (dict(mask=torch.zeros((4, 2), dtype=torch.bool).t()), "last dim"),
    (dict(qo=_i32(0, 2)), "entries"), (dict(out=torch.zeros((2, 8, 64))), "out must be"), ({}, "GPU"),
])
def test_tree_wrapper(change, text):
    t = _step(**change)
    with pytest.raises(YirageHipError, match=text):
        F.gqa_tree_paged(t["q"], t["kc"], t["vc"], t["ptr"], t["idx"], t["lens"], tree_mask=t["mask"], qo_indptr=t["qo"], k_scale=t["ks"],
                         v_scale=t["vs"], max_kv_len=16, out=t["out"])


@pytest.mark.parametrize("change,text", [
    (dict(path=torch.zeros((2, 3), dtype=torch.int64)), "path"), (dict(path=torch.zeros((1, 3), dtype=torch.int32)), "path"),
    (dict(path=torch.zeros((2, 0), dtype=torch.int32)), "path"), (dict(path=torch.zeros((3, 2), dtype=torch.int32).t()), "path"),
    (dict(bounds=torch.zeros((4, 2, 2, 64), dtype=BF)), "16 bits"), (dict(vs=None), "e8m0"), (dict(out="kv_len"), "another"),
    (dict(out=torch.zeros(2)), "another"), (dict(kc=torch.zeros((4, 16, 2, 64)), vc=torch.zeros((4, 16, 2, 64))), "dtype"),
    (dict(kc=torch.zeros((4, 16, 2, 64), dtype=BF), vc=torch.zeros((4, 16, 2, 64), dtype=BF)), "go with"),
    (dict(kc=torch.zeros((4, 16, 2, 64), dtype=BF), vc=torch.zeros((4, 16, 2, 64), dtype=BF), ks=None, vs=None, bounds=torch.zeros((4, 2, 64), dtype=BF)), "page_bounds"),
    ({}, "GPU"),
])
def test_keep_wrapper(change, text):
    t = _step(**change)
    out = t["lens"] if t["out"] == "kv_len" else t["out"]
    with pytest.raises(YirageHipError, match=text):
        F.keep_kv_paged(t["kc"], t["vc"], t["ptr"], t["idx"], t["lens"], t["path"], qo_indptr=t["qo"], k_scale=t["ks"], v_scale=t["vs"],
                        page_bounds=t["bounds"], out=out)


def test_nothing_to_do(monkeypatch):
    """No rows, no sequences: results of that shape, no launch."""
    monkeypatch.setattr(F, "_one_device", lambda *ts: 0)
    monkeypatch.setattr(F, "_launch", lambda *a: pytest.fail("a launch"))
    t, none = _step(), torch.zeros(0, dtype=torch.int32)
    empty = dict(k=torch.zeros((0, 2, 64), dtype=BF), q=torch.zeros((0, 8, 64), dtype=BF))
    qo = _i32(0, 0, 0)
    got = F.append_kv_paged_fp8(empty["k"], empty["k"], t["kc"], t["vc"], t["ks"], t["vs"], t["ptr"], t["idx"], t["lens"], q=empty["q"], qo_indptr=qo)
    assert got.shape == (0, 8, 64)
    assert F.gqa_tree_paged(empty["q"], t["kc"], t["vc"], t["ptr"], t["idx"], t["lens"], qo_indptr=qo, k_scale=t["ks"], v_scale=t["vs"]).shape == (0, 8, 64)
    k, v = F.read_kv_paged_fp8(t["kc"], t["vc"], t["ks"], t["vs"], t["ptr"], t["idx"], t["lens"], qo, 0)
    assert k.shape == v.shape == (0, 2, 64)
    assert F.keep_kv_paged(t["kc"], t["vc"], _i32(0), none, none, torch.zeros((0, 3), dtype=torch.int32), k_scale=t["ks"], v_scale=t["vs"],
                           out=none.clone()).shape == (0,)
    kept = F.keep_kv_paged(t["kc"], t["vc"], _i32(0), none, none, torch.zeros((0, 3), dtype=torch.int32), k_scale=t["ks"], v_scale=t["vs"])
    assert kept.shape == (0,)


def _attend():
    t = _step()
    return F.gqa_tree_paged(t["q"], t["kc"], t["vc"], t["ptr"], t["idx"], t["lens"], k_scale=t["ks"], v_scale=t["vs"])


@pytest.mark.parametrize("capturing", [False, True], ids=["eager", "captured"])
def test_scratch_outlives_a_replaced_cache_entry(capturing, monkeypatch):
    Scratch.test_scratch_outlives_a_replaced_cache_entry(_attend, capturing, monkeypatch)


def test_the_other_operators_workspace_stays(monkeypatch):
    Scratch.test_the_other_operators_workspace_stays(_attend, monkeypatch)

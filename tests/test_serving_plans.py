"""Which kernel page selection and sparse attention run on (host only), and that the
GPU tests written for a kernel reach it."""
import ctypes

import pytest

import test_gpu_select_pages as S
import test_gpu_serving_edges as E
import test_gpu_sparse_attn as A
from yirage_amd import _lib


def shapes(test):
    """The tuples that a test's shapes are drawn from."""
    return [m.args[1] for m in test.pytestmark if m.name == "parametrize" and m.args[0].startswith(("lens", "hq"))][0]


def select_plan(rows, batch, hkv, page, most, ragged=True):
    plan = (ctypes.c_int * 3)()
    assert _lib.lib().yr_hip_select_pages_plan(rows, batch, int(ragged), hkv, page, most, plan) == 0, _lib.last_error()
    return tuple(plan)


def sparse_plan(rows, batch, hq, hkv, page, top, ragged=True):
    plan = (ctypes.c_int * 3)()
    assert _lib.lib().yr_hip_gqa_sparse_plan(rows, batch, int(ragged), hq, hkv, page, top, plan) == 0, _lib.last_error()
    return tuple(plan)


@pytest.mark.parametrize("rows,batch,hkv,page,most,plan", [
    (1, 1, 8, 64, 131072, (0, 8, 16)), (32, 32, 8, 16, 16384, (0, 16, 1)), (64, 64, 8, 64, 4096, (0, 4, 1)),
    (2, 2, 2, 1, 16384, (0, 16, 64)), (600, 600, 8, 16, 16384, (0, 4, 1)),
])
def test_selection_row_by_row(rows, batch, hkv, page, most, plan):
    assert select_plan(rows, batch, hkv, page, most, ragged=False) == plan


@pytest.mark.parametrize("most,tile", [(1, 0), (32768, 16), (65536, 16), (65537, 8), (131072, 8), (131073, 4), (262144, 4), (262145, 0)])
def test_selection_tiles_have_as_many_rows_as_their_keys_have_room(most, tile):
    assert select_plan(512, 1, 8, 64, most)[0] == tile


def test_selection_tests_reach_their_tiles():
    for lens, news, hq, hkv, d, page, top, first, last in shapes(S.test_tiles):
        assert select_plan(sum(news), len(news), hkv, page, max(lens))[0] > 0
    assert select_plan(700, 1, 1, 16, 4800)[0] == 16       # near the border
    assert select_plan(600 + 100 + 5, 2, 2, 16, 4800)[0] == 16  # with rows left alone
    assert select_plan(720, 1, 1, 16, 260 * 16)[0] == 16   # scores that cancel
    got = [select_plan(sum(news), len(news), hkv, page, max(lens))[0]
           for lens, news, hq, hkv, d, page, top, first, last in shapes(E.test_tiles_of_each_size)]
    assert got == [16, 8, 8, 8, 4, 4]
    for kind, tile in (("rows", 0), ("tiles", 16)):
        lens, news = E.many(kind)
        assert select_plan(sum(news), len(news), 2, 16, max(lens))[0] == tile


def test_attention_tests_reach_their_tiles():
    for lens, news, hq, hkv, d, page, top in shapes(A.test_rows_of_wide_tiles):
        assert sparse_plan(sum(news), len(news), hq, hkv, page, top)[1] == 1
    for hq, page, before, rows, hkv in shapes(A.test_values_that_other_rows_of_wide_tiles_see):
        assert sparse_plan(rows, 1, hq, hkv, page, 4)[1] == 1
    assert sparse_plan(390 + 100, 2, 64, 8, 24, 12)[1] == 1
    for lens, news, hq, hkv, d, page, top, wide in shapes(E.test_more_pages_than_a_table_of_masks):
        assert sparse_plan(sum(news), len(news), hq, hkv, page, top)[1] == wide
    for kind, hq, hkv, wide in (("few", 8, 2, 0), ("wide", 64, 8, 1), ("ones", 64, 8, 1)):
        lens, news = E.many(kind)
        assert sparse_plan(sum(news), len(news), hq, hkv, 24, 4)[1] == wide


def test_refusals():
    plan = (ctypes.c_int * 3)()
    lib = _lib.lib()
    for args in ((0, 1, 1, 8, 64, 100), (1, 0, 1, 8, 64, 100), (1, 1, 1, 0, 64, 100), (1, 1, 1, 8, 0, 100), (1, 1, 1, 8, 64, 0),
                 (1, 1, 1, 8, 1, 16385)):
        assert lib.yr_hip_select_pages_plan(*args, plan) == -1 and "shape" in _lib.last_error()
    assert lib.yr_hip_select_pages_plan(1, 1, 1, 8, 64, 100, None) == -1
    for args in ((0, 1, 1, 8, 8, 64, 4), (1, 0, 1, 8, 8, 64, 4), (1, 1, 1, 9, 8, 64, 4), (1, 1, 1, 136, 8, 64, 4), (1, 1, 1, 8, 8, 0, 4),
                 (1, 1, 1, 8, 8, 64, 0), (1, 1, 1, 8, 8, 64, 1025)):
        assert lib.yr_hip_gqa_sparse_plan(*args, plan) == -1 and "shape" in _lib.last_error()
    assert lib.yr_hip_gqa_sparse_plan(1, 1, 1, 8, 8, 64, 4, None) == -1

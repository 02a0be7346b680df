"""Which kernel attention of new rows runs on (host only), and that the GPU tests reach each."""
import ctypes

import pytest

import test_gpu_tree_attn as A
import test_gpu_tree_edges as E
from yirage_amd import _lib


def plan(rows, batch, hq, hkv, d, most, cache, ragged=True):
    got = (ctypes.c_int * 3)()
    assert _lib.lib().yr_hip_gqa_tree_plan(rows, batch, int(ragged), hq, hkv, d, most, cache, got) == 0, _lib.last_error()
    return tuple(got)


@pytest.mark.parametrize("args,want", [
    ((1, 1, 32, 8, 128, 32768, _lib.DTYPE_E4M3, False), (16, 1, 32)), ((32, 32, 32, 8, 128, 8192, _lib.DTYPE_BF16, False), (16, 1, 32)),
    ((8, 1, 32, 8, 128, 32768, _lib.DTYPE_E4M3), (32, 8, 32)), ((16, 1, 32, 8, 128, 32768, _lib.DTYPE_E4M3), (64, 16, 64)),
    ((64, 1, 32, 8, 128, 32768, _lib.DTYPE_F16), (128, 32, 64)), ((2048, 1, 32, 8, 128, 16384, _lib.DTYPE_F16), (128, 32, 64)),
    ((2048, 1, 35, 7, 64, 16384, _lib.DTYPE_F16), (128, 25, 73)),  # 5 heads a group: 125 columns
    ((1, 1, 32, 8, 128, 512, _lib.DTYPE_E4M3, False), (16, 1, 0)),  # short: not split
    ((300, 300, 16, 8, 64, 4096, _lib.DTYPE_E4M3, False), (16, 1, 0)),  # enough of them
    ((1, 1, 32, 8, 128, 0, _lib.DTYPE_E4M3, False), (16, 1, 32)),  # no length given
])
def test_plans(args, want):
    assert plan(*args) == want


def test_plan_refuses():
    got = (ctypes.c_int * 3)()
    for bad in ((0, 1, 1, 32, 8, 128, 1, 930), (1, 1, 1, 33, 8, 128, 1, 930), (1, 1, 1, 32, 8, 96, 1, 930), (1, 1, 1, 136, 8, 128, 1, 930)):
        assert _lib.lib().yr_hip_gqa_tree_plan(*bad, got) == -1
    assert _lib.lib().yr_hip_gqa_tree_plan(1, 1, 1, 32, 8, 128, 1, 930, None) == -1


def test_cases_reach_every_width():
    seen = set()
    cases = [(*c, 0) for c in A.CASES] + [(c[0], c[1], c[2], c[3], c[4], c[5], c[7], c[6] or 0) for c in E.CASES]
    for lens, news, hq, hkv, d, page, tree, most in cases:
        for cache in (_lib.DTYPE_E4M3, _lib.DTYPE_BF16):
            p = plan(sum(news), len(news), hq, hkv, d, most, cache, any(n != 1 for n in news))
            seen.add((d, p[0], p[2] > 0))
    assert seen >= {(d, w, True) for d in (64, 128) for w in (16, 32, 64, 128)} and {s for _, _, s in seen} == {True, False}

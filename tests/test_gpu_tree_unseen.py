"""Infinity and NaN where attention of new rows does not look, in every width of a tile: tokens that no row
or not every row sees, slots behind a sequence, and the first slot of the cache, which stands in for missing tokens."""
import math

import pytest
import torch

import yirage_amd.fused as F
from tests.paged_plain import Batch
from tests.test_gpu_tree_attn import DTS, Q8, _cache
from tests.tree_plain import check_attention

pytestmark = pytest.mark.gpu

PAGE = 16
WIDTHS = pytest.mark.parametrize("news", [[1, 3], [8, 7], [15, 16], [20, 27]], ids=["16", "32", "64", "128"])
DIMS = pytest.mark.parametrize("d", [64, 128])


def _batch(lens, news):
    for seed in range(100):
        b = Batch(lens, news, PAGE, seed=seed)
        if 0 not in b.indices:  # (page 0 is nobody's)
            return b
    raise AssertionError


def _spoil(caches, scales, places, kinds=("k", "v")):
    for i, c in enumerate(caches):
        if "kv"[i] not in kinds:
            continue
        for j, (p, s) in enumerate(places):
            if not scales:
                c[p, s, :, ::2], c[p, s, :, 1::2] = math.nan, (-1) ** i * math.inf
            else:
                c.view(torch.uint8)[p, s] = 0x7f
                if j % 2:
                    list(scales.values())[i].view(torch.uint8)[p, s] = 255


def _outside(b):
    """Slots of no sequence."""
    places = [(p, s) for p in range(b.pool) if p not in b.indices for s in range(PAGE)]
    for L, e in zip(b.lens, b.kv_ptr[1:]):
        places += [(int(b.indices[e - 1]), s) for s in range((L - 1) % PAGE + 1, PAGE)]
    return places


def _slot(b, s, p):
    return int(b.indices[b.kv_ptr[s] + p // PAGE]), p % PAGE


@DTS
@Q8
@DIMS
@WIDTHS
def test_no_row_sees_it(news, d, q8, dt):
    gen = torch.Generator().manual_seed(31)
    hq, hkv, lens = 8, 2, [70 + news[0], 611]
    b = _batch(lens, news)
    q = torch.randn((b.rows, hq, d), generator=gen).to(dt)
    caches, scales, k, v = _cache(b, hkv, d, dt, q8, gen)
    mask = torch.rand((b.rows, max(news)), generator=gen) < 0.6
    hidden = [0, 2]
    mask[:, hidden] = False
    _spoil(caches, scales, _outside(b) + [_slot(b, s, L - n + j) for s, (L, n) in enumerate(zip(lens, news)) for j in hidden if j < n])
    out = F.gqa_tree_paged(q.cuda(), *caches, *b.args(), tree_mask=mask.cuda(), qo_indptr=b.qo(), **scales)
    check_attention(b, hq, hkv, q, k, v, out.cpu(), mask, torch.bfloat16 if q8 else None)


@DTS
@Q8
@DIMS
@WIDTHS
def test_the_last_row_sees_it(news, d, q8, dt):
    """V of the last new token: the rows before it are as they were, its own is not finite."""
    gen = torch.Generator().manual_seed(32)
    hq, hkv, lens = 8, 2, [70 + news[0], 611]
    b = _batch(lens, news)
    q = torch.randn((b.rows, hq, d), generator=gen).to(dt)
    caches, scales, k, v = _cache(b, hkv, d, dt, q8, gen)
    call = lambda: F.gqa_tree_paged(q.cuda(), *caches, *b.args(), qo_indptr=b.qo(), **scales).cpu()
    clean = call()
    check_attention(b, hq, hkv, q, k, v, clean, None, torch.bfloat16 if q8 else None)
    for s, L in enumerate(lens):
        _spoil(caches, scales, [_slot(b, s, L - 1)], ("v",))
    out = call()
    last = torch.zeros(b.rows, dtype=torch.bool)
    last[[news[0] - 1, b.rows - 1]] = True
    assert torch.equal(out[~last], clean[~last])
    assert not out[last].isfinite().any()


@DTS
@Q8
@DIMS
@pytest.mark.parametrize("lens", [[70, 33, 1, 300], [5000, 77], [40] * 300], ids=["short", "split", "many"])
def test_single_rows(lens, d, q8, dt):
    """Without qo_indptr: what lies behind each sequence."""
    gen = torch.Generator().manual_seed(33)
    hq, hkv = 8, 4
    b = _batch(lens, [1] * len(lens))
    q = torch.randn((b.rows, hq, d), generator=gen).to(dt)
    caches, scales, k, v = _cache(b, hkv, d, dt, q8, gen)
    _spoil(caches, scales, _outside(b))
    out = F.gqa_tree_paged(q.cuda(), *caches, *b.args(), **scales)
    check_attention(b, hq, hkv, q, k, v, out.cpu(), None, torch.bfloat16 if q8 else None)

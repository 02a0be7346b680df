"""gqa_tree_paged against 64 bits: single tokens, trees and chunks over caches in 16
bits and in e4m3, odd lengths and page sizes, masks that leave nothing, missing pages,
infinities and NaN in unseen places."""
import math

import numpy as np
import pytest
import torch

import yirage_amd.fused as F
from tests.paged_plain import Batch
from tests.tree_plain import E4M3, E8M0, check_attention, random_cache, trees, values

pytestmark = pytest.mark.gpu

DTS = pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
Q8 = pytest.mark.parametrize("q8", [False, True], ids=["16", "e4m3"])


def _cache(b, hkv, d, dt, q8, gen):
    """on the GPU: caches and scales; k, v in 64 bits"""
    if q8:
        kc, vc, ks, vs = random_cache(b.pool, b.page, hkv, d, gen, 118, 121)
        return (kc.cuda(), vc.cuda()), dict(k_scale=ks.cuda(), v_scale=vs.cuda()), values(kc, ks), values(vc, vs)
    k, v = (torch.randn((b.pool, b.page, hkv, d), generator=gen).to(dt) for _ in range(2))
    return (k.cuda(), v.cuda()), {}, k.double(), v.double()


CASES = [
    # lens, new rows, query heads, kv heads, d, page, tree
    ([1], [1], 4, 4, 64, 16, False), ([64], [1], 32, 8, 128, 64, False), ([65], [1], 32, 8, 128, 64, False),
    ([127, 1, 300, 33], [1, 1, 1, 1], 10, 2, 128, 16, False),
    ([1000], [1], 16, 1, 128, 64, False),                     # several splits, a full group
    ([5000, 77], [1, 1], 8, 2, 64, 32, False),
    ([5, 70, 16, 33], [5, 1, 0, 20], 14, 2, 64, 16, True),    # a tree without a prefix, a sequence without rows
    ([200, 131], [37, 131], 8, 1, 128, 48, True),             # odd pages
    ([90, 90], [2, 3], 4, 4, 128, 16, True),                  # one head a group
    ([700], [64], 8, 2, 128, 64, True), ([700, 650], [64, 33], 16, 2, 64, 16, True),
    ([300], [300], 4, 1, 128, 64, False), ([1030], [517], 8, 2, 64, 128, False),  # chunks
    ([513, 300], [100, 260], 10, 2, 128, 32, False),
    ([33], [9], 6, 2, 128, 1, True),                          # one token a page
    ([40 + i for i in range(70)], [1 + i % 3 for i in range(70)], 5, 1, 128, 32, True),
    ([17] * 130, [1] * 130, 2, 2, 64, 16, False),
]


@DTS
@Q8
@pytest.mark.parametrize("lens,news,hq,hkv,d,page,tree", CASES)
def test_rows(lens, news, hq, hkv, d, page, tree, q8, dt):
    print("case", len(lens), max(lens), sum(news), hq, hkv, d, page, tree, q8, dt, flush=True)
    gen = torch.Generator().manual_seed(hq + page)
    b = Batch(lens, news, page, seed=page)
    q = torch.randn((b.rows, hq, d), generator=gen).to(dt)
    caches, scales, k, v = _cache(b, hkv, d, dt, q8, gen)
    mask = trees(news, seed=2)[2] if tree else None
    args = (q.cuda(), *caches, *b.args())
    more = dict(tree_mask=None if mask is None else mask.cuda(), qo_indptr=b.qo(), **scales)
    out = F.gqa_tree_paged(*args, **more)
    check_attention(b, hq, hkv, q, k, v, out.cpu(), mask, torch.bfloat16 if q8 else None)
    for most in (1, 100000):  # how finely the work is split changes nothing but roundings
        check_attention(b, hq, hkv, q, k, v, F.gqa_tree_paged(*args, max_kv_len=most, **more).cpu(), mask, torch.bfloat16 if q8 else None)


@DTS
@Q8
def test_any_mask(q8, dt):
    """Masks that are no trees: rows that see nothing, later tokens, not themselves; wider and narrower
    than the new tokens, with a row stride."""
    gen = torch.Generator().manual_seed(5)
    hq, hkv, d, page = 8, 2, 64, 16
    b = Batch([40, 9, 100], [12, 9, 40], page)
    q = torch.randn((b.rows, hq, d), generator=gen).to(dt)
    caches, scales, k, v = _cache(b, hkv, d, dt, q8, gen)
    for width, stride in ((64, 64), (40, 57), (7, 7), (1, 3)):
        mask = torch.rand((b.rows, stride), generator=gen) < 0.4
        mask[12:15] = False   # the second sequence has no prefix: these rows see nothing
        mask = mask[:, :width]
        out = F.gqa_tree_paged(q.cuda(), *caches, *b.args(), tree_mask=mask.cuda() if stride == width else
                               torch.cat([mask, ~mask], 1).cuda()[:, :width], qo_indptr=b.qo(), **scales)
        check_attention(b, hq, hkv, q, k, v, out.cpu(), mask, torch.bfloat16 if q8 else None)
        assert (out[12:15] == 0).all()


@DTS
@Q8
@pytest.mark.parametrize("d", [64, 128])
def test_unseen_places_hold_anything(d, q8, dt):
    """Infinity and NaN in tokens that a row does not see, in slots behind the sequence and in page 0
    (what stands in for a missing token) do not reach it; in tokens that it sees they do."""
    gen = torch.Generator().manual_seed(6)
    hq, hkv, page, L, n = 8, 2, 16, 71, 20
    b = Batch([L], [n], page, seed=3)
    q = torch.randn((n, hq, d), generator=gen).to(dt)
    caches, scales, k, v = _cache(b, hkv, d, dt, q8, gen)
    ids, first = b.indices, L - n
    mask = torch.rand((n, n), generator=gen) < 0.5
    mask[:, 3] = False
    mask[:, 7] = False
    mask[4, 7] = mask[9, 11] = mask[10, 11] = True
    places = [(ids[-1], s) for s in range(L % page, page)] + [(p, s) for p in set(range(b.pool)) - set(ids.tolist()) for s in range(page)]
    unseen = lambda j: (ids[(first + j) // page], (first + j) % page)
    if q8:
        for c in caches:
            for p, s in places + [unseen(3)]:
                c.view(torch.uint8)[p, s] = 0x7f  # NaN
        for s in scales.values():
            for p, sl in places[::2] + [unseen(3)]:
                s.view(torch.uint8)[p, sl] = 255
        caches[1].view(torch.uint8)[unseen(7)] = 0xff
        scales["v_scale"].view(torch.uint8)[unseen(11)] = 255
    else:
        for i, c in enumerate(caches):
            for p, s in places + [unseen(3)]:
                c[p, s, :, ::2], c[p, s, :, 1::2] = math.nan, (-1) ** i * math.inf
        caches[1][unseen(7)] = math.inf
        caches[1][unseen(11)] = math.nan
    out = F.gqa_tree_paged(q.cuda(), *caches, *b.args(), tree_mask=mask.cuda(), qo_indptr=b.qo(), **scales).cpu()
    sees7, sees11 = mask[:, 7], mask[:, 11]
    ok = ~(sees7 | sees11)
    assert ok.sum() > 2 and out[ok].isfinite().all()
    # the rows that see them: NaN, or infinity where only infinite values are seen
    assert out[sees11].isnan().all()
    only7 = sees7 & ~sees11
    assert only7[4] or sees11[4]
    assert (out[only7].isnan().all() if q8 else (out[only7] == math.inf).all())
    # and the others as if those tokens were not there
    keep = torch.where(ok[:, None], mask, False)
    clean = [torch.nan_to_num(x, 0.0, 0.0, 0.0) for x in (k, v)]
    ref = F.gqa_tree_paged(q.cuda(), *[torch.nan_to_num(c.float(), 0.0, 0.0, 0.0).to(c.dtype) for c in caches], *b.args(), tree_mask=keep.cuda(),
                           qo_indptr=b.qo(), **{n_: torch.where(s.view(torch.uint8) == 255, 120, s.view(torch.uint8)).view(E8M0) for n_, s in scales.items()}).cpu()
    assert torch.equal(out[ok], ref[ok])
    del clean


@Q8
def test_missing_pages_and_short_tables(q8):
    """Pages outside the cache and tables too short for the length: their tokens are not seen; padded
    rows stay as they were; an empty sequence and one without pages give 0."""
    gen = torch.Generator().manual_seed(7)
    dt, hq, hkv, d, page = torch.bfloat16, 4, 1, 128, 16
    b = Batch([100, 64, 0, 50, 30], [3, 3, 0, 3, 3], page)
    rows = b.rows + 4
    q = torch.randn((rows, hq, d), generator=gen).to(dt)
    caches, scales, k, v = _cache(b, hkv, d, dt, q8, gen)
    bad = b.indices.copy()
    gone = [int(bad[1]), int(bad[b.kv_ptr[1]])]
    bad[1], bad[b.kv_ptr[1]] = -1, b.pool + 5
    ptr = b.kv_ptr.copy()
    ptr[5] = ptr[4]          # the last sequence has no pages
    ptr2 = ptr.copy()
    out = torch.full((rows, hq, d), 3.0, dtype=dt, device="cuda")
    F.gqa_tree_paged(q.cuda(), *caches, torch.from_numpy(ptr2).cuda(), torch.from_numpy(bad).cuda(), b.args()[2],
                     qo_indptr=torch.from_numpy(b.qo_ptr).cuda(), out=out, **scales)
    assert (out[b.rows:] == 3).all() and (out[b.rows - 3:b.rows] == 0).all()
    b.kv_ptr = ptr
    check_attention(b, hq, hkv, q, k, v, out.cpu(), None, torch.bfloat16 if q8 else None, skip=gone)


@DTS
def test_large_scores(dt):
    """Scores far beyond 2^20: the largest of each row takes the weight (16 bits)."""
    gen = torch.Generator().manual_seed(8)
    hq, hkv, d, page = 4, 1, 64, 16
    big = 2.0 ** 14 if dt == torch.float16 else 2.0 ** 40
    b = Batch([200], [20], page)
    q = (torch.randn((b.rows, hq, d), generator=gen) * big).to(dt).clamp(-6e4 if dt == torch.float16 else -1e30, 6e4 if dt == torch.float16 else 1e30)
    k = (torch.randn((b.pool, page, hkv, d), generator=gen) * 2.0 ** 12).to(dt).clamp(-6e4 if dt == torch.float16 else -1e30, 6e4 if dt == torch.float16 else 1e30)
    v = torch.randn(k.shape, generator=gen).to(dt)
    out = F.gqa_tree_paged(q.cuda(), k.cuda(), v.cuda(), *b.args(), qo_indptr=b.qo()).cpu()
    assert out.isfinite().all()
    ids = torch.from_numpy(b.indices).long()
    kk, vv = k[ids].flatten(0, 1)[:, 0].double(), v[ids].flatten(0, 1)[:, 0].double()
    checked = 0
    for i in range(20):
        s = q[i].double() @ kk[:181 + i].t()
        top = s.topk(2, -1).values
        # products of 64 terms in fp32: at most 2^-18 of their magnitudes apart
        sure = top[:, 0] - top[:, 1] > 2.0 ** -16 * (q[i].double().abs() @ kk[:181 + i].abs().t()).amax(-1) + 400
        for h in sure.nonzero()[:, 0].tolist():
            checked += 1
            assert torch.equal(out[i, h], vv[s[h].argmax()].to(dt))
    assert checked > 40


def test_all_scores_minus_infinity():
    """A row whose visible scores are all -inf is 0, as in the paged decode."""
    dt, b = torch.bfloat16, Batch([40], [4], 16)
    q = torch.full((4, 2, 64), 1.0).to(dt)
    k = torch.full((b.pool, 16, 1, 64), -math.inf).to(dt)
    v = torch.ones_like(k)
    out = F.gqa_tree_paged(q.cuda(), k.cuda(), v.cuda(), *b.args(), qo_indptr=b.qo())
    assert (out == 0).all()

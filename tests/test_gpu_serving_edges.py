"""The operators around a paged cache at the ends of their ranges: batches of many
sequences, some without new rows; tiles of 16, 8 and 4 rows; lists of up to 1024
pages; contexts of more pages than a table of masks holds; bounds of pages that a
call writes in part."""
import math

import pytest
import torch

import yirage_amd.fused as F
from paged_plain import Batch, norm_rotate, tables
from test_gpu_append_kv import _caches, _half_step
from test_gpu_select_pages import _reference as select_reference
from test_gpu_sparse_attn import _inputs, _lists
from test_gpu_sparse_attn import _reference as attention_reference

pytestmark = pytest.mark.gpu

DTS = pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])


def many(kind):
    """Lengths and new rows of many sequences, with their tables given whatever the rows."""
    if kind == "rows":      # few rows each, none in every fourth
        news = [i % 4 for i in range(100)]
        return [n + 37 + 9 * i for i, n in enumerate(news)], news
    if kind == "tiles":     # up to a tile each
        news = [7 * i % 17 for i in range(90)]
        return [n + 40 + 88 * i for i, n in enumerate(news)], news
    if kind == "few":
        news = [(i + 3) % 4 for i in range(130)]
        return [n + 1 + 5 * i for i, n in enumerate(news)], news
    if kind == "wide":
        news = [5 * i % 9 for i in range(120)]
        return [n + 60 + 3 * i for i, n in enumerate(news)], news
    if kind == "ones":
        return [1 + 2 * i % 301 for i in range(480)], [1] * 480
    assert False


def _qo(b):
    return torch.from_numpy(b.qo_ptr).cuda()


# ------------------------------------------------------------------ selection
def _select(lens, news, hq, hkv, d, page, top, first, last, dt):
    print("case", lens[:4], news[:4], len(lens), hq, hkv, d, page, top, first, last, dt, flush=True)
    gen = torch.Generator().manual_seed(top + page)
    b = Batch(lens, news, page, seed=top)
    q = torch.randn((b.rows, hq, d), generator=gen).to(dt)
    mid, half = torch.randn((b.pool, hkv, d), generator=gen), torch.rand((b.pool, hkv, d), generator=gen)
    bounds = torch.stack([mid - half, mid + half], 2).to(dt)
    got = F.select_pages(q.cuda(), bounds.cuda(), *b.args(), page_size=page, top_pages=top, qo_indptr=_qo(b),
                         first_pages=first, last_pages=last, max_kv_len=max(lens))
    assert torch.equal(got.cpu(), select_reference(b, q, bounds, hkv, top, first, last))


@DTS
@pytest.mark.parametrize("kind,top", [("rows", 6), ("tiles", 20), ("ones", 3)])
def test_selection_of_many_sequences(kind, top, dt):
    lens, news = many(kind)
    _select(lens, news, 4, 2, 64, 16, top, 1, 1, dt)


@DTS
@pytest.mark.parametrize("lens,news,hq,hkv,d,page,top,first,last", [
    ([1024], [450], 2, 2, 64, 1, 40, 2, 3), ([1025], [450], 2, 2, 64, 1, 40, 2, 3), ([1500, 2000], [203, 230], 4, 4, 128, 1, 100, 1, 1),
    ([2048], [400], 4, 2, 64, 1, 9, 0, 1), ([2049], [400], 2, 2, 128, 1, 9, 0, 1), ([4096], [300], 2, 2, 64, 1, 30, 1, 1),
])
def test_tiles_of_each_size(lens, news, hq, hkv, d, page, top, first, last, dt):
    _select(lens, news, hq, hkv, d, page, top, first, last, dt)


@pytest.mark.parametrize("pages", [1500, 4000])
def test_undecided_rows_of_short_tiles(pages):
    """Tiles of 8 and of 4 rows whose scores all have to be exact: alike, infinite, too large."""
    dt, d, rows = torch.bfloat16, 64, 330
    b = Batch([pages], [rows], 1)
    gen = torch.Generator().manual_seed(pages)
    q = torch.randn((rows, 2, d), generator=gen).to(dt)
    ids = torch.from_numpy(b.indices).long()
    for kind in range(3):
        bounds = torch.zeros((b.pool, 1, 2, d))
        if kind == 0:
            bounds[ids] = torch.randn((1, 1, 2, d), generator=gen).sort(2).values
            bounds[ids, 0, 1, 5] = torch.randint(0, 9, (pages,), generator=gen) * 2.0 ** -30
        else:
            bounds[ids] = torch.randn((pages, 1, 2, d), generator=gen).sort(2).values
            bounds[ids[10:20], 0, 1, 3] = math.inf if kind == 1 else 1e38
        bounds = bounds.to(dt)
        got = F.select_pages(q.cuda(), bounds.cuda(), *b.args(), page_size=1, top_pages=70, qo_indptr=_qo(b), max_kv_len=pages)
        assert torch.equal(got.cpu(), select_reference(b, q, bounds, 1, 70, 1, 1)), kind


# ------------------------------------------------------------------ attention
def _attend(b, q, k, v, pages, hkv):
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    F.gqa_sparse_paged(q.cuda(), k.cuda(), v.cuda(), *b.args(), pages.cuda(), qo_indptr=_qo(b), out=out)
    ref, tol = attention_reference(b, q, k, v, pages, hkv)
    err = (out.cpu().double() - ref).abs()
    assert (err <= tol).all(), (err - tol).max()


@DTS
@pytest.mark.parametrize("kind,hq,hkv", [("few", 8, 2), ("wide", 64, 8), ("ones", 64, 8)])
def test_attention_of_many_sequences(kind, hq, hkv, dt):
    lens, news = many(kind)
    print("case", kind, len(lens), sum(news), dt, flush=True)
    b = Batch(lens, news, 24, seed=3)
    q, k, v, gen = _inputs(b, hq, hkv, 64, dt, 4)
    _attend(b, q, k, v, _lists(b, hkv, 4, gen), hkv)


@DTS
@pytest.mark.parametrize("order", ["ascending", "shuffled", "repeated"])
@pytest.mark.parametrize("lens,news,hq,hkv,d,page,top", [
    ([2400, 900], [1, 1], 4, 2, 64, 8, 257), ([1300], [1], 8, 1, 128, 2, 600), ([16384], [1], 4, 2, 64, 16, 1024),
    ([1100, 700], [3, 2], 8, 2, 64, 1, 300),  # tiles of 3 rows
    ([1050], [2], 4, 1, 128, 1, 1024),        # a tile of one row
])
def test_long_lists(lens, news, hq, hkv, d, page, top, order, dt):
    print("case", lens, news, hq, hkv, d, page, top, order, dt, flush=True)
    b = Batch(lens, news, page, seed=top)
    q, k, v, gen = _inputs(b, hq, hkv, d, dt, top)
    pages = _lists(b, hkv, top, gen)
    if order == "shuffled":
        pages = pages[:, :, torch.randperm(top, generator=gen)].contiguous()
    elif order == "repeated":
        pages = torch.randint(-3, max(lens) // page + 3, pages.shape, generator=gen, dtype=torch.int32)
    _attend(b, q, k, v, pages, hkv)


@DTS
@pytest.mark.parametrize("lens,news,hq,hkv,d,page,top,wide", [
    ([8300], [5], 8, 2, 64, 1, 40, 0), ([8192, 8500], [3, 2], 8, 2, 64, 1, 40, 0), ([16500], [4], 8, 2, 128, 1, 30, 0),
    ([4500], [480], 64, 8, 64, 1, 6, 1), ([4300], [460], 64, 8, 64, 1, 6, 1),
])
def test_more_pages_than_a_table_of_masks(lens, news, hq, hkv, d, page, top, wide, dt):
    print("case", lens, news, hq, hkv, d, page, top, dt, flush=True)
    b = Batch(lens, news, page, seed=top)
    q, k, v, gen = _inputs(b, hq, hkv, d, dt, top)
    base = torch.randint(0, min(lens) - max(news), (hkv, top), generator=gen, dtype=torch.int32)
    pages = base.expand(b.rows, hkv, top).clone()  # the rows share half of their pages
    pages[:, :, ::2] = torch.randint(0, max(lens), pages[:, :, ::2].shape, generator=gen, dtype=torch.int32)
    _attend(b, q, k, v, pages, hkv)


# ------------------------------------------------------------------ append
@DTS
def test_bounds_of_pages_written_in_part(dt):
    """Tokens whose page is missing or whose position has no angle leave no trace in the bounds;
    what a page held before its first new slot stays in them; a page that starts anew forgets."""
    gen = torch.Generator().manual_seed(3)
    d, hkv = 64, 2
    b = Batch([40, 40, 40, 33, 25], [10, 10, 10, 1, 10], 16)
    k, v = (torch.randn((b.rows, hkv, d), generator=gen).to(dt) for _ in range(2))
    cos, sin = (t.float() for t in tables(36, d))  # positions 36 .. 39 have no angle
    before = _caches(b, hkv, d, dt, gen)
    bad = b.indices.copy()
    bad[b.kv_ptr[0] + 2] = -1            # sequence 0: tokens 32 ..
    bad[b.kv_ptr[1] + 1] = b.pool        # sequence 1: tokens 16 .. 31
    bad = bad[:-1]                       # sequence 4: the table ends before tokens 16 ..
    kc, vc, bd = (t.cuda() for t in before)
    indptr, idx, kv_len = torch.from_numpy(b.kv_ptr).cuda(), torch.from_numpy(bad).cuda(), b.args()[2]
    F.append_kv_paged(k.cuda(), v.cuda(), kc, vc, indptr, idx, kv_len, cos=cos.cuda(), sin=sin.cuda(), qo_indptr=_qo(b),
                      page_bounds=bd)
    got_k, got_b, want = kc.cpu(), bd.cpu(), before[2].clone()
    joined = 0
    for s, (L, n) in enumerate(zip(b.lens, b.news)):
        for u in range((L - n) // 16, -(-L // 16)):
            e = b.kv_ptr[s] + u
            if e >= len(bad) or not 0 <= bad[e] < b.pool:
                continue
            slots = [p % 16 for p in range(max(L - n, u * 16), min(L, (u + 1) * 16, 36))]
            if not slots:
                continue
            new = got_k[bad[e], slots]
            lo, hi = new.amin(0), new.amax(0)
            if slots[0] > 0:
                lo, hi = torch.minimum(lo, before[2][bad[e], :, 0]), torch.maximum(hi, before[2][bad[e], :, 1])
                joined += 1
            want[bad[e], :, 0], want[bad[e], :, 1] = lo, hi
    assert joined >= 3
    assert torch.equal(got_b, want)


@DTS
@pytest.mark.parametrize("which", ["both", "q", "k"])
def test_norms_without_rotation(which, dt):
    gen = torch.Generator().manual_seed(5)
    d, hq, hkv = 128, 6, 2
    b = Batch([50, 33], [20, 1], 16)
    q = torch.randn((b.rows, hq, d), generator=gen).to(dt)
    k, v = (torch.randn((b.rows, hkv, d), generator=gen).to(dt) for _ in range(2))
    qn, kn = ((1 + 0.2 * torch.randn(d, generator=gen)).to(dt) for _ in range(2))
    qn, kn = qn if which != "k" else None, kn if which != "q" else None
    kc, vc, bd = (t.cuda() for t in _caches(b, hkv, d, dt, gen))
    dev = lambda t: None if t is None else t.cuda()
    got = F.append_kv_paged(k.cuda(), v.cuda(), kc, vc, *b.args(), q=q.cuda(), q_norm=dev(qn), k_norm=dev(kn), qo_indptr=_qo(b),
                            page_bounds=bd).cpu()
    kc = kc.cpu()
    for t, p, ids in b.each_row():
        for x, w, y in ((q[t], qn, got[t]), (k[t], kn, kc[ids[p // 16], p % 16])):
            ref, mag = norm_rotate(x, w, None, None, 1e-6)
            assert ((y.double() - ref).abs() <= _half_step(ref, mag, dt)).all() if w is not None else torch.equal(y, x)


def test_more_new_rows_than_tokens():
    """A sequence of 5 tokens with 8 rows: the first three have no position."""
    dt, d = torch.bfloat16, 64
    gen = torch.Generator().manual_seed(6)
    b = Batch([5, 20], [8, 2], 16)
    q = torch.randn((b.rows, 2, d), generator=gen).to(dt)
    k, v = (torch.randn((b.rows, 2, d), generator=gen).to(dt) for _ in range(2))
    cos, sin = (t.float() for t in tables(20, d))
    kc, vc, bd = (t.cuda() for t in _caches(b, 2, d, dt, gen))
    old = vc.cpu()
    got = F.append_kv_paged(k.cuda(), v.cuda(), kc, vc, *b.args(), q=q.cuda(), cos=cos.cuda(), sin=sin.cuda(), qo_indptr=_qo(b),
                            page_bounds=bd)
    assert got[:3].isnan().all() and not got[3:].isnan().any()
    for i in range(5):
        old[b.indices[0], i] = v[3 + i]
    for i in range(2):
        old[b.indices[2], 2 + i] = v[8 + i]
    assert torch.equal(vc.cpu(), old)
    seen = kc[b.indices[0], :5].cpu()
    assert torch.equal(bd[b.indices[0], :, 0].cpu(), seen.amin(0)) and torch.equal(bd[b.indices[0], :, 1].cpu(), seen.amax(0))
    pages = F.select_pages(got, bd, *b.args(), page_size=16, top_pages=2, qo_indptr=_qo(b), max_kv_len=20)
    assert (pages[:3] == -1).all() and (pages[3:8, :, 0] == 0).all()
    out = F.gqa_sparse_paged(got, kc, vc, *b.args(), pages, qo_indptr=_qo(b))
    assert (out[:3] == 0).all() and not out[3:].isnan().any()

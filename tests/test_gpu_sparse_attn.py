"""gqa_sparse_paged against 64 bits: every group size, pages on and off the
32-token blocks, lists in any order with what counts for nothing, tiles whose
rows choose differently, values that are not finite."""
import pytest
import torch

import yirage_amd.fused as F
from tests.paged_plain import Batch, attend, attend_tolerance

pytestmark = pytest.mark.gpu

DTS = pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])


def _reference(b, q, k, v, pages, hkv):
    """Also the tolerance."""
    T, hq, d = q.shape
    G = hq // hkv
    out, tol = torch.zeros((T, hq, d), dtype=torch.float64), torch.zeros((T, hq, d), dtype=torch.float64)
    vmax = v[v.isfinite()].abs().max().item() if v.isfinite().any() else 0.0
    for t, p, ids in b.each_row():
        for h in range(hkv):
            kept = sorted({u for u in pages[t, h].tolist() if 0 <= u < len(ids) and u * b.page <= p and
                           0 <= ids[u] < b.pool})
            kk = [k[ids[u], : min(b.page, p + 1 - u * b.page), h] for u in kept]
            vv = [v[ids[u], : min(b.page, p + 1 - u * b.page), h] for u in kept]
            kk = torch.cat(kk) if kk else k[:0, 0, 0]
            vv = torch.cat(vv) if vv else v[:0, 0, 0]
            hs = slice(h * G, (h + 1) * G)
            out[t, hs], pv, a = attend(q[t, hs], kk, vv)
            tol[t, hs] = attend_tolerance(out[t, hs], pv, a, kk.shape[0], vmax, q.dtype)
    return out, tol


def _inputs(b, hq, hkv, d, dt, seed, qstd=1.0):
    gen = torch.Generator().manual_seed(seed)
    q = (qstd * torch.randn((b.rows, hq, d), generator=gen)).to(dt)
    k, v = (torch.randn((b.pool, b.page, hkv, d), generator=gen).to(dt) for _ in range(2))
    # what lies behind a sequence's last token is never read
    for L, p0 in zip(b.lens, b.kv_ptr):
        if L % b.page:
            k[b.indices[p0 + L // b.page], L % b.page:] = float("nan")
            v[b.indices[p0 + L // b.page], L % b.page:] = float("inf")
    return q, k, v, gen


def _lists(b, hkv, top, gen, own=True):
    """A random choice of the visible pages, the row's own page among them."""
    pages = torch.full((b.rows, hkv, top), -1, dtype=torch.int32)
    for t, p, ids in b.each_row():
        for h in range(hkv):
            n = p // b.page + 1
            u = torch.randperm(n, generator=gen)[:top]
            if own and n > top:
                u[0] = n - 1
            pages[t, h, : min(n, top)] = u.unique().sort().values.int() if not own else torch.tensor(sorted(set(u.tolist())) + [-1] * (min(n, top) - len(set(u.tolist()))))
    return pages


def _run(b, q, k, v, pages, **kw):
    return F.gqa_sparse_paged(q.cuda(), k.cuda(), v.cuda(), *b.args(), pages.cuda(), qo_indptr=b.qo(), **kw)


@DTS
@pytest.mark.parametrize("lens,news,hq,hkv,d,page,top", [
    ([1], [1], 1, 1, 64, 16, 1), ([33], [1], 16, 1, 128, 32, 2), ([1000, 64, 65], [1, 1, 1], 32, 8, 128, 64, 4),
    ([3000], [1], 8, 2, 128, 64, 32), ([777, 31], [1, 1], 5, 1, 64, 16, 20), ([500], [1], 14, 2, 128, 1, 100),
    ([900, 400], [1, 1], 12, 4, 64, 48, 7), ([600] * 40, [1] * 40, 8, 2, 128, 16, 9),
    ([700, 9, 33], [5, 9, 17], 8, 2, 128, 16, 6),              # tiles of 4 rows
    ([400], [37], 2, 2, 64, 32, 5), ([260, 300], [20, 1], 16, 1, 64, 64, 3),  # 16 rows, one row
    ([300, 1], [50, 1], 7, 1, 128, 24, 8), ([640], [64], 16, 2, 128, 128, 2),
    ([200], [200], 12, 4, 128, 16, 3),                         # a whole prompt
    ([700, 500], [300, 200], 16, 16, 64, 32, 3), ([400], [330], 16, 8, 128, 24, 4),  # more tiles than CUs
    ([600], [520], 32, 8, 128, 64, 4), ([450, 300], [430, 290], 40, 8, 64, 16, 5),   # tiles of 16, 12 and 4 rows
    ([300], [290], 64, 4, 128, 32, 3), ([200, 700], [1, 660], 28, 4, 64, 48, 6),
])
def test_rows(lens, news, hq, hkv, d, page, top, dt):
    print("case", lens[:4], news[:4], hq, hkv, d, page, top, dt, flush=True)
    b = Batch(lens, news, page, seed=top)
    q, k, v, gen = _inputs(b, hq, hkv, d, dt, top)
    pages = _lists(b, hkv, top, gen)
    out = _run(b, q, k, v, pages)
    ref, tol = _reference(b, q, k, v, pages, hkv)
    err = (out.cpu().double() - ref).abs()
    assert (err <= tol).all(), (err - tol).max()
    assert torch.equal(_run(b, q, k, v, pages), out)  # the same bits again


@DTS
@pytest.mark.parametrize("news", [[1, 1], [6, 3]])
def test_lists_with_what_counts_for_nothing(news, dt):
    """Any order, the same page twice, pages not yet visible, behind the table, outside the pool;
    rows that are left with nothing are 0."""
    b = Batch([300, 170], news, 16)
    b.indices[4] = -1
    b.indices[b.kv_ptr[1] + 2] = b.pool + 7
    q, k, v, gen = _inputs(b, 8, 2, 64, dt, 3)
    pages = torch.randint(-2, 25, (b.rows, 2, 12), generator=gen, dtype=torch.int32)
    pages[:, :, 5], pages[:, :, 6] = pages[:, :, 0], 2 ** 31 - 1
    pages[0, 1] = -1                      # an empty list
    pages[b.news[0], 0] = 2               # a page outside the pool alone
    out = torch.full((b.rows, 8, 64), 9.0, dtype=dt, device="cuda")
    assert _run(b, q, k, v, pages, out=out) is out
    ref, tol = _reference(b, q, k, v, pages, 2)
    assert ((out.cpu().double() - ref).abs() <= tol).all()
    assert (out[0, 4:] == 0).all() and (out[b.news[0], :4] == 0).all()


@DTS
@pytest.mark.parametrize("hq,page,before,rows,hkv", [(2, 32, 6, 14, 1), (8, 16, 6, 14, 1), (4, 24, 6, 14, 1),
                                                     (32, 32, 20, 600, 8), (64, 24, 20, 300, 8)])
def test_values_that_other_rows_see(hq, page, before, rows, hkv, dt):
    """A tile's rows read each other's pages: what a row did not choose or cannot see yet must
    not reach it, not even infinity or NaN."""
    b = Batch([max(before * page + 9, rows)], [rows], page)
    q, k, v, gen = _inputs(b, hq, hkv, 64, dt, 8)
    h = hkv - 1
    v[b.indices[1], 3, h, 5] = float("inf")
    v[b.indices[2], 2, h, 7] = float("nan")
    k[b.indices[3], 1, h, 0] = float("nan")
    L = b.lens[0]
    v[b.indices[(L - 3) // page], (L - 3) % page, h, 9] = float("-inf")  # the third last token
    pages = torch.full((b.rows, hkv, 4), -1, dtype=torch.int32)
    for t in range(b.rows):
        pages[t, :, 0] = t % 6                     # one of six pages each
        pages[t, :, 1] = (L - b.rows + t) // page  # and its own
    out = _run(b, q, k, v, pages).cpu().double()
    ref, tol = _reference(b, q, k, v, pages, hkv)
    fin = ref.isfinite()
    assert torch.equal(out.isfinite(), fin)
    assert torch.equal(out.isnan(), ref.isnan())
    assert ((out - ref).abs()[fin] <= tol[fin]).all()


@DTS
def test_sharp_and_flat_softmax(dt):
    """Scores far apart (one weight of 1), and 4000 weights of 1 / 4000 below one 40 times as large."""
    b = Batch([4096], [1], 64)
    for qstd in (30.0, 0.0):
        q, k, v, gen = _inputs(b, 4, 1, 128, dt, 9, qstd)
        pages = torch.arange(64, dtype=torch.int32).view(1, 1, 64)
        out = _run(b, q, k, v, pages).cpu().double()
        ref, tol = _reference(b, q, k, v, pages, 1)
        assert ((out - ref).abs() <= tol).all()


@DTS
def test_all_pages_agree_with_the_paged_decode(dt):
    b = Batch([1000, 130], [1, 1], 64)
    q, k, v, gen = _inputs(b, 32, 8, 128, dt, 10)
    pages = torch.arange(16, dtype=torch.int32).expand(2, 8, 16).contiguous()
    out = _run(b, q, k, v, pages).double()
    dense = F.gqa_decode_paged(q.cuda(), k.cuda(), v.cuda(), *b.args()).double()
    _, tol = _reference(b, q, k, v, pages, 8)
    assert ((out - dense).abs().cpu() <= 2 * tol).all()


def test_padded_rows_are_left_alone():
    dt = torch.bfloat16
    b = Batch([100, 50], [5, 3], 16)
    q, k, v, gen = _inputs(b, 8, 2, 64, dt, 11)
    pages = _lists(b, 2, 4, gen)
    q = torch.cat([q, q[:3]])
    pages = torch.cat([pages, pages[:3]])
    out = torch.full(q.shape, 5.0, dtype=dt, device="cuda")
    _run(b, q, k, v, pages, out=out)
    ref, tol = _reference(b, q[:8], k, v, pages[:8], 2)
    assert ((out[:8].cpu().double() - ref).abs() <= tol).all()
    assert (out[8:] == 5).all()


# Rows enough for four groups of them to a tile.


@DTS
@pytest.mark.parametrize("lens,news,hq,hkv,d,page,top", [
    ([1100], [1010], 32, 8, 128, 64, 4), ([400, 360], [390, 310], 40, 8, 64, 16, 5), ([300], [250], 128, 8, 64, 64, 3),
    ([600, 500], [560, 440], 28, 4, 128, 48, 6), ([1010], [1010], 32, 8, 64, 128, 2),
])
def test_rows_of_wide_tiles(lens, news, hq, hkv, d, page, top, dt):
    test_rows(lens, news, hq, hkv, d, page, top, dt)


@DTS
@pytest.mark.parametrize("hq,page,before,rows,hkv", [(64, 24, 20, 480, 8), (32, 64, 20, 1000, 8)])
def test_values_that_other_rows_of_wide_tiles_see(hq, page, before, rows, hkv, dt):
    test_values_that_other_rows_see(hq, page, before, rows, hkv, dt)


@DTS
def test_wide_tiles_with_lists_that_count_for_nothing(dt):
    """Any order, the same page twice, pages not yet visible, behind the table, outside the pool."""
    b = Batch([900, 300], [390, 100], 24)
    b.indices[4] = -1
    b.indices[b.kv_ptr[1] + 2] = b.pool + 7
    q, k, v, gen = _inputs(b, 64, 8, 64, dt, 3)
    pages = torch.randint(-2, 45, (b.rows, 8, 12), generator=gen, dtype=torch.int32)
    pages[:, :, 5], pages[:, :, 6] = pages[:, :, 0], 2 ** 31 - 1
    pages[0, 1] = -1                      # an empty list
    pages[b.news[0], 0] = 2               # a page outside the pool alone
    out = torch.full((b.rows, 64, 64), 9.0, dtype=dt, device="cuda")
    assert _run(b, q, k, v, pages, out=out) is out
    ref, tol = _reference(b, q, k, v, pages, 8)
    assert ((out.cpu().double() - ref).abs() <= tol).all()
    assert (out[0, 8:16] == 0).all() and (out[b.news[0], :8] == 0).all()

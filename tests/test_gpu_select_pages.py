"""select_pages against 64 bits: the lists are whole numbers and have to be equal,
ties included."""
import pytest
import torch

import yirage_amd.fused as F
from tests.paged_plain import Batch, score, select

pytestmark = pytest.mark.gpu


def _reference(b, q, bounds, hkv, top, first, last, max_pages=1 << 30, ids_of=None):
    T, hq, d = q.shape
    G = hq // hkv
    out = torch.full((T, hkv, top), -1, dtype=torch.int32)
    for t, p, ids in b.each_row():
        ids = ids if ids_of is None else ids_of(ids)
        n = min(p // b.page + 1, len(ids), max_pages) if p >= 0 else 0
        for h in range(hkv):
            s = []
            if n:
                at = torch.from_numpy(ids[:n]).long()
                ok = (at >= 0) & (at < b.pool)
                sc = score(q[t, h * G:(h + 1) * G], bounds[at.clamp(0, b.pool - 1), h, 0], bounds[at.clamp(0, b.pool - 1), h, 1])
                s = torch.where(ok, sc, float("nan")).tolist()
            take = select(s, n, top, first, last)
            out[t, h, : len(take)] = torch.tensor(take, dtype=torch.int32)
    return out


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("lens,news,hq,hkv,d,page,top,first,last", [
    ([1], [1], 4, 4, 64, 16, 4, 1, 1), ([64, 65, 1000], [1, 1, 1], 32, 8, 128, 64, 6, 1, 1),
    ([4097], [1], 8, 1, 128, 16, 32, 1, 2), ([700, 9, 33], [3, 9, 17], 10, 2, 64, 16, 8, 2, 3),
    ([300], [300], 4, 2, 128, 16, 5, 0, 1), ([2000, 1300], [40, 5], 16, 1, 64, 1, 64, 4, 8),
    ([900], [20], 14, 2, 128, 128, 20, 1, 1),       # fewer pages than asked for
    ([5000] * 3, [1] * 3, 2, 2, 64, 48, 3, 1, 2),   # nothing left to choose
    ([2500], [130], 8, 2, 128, 16, 33, 1, 1),
    ([20000], [1], 4, 1, 64, 16, 400, 1, 1), ([16384], [1], 1, 1, 64, 1, 900, 1, 1), ([16384], [2], 2, 2, 64, 1, 16384, 1, 1),
    ([16000, 9000], [1, 20], 2, 1, 64, 1, 8, 2, 2), ([5000, 4000], [33, 2], 8, 4, 128, 16, 16, 1, 1),
])
def test_lists(lens, news, hq, hkv, d, page, top, first, last, dt):
    print("case", lens, news, hq, hkv, d, page, top, first, last, dt, flush=True)
    gen = torch.Generator().manual_seed(top + page)
    b = Batch(lens, news, page, seed=top)
    q = torch.randn((b.rows, hq, d), generator=gen).to(dt)
    mid, half = torch.randn((b.pool, hkv, d), generator=gen), torch.rand((b.pool, hkv, d), generator=gen)
    bounds = torch.stack([mid - half, mid + half], 2).to(dt)
    got = F.select_pages(q.cuda(), bounds.cuda(), *b.args(), page_size=page, top_pages=top, qo_indptr=b.qo(),
                         first_pages=first, last_pages=last, max_kv_len=max(lens))
    ref = _reference(b, q, bounds, hkv, top, first, last)
    assert torch.equal(got.cpu(), ref)
    # the bound on the lengths may be larger than they are, or come from them
    again = F.select_pages(q.cuda(), bounds.cuda(), *b.args(), page_size=page, top_pages=top, qo_indptr=b.qo(),
                           first_pages=first, last_pages=last,
                           max_kv_len=min(max(lens) + 5 * page, 16384 * page))
    assert torch.equal(again, got)
    none = F.select_pages(q.cuda(), bounds.cuda(), *b.args(), page_size=page, top_pages=top, qo_indptr=b.qo(),
                          first_pages=first, last_pages=last)
    assert torch.equal(none, got)


@pytest.mark.parametrize("rows", [1, 7, 40])
def test_ties_zeros_and_close_scores(rows):
    """Equal pages tie to the lower number, -0 equals 0, scores one unit in the last place of 40
    bits apart are told apart."""
    dt, d, page, n = torch.float16, 64, 16, 300
    b = Batch([n * page], [rows], page)
    gen = torch.Generator().manual_seed(5)
    q = torch.randn((b.rows, 2, d), generator=gen).to(dt)
    for kind in range(4):
        bounds = torch.zeros((b.pool, 1, 2, d))
        ids = torch.from_numpy(b.indices).long()
        if kind == 0:    # four kinds of page
            bounds[ids] = torch.randn((4, 1, 2, d), generator=gen).sort(2).values[torch.arange(n) % 4]
        elif kind == 1:  # zeros of both signs
            bounds[ids[::2]] = -0.0
        elif kind == 2:  # large sums that differ by little
            bounds[..., 0] = 1000.0
            bounds[ids, 0, :, 1] = (torch.randperm(n, generator=gen) * 2.0 ** -24)[:, None]
        else:            # infinities and NaN
            bounds[ids] = torch.randn((n, 1, 2, d), generator=gen).sort(2).values
            bounds[ids[10:20], 0, 1, 3] = float("inf")
            bounds[ids[30:40], 0, 0, 3] = float("-inf")
            bounds[ids[50:60], 0, 0, 7] = float("nan")
            bounds[ids[70:80], 0, 0], bounds[ids[70:80], 0, 1] = float("inf"), float("-inf")
        bounds = bounds.to(dt)
        got = F.select_pages(q.cuda(), bounds.cuda(), *b.args(), page_size=page, top_pages=37, qo_indptr=b.qo(),
                             max_kv_len=n * page)
        assert torch.equal(got.cpu(), _reference(b, q, bounds, 1, 37, 1, 1)), kind


@pytest.mark.parametrize("news", [[1, 1, 1], [4, 1, 30]])
def test_missing_pages_and_short_bounds(news):
    """Ids outside the pool rank last, a short page table or max_kv_len hides what lies behind,
    rows behind the last sequence are left alone."""
    gen = torch.Generator().manual_seed(6)
    dt, d, page = torch.bfloat16, 64, 16
    b = Batch([400, 300, 350], news, page)
    b.indices[3:9] = [-1, b.pool, 1 << 30, -5, b.pool + 1, -(1 << 31)]
    pad = 0 if max(news) == 1 else 3
    q = torch.randn((b.rows + pad, 4, d), generator=gen).to(dt)
    bounds = torch.randn((b.pool, 2, 2, d), generator=gen).sort(2).values.to(dt)
    out = torch.full((b.rows + pad, 2, 20), 99, dtype=torch.int32, device="cuda")
    F.select_pages(q.cuda(), bounds.cuda(), *b.args(), page_size=page, top_pages=20, qo_indptr=b.qo(),
                   max_kv_len=320, out=out)
    assert torch.equal(out[: b.rows].cpu(), _reference(b, q[: b.rows], bounds, 2, 20, 1, 1, max_pages=20))
    assert (out[b.rows:] == 99).all()
    ptr, idx, lens = b.args()
    got = F.select_pages(q.cuda(), bounds.cuda(), ptr, idx[:30], lens, page_size=page, top_pages=6,
                         qo_indptr=b.qo(), max_kv_len=400)
    assert torch.equal(got[: b.news[0]].cpu(), _reference(b, q[: b.rows], bounds, 2, 6, 1, 1)[: b.news[0]])
    assert int(got[b.news[0]: b.news[0] + b.news[1]].max()) < 30 - int(ptr[1])  # the second sequence lost pages
    assert (got[b.news[0] + b.news[1]: b.rows] == -1).all()                     # the third all of them


# Rows enough for tiles of them (the ones above are mostly taken row by row).


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("lens,news,hq,hkv,d,page,top,first,last", [
    ([4800], [700], 4, 1, 64, 16, 33, 1, 1), ([900, 5000, 40], [300, 420, 40], 14, 2, 128, 16, 16, 1, 2),
    ([2200], [450], 2, 2, 64, 1, 40, 2, 3),          # 8 rows a tile
    ([300, 3900], [200, 330], 4, 4, 128, 1, 20, 1, 1),  # 4 rows a tile
    ([9000], [400], 4, 4, 64, 16, 130, 3, 4),        # more pages taken than a wave has lanes
    ([6000], [700], 16, 2, 128, 64, 8, 0, 1), ([1000], [600], 8, 8, 64, 16, 60, 1, 1),
])
def test_tiles(lens, news, hq, hkv, d, page, top, first, last, dt):
    test_lists(lens, news, hq, hkv, d, page, top, first, last, dt)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("top", [20, 100])
@pytest.mark.parametrize("kind", ["kinds", "zeros", "groups", "all alike", "special", "scales", "small"])
def test_tiles_near_the_border(kind, top, dt):
    """Scores that fp32 cannot tell apart, equal ones, and rows beyond its range."""
    print("case", kind, top, dt, flush=True)
    d, page, n, rows = 64, 16, 300, 700
    b = Batch([n * page], [rows], page)
    gen = torch.Generator().manual_seed(top)
    q = torch.randn((b.rows, 2, d), generator=gen).to(dt)
    ids = torch.from_numpy(b.indices).long()
    bounds = torch.zeros((b.pool, 1, 2, d))
    base = lambda k: torch.randn((k, 1, 2, d), generator=gen).sort(2).values
    if kind == "kinds":
        bounds[ids] = base(4)[torch.arange(n) % 4]
    elif kind == "zeros":
        bounds[ids[::2]] = -0.0
    elif kind in ("groups", "all alike"):  # groups of 20 (of all) that differ in one tiny channel
        bounds[ids] = base(15 if kind == "groups" else 1).repeat_interleave(20 if kind == "groups" else n, 0)
        tiny = 2.0 ** -24 if dt is torch.float16 else 2.0 ** -30
        bounds[ids, 0, 1, 5] = (torch.randint(0, 9, (n,), generator=gen) * tiny).float()
    elif kind == "special":
        bounds[ids] = base(n)
        bounds[ids[10:20], 0, 1, 3] = float("inf")
        bounds[ids[30:40], 0, 0, 3] = float("-inf")
        bounds[ids[50:60], 0, 0, 7] = float("nan")
    elif kind == "scales":  # (what f16 cannot hold is infinite or zero)
        bounds[ids] = base(n)
        q = (q.float() * 10.0 ** torch.linspace(-36, 36, rows)[:, None, None]).to(dt)
        q[::50] = 0
    else:                   # bounds and q at the bottom of the type's range
        bounds[ids] = base(n) * (2.0 ** -20 if dt is torch.float16 else 2.0 ** -130)
        q = (q.float() * 2.0 ** -16).to(dt)
    bounds = bounds.to(dt)
    got = F.select_pages(q.cuda(), bounds.cuda(), *b.args(), page_size=page, top_pages=top, qo_indptr=b.qo(),
                         max_kv_len=n * page)
    assert torch.equal(got.cpu(), _reference(b, q, bounds, 1, top, 1, 1))


def test_tiles_with_missing_pages_and_rows_left_alone():
    """Ids outside the pool rank last, max_kv_len hides what lies behind, rows behind the last
    sequence are left as they were, two streams at once."""
    dt, d, page, rows = torch.bfloat16, 64, 16, 600
    b = Batch([4800, 700], [rows, 100], page)
    gen = torch.Generator().manual_seed(9)
    q = torch.randn((b.rows + 5, 4, d), generator=gen).to(dt)
    bounds = torch.randn((b.pool, 2, 2, d), generator=gen).sort(2).values.to(dt)
    whole = b.indices.copy()
    b.indices[3:9] = [-1, b.pool, 1 << 30, -5, b.pool + 1, -(1 << 31)]
    ref = _reference(b, q[: b.rows], bounds, 2, 20, 1, 1, max_pages=280)
    bad = b.args()
    b.indices = whole
    ref2 = _reference(b, q[: b.rows], bounds, 2, 20, 1, 1)
    good, qd, bd, streams, outs = b.args(), q.cuda(), bounds.cuda(), [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for i in range(4):
        with torch.cuda.stream(streams[i % 2]):
            out = torch.full((b.rows + 5, 2, 20), 99, dtype=torch.int32, device="cuda")
            table, most = (bad, 280 * page) if i % 2 else (good, 4800)
            F.select_pages(qd, bd, *table, page_size=page, top_pages=20, qo_indptr=b.qo(), max_kv_len=most, out=out)
            outs.append(out)
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        assert torch.equal(out[: b.rows].cpu(), ref if i % 2 else ref2), i
        assert (out[b.rows:] == 99).all()


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("offset,spread", [(2.0, 0.5), (8.0, 0.1), (64.0, 0.25), (500.0, 1.0)])
def test_tiles_of_scores_that_cancel(offset, spread, dt):
    """Keys around a common value: sums of large terms of both signs, close to one another."""
    print("case", offset, spread, dt, flush=True)
    d, page, n, rows = 128, 16, 260, 720
    b = Batch([n * page], [rows], page)
    gen = torch.Generator().manual_seed(int(offset))
    q = torch.randn((b.rows, 3, d), generator=gen).to(dt)
    sign = torch.randint(0, 2, (1, 1, 1, d), generator=gen) * 2 - 1
    bounds = (offset * sign + spread * torch.randn((b.pool, 1, 2, d), generator=gen)).sort(2).values.to(dt)
    for top in (9, 40):
        got = F.select_pages(q.cuda(), bounds.cuda(), *b.args(), page_size=page, top_pages=top, qo_indptr=b.qo(),
                             max_kv_len=n * page)
        assert torch.equal(got.cpu(), _reference(b, q, bounds, 1, top, 1, 1))

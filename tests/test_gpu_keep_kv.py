"""keep_kv_paged against moves made one after another on the host: paths over page
borders, 16 and 8 bits, bounds, bad entries, missing pages."""
import pytest
import torch

import yirage_amd.fused as F
from tests.paged_plain import Batch
from tests.tree_plain import E4M3, random_cache

pytestmark = pytest.mark.gpu

I32 = dict(dtype=torch.int32)


def _keep(b, tensors, bounds, path, ids):
    """tensors [pool, page, ...] moved on the host; returns the new lengths"""
    lens = []
    for s, (L, n) in enumerate(zip(b.lens, b.news)):
        last, j, pages = -1, 0, ids[b.kv_ptr[s]:b.kv_ptr[s + 1]]
        where = lambda p: (int(pages[p // b.page]), p % b.page) if 0 <= p and p // b.page < len(pages) and 0 <= pages[p // b.page] < b.pool else None
        for p in path[s].tolist():
            if p <= last or p >= n:
                break
            src, dst = where(L - n + p), where(L - n + j)
            if src and dst:
                for t in tensors:
                    t[dst] = t[src]
                if bounds is not None:
                    key = tensors[0][dst].float()
                    lo, hi = bounds[dst[0], :, 0].float(), bounds[dst[0], :, 1].float()
                    bounds[dst[0], :, 0], bounds[dst[0], :, 1] = torch.fmin(lo, key), torch.fmax(hi, key)
            last, j = p, j + 1
        lens.append(L - n + j)
    return lens


@pytest.mark.parametrize("kind", ["f16", "bf16", "bf16 bounds", "e4m3"])
@pytest.mark.parametrize("lens,news,hkv,d,page,depth", [
    ([1], [1], 1, 64, 16, 1), ([20], [8], 8, 128, 16, 5), ([100, 40, 7], [30, 0, 7], 2, 64, 16, 20),
    ([70, 33], [64, 17], 3, 128, 48, 40), ([50 + i for i in range(70)], [1 + i % 9 for i in range(70)], 1, 64, 32, 6),
    ([90], [40], 40, 128, 1, 12),
])
def test_paths(lens, news, hkv, d, page, depth, kind):
    print("case", len(lens), max(lens), sum(news), hkv, d, page, depth, kind, flush=True)
    gen = torch.Generator().manual_seed(page + depth)
    b = Batch(lens, news, page, seed=2)
    path = torch.full((len(lens), depth), -1, **I32)
    for s, n in enumerate(news):
        some = torch.randperm(n, generator=gen)[: min(n, int(torch.randint(0, depth + 1, (1,), generator=gen)))].sort().values
        path[s, : len(some)] = some.int()
    if kind == "e4m3":
        cache, bounds = list(random_cache(b.pool, page, hkv, d, gen)), None
        raw = [t.view(torch.uint8) for t in cache]
    else:
        dt = torch.float16 if kind == "f16" else torch.bfloat16
        cache = [torch.randn((b.pool, page, hkv, d), generator=gen).to(dt) for _ in range(2)]
        raw, bounds = [t.view(torch.int16) for t in cache], None
        if kind.endswith("bounds"):
            bounds = torch.stack([cache[0].amin(1), cache[0].amax(1)], 2) * 0.25
            cache[0][b.indices[0], 0, 0, 0] = float("nan")
    dev = [t.cuda() for t in cache]
    dev_bounds = None if bounds is None else bounds.cuda()
    scales = dict(k_scale=dev[2], v_scale=dev[3]) if kind == "e4m3" else {}
    got = F.keep_kv_paged(dev[0], dev[1], *b.args(), path.cuda(), qo_indptr=b.qo(), page_bounds=dev_bounds, **scales)
    want = _keep(b, cache if bounds is not None else raw, bounds, path, b.indices)
    assert got.tolist() == want
    for t, r in zip(dev, raw):
        assert torch.equal(t.cpu().view(r.dtype), r)
    if bounds is not None:
        assert torch.equal(dev_bounds.cpu(), bounds)


def test_entries_that_end_a_path_and_missing_pages():
    gen = torch.Generator().manual_seed(4)
    b = Batch([40] * 6, [20] * 6, 16, seed=5)
    path = torch.tensor([[2, 5, 5, 9], [2, 5, 4, 9], [20, 1, 2, 3], [-5, 1, 2, 3], [0, 1, 2, 3], [1, 3, 2 ** 31 - 1, 4]], **I32)
    ids = b.indices.copy()
    ids[b.kv_ptr[4] + 1], ids[b.kv_ptr[5] + 1] = -1, b.pool  # slots 16 .. 31 of the last two
    cache = [torch.randn((b.pool, 16, 2, 64), generator=gen).half() for _ in range(2)]
    dev = [t.cuda() for t in cache]
    ptr, _, lens = b.args()
    out = torch.zeros(6, dtype=torch.int32, device="cuda")
    got = F.keep_kv_paged(*dev, ptr, torch.from_numpy(ids).cuda(), lens, path.cuda(), qo_indptr=b.qo(), out=out)
    assert got is out and got.tolist() == _keep(b, cache, None, path, ids)
    for t, r in zip(dev, cache):
        assert torch.equal(t.cpu(), r)
    assert lens.tolist() == b.lens


def test_without_qo_indptr():
    """One new token a sequence: kept or not."""
    b = Batch([5, 9], [1, 1], 16)
    cache = torch.zeros((b.pool, 16, 1, 64), dtype=torch.float16, device="cuda")
    got = F.keep_kv_paged(cache, cache.clone(), *b.args(), torch.tensor([[0], [-1]], device="cuda", **I32))
    assert got.tolist() == [5, 8]

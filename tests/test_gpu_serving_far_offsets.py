"""The serving operators on caches, bounds and logits of more than 2^32 elements: the
pages and rows in use lie at both ends."""
import pytest
import torch

import yirage_amd.fused as F
from paged_plain import Batch, attend, attend_tolerance, score, select
from test_gpu_logprobs import _check as check_logprobs

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def give_back():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("news", [[1, 1], [3, 5]])
def test_cache_and_bounds(news):
    dt, hkv, hq, d, page, pool = torch.bfloat16, 8, 16, 128, 1, (1 << 22) + 64  # 2^32 + 2^16 elements a cache
    lens, top = [60, 50], 12
    b = Batch(lens, news, page, seed=2)
    # pages below 2^21 bounds (2^32 elements), around that and at the very end
    ids = torch.cat([torch.arange(7), (1 << 21) - 20 + torch.arange(40), pool - 63 + torch.arange(63)])
    gen = torch.Generator().manual_seed(4)
    b.pool, b.indices = pool, ids[torch.randperm(110, generator=gen)].to(torch.int32).numpy()
    kc, vc = (torch.empty((pool, page, hkv, d), dtype=dt, device="cuda") for _ in range(2))
    bd = torch.empty((pool, hkv, 2, d), dtype=dt, device="cuda")
    assert kc.numel() > 1 << 32 and bd.numel() > 1 << 33
    at = torch.from_numpy(b.indices).long().cuda()
    kc[at] = torch.randn((110, page, hkv, d), generator=gen).to(dt).cuda()
    vc[at] = torch.randn((110, page, hkv, d), generator=gen).to(dt).cuda()
    bd[at, :, 0], bd[at, :, 1] = kc[at, 0], kc[at, 0]
    q = torch.randn((b.rows, hq, d), generator=gen).to(dt)
    k, v = (torch.randn((b.rows, hkv, d), generator=gen).to(dt) for _ in range(2))
    F.append_kv_paged(k.cuda(), v.cuda(), kc, vc, *b.args(), qo_indptr=b.qo(), page_bounds=bd)
    pages = F.select_pages(q.cuda(), bd, *b.args(), page_size=page, top_pages=top, qo_indptr=b.qo(), max_kv_len=64)
    out = F.gqa_sparse_paged(q.cuda(), kc, vc, *b.args(), pages, qo_indptr=b.qo()).cpu().double()
    keys, values, low, high = (t.cpu() for t in (kc[at, 0], vc[at, 0], bd[at, :, 0], bd[at, :, 1]))
    pages = pages.cpu()
    for s, (L, n) in enumerate(zip(lens, news)):
        p0 = int(b.kv_ptr[s])
        for i in range(n):
            t, p = int(b.qo_ptr[s]) + i, L - n + i
            assert torch.equal(keys[p0 + p], k[t]) and torch.equal(values[p0 + p], v[t])
            assert torch.equal(low[p0 + p], k[t]) and torch.equal(high[p0 + p], k[t])
            for h in range(hkv):
                qh = q[t, 2 * h: 2 * h + 2]
                want = select(score(qh, low[p0: p0 + p + 1, h], high[p0: p0 + p + 1, h]).tolist(), p + 1, top, 1, 1)
                assert pages[t, h].tolist() == want
                seen = torch.tensor(want) + p0
                ref, pv, a = attend(qh, keys[seen, h], values[seen, h])
                tol = attend_tolerance(ref, pv, a, len(want), values.abs().max().item(), dt)
                assert ((out[t, 2 * h: 2 * h + 2] - ref).abs() <= tol).all()


def test_logits():
    rows, n = 33000, 131072  # 2^32 + 2^24 elements and more
    x = torch.empty((rows, n), dtype=torch.bfloat16, device="cuda")
    assert x.numel() > 1 << 32
    gen = torch.Generator().manual_seed(5)
    some = torch.tensor([0, 1, 16383, 16384, 32767, 32768, rows - 1])
    own = (2 * torch.randn((len(some), n), generator=gen)).bfloat16()
    x[some.cuda()] = own.cuda()
    tok = torch.randint(0, n, (rows,), generator=gen)
    got = F.token_logprobs(x, tok.cuda(), top_n=3)
    check_logprobs(own, tok[some], 3, tuple(t[some.cuda()] for t in got))

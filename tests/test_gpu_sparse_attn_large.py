"""gqa_sparse_paged where scores are very large: keys and queries of few bits, so scores are
exact, and the tokens with the largest share the weight evenly."""
import pytest
import torch

import yirage_amd.fused as F
from tests.paged_plain import Batch

pytestmark = pytest.mark.gpu


def _run(lens, news, hq, hkv, d, page, top, dt, exps, seed=0):
    gen = torch.Generator().manual_seed(seed)
    b = Batch(lens, news, page, seed=1)
    v = torch.randn((b.pool, page, hkv, d), generator=gen).to(dt)
    pages = torch.full((b.rows, hkv, top), -1, dtype=torch.int32)
    for t, p, ids in b.each_row():
        n = p // page + 1
        pages[t, :, : min(n, top)] = torch.arange(n - min(n, top), n, dtype=torch.int32)
    best = torch.rand((b.pool, page, hkv), generator=gen) < 0.05  # the keys with the largest scores
    vd = v.double()
    for e in exps:
        k = torch.where(best, 3 * 2.0 ** (e - 1), 2.0 ** e)[..., None].expand(b.pool, page, hkv, d).to(dt)
        q = torch.full((b.rows, hq, d), 5 * 2.0 ** (e - 2)).to(dt)  # (15 2^x log2 e has no 24-bit value)
        assert k.isfinite().all() and q.isfinite().all()
        got = F.gqa_sparse_paged(q.cuda(), k.contiguous().cuda(), v.cuda(), *b.args(), pages.cuda(), qo_indptr=b.qo()).cpu().double()
        for t, p, ids in b.each_row():
            for h in range(hkv):
                kept = [u for u in pages[t, h].tolist() if u >= 0]
                seen = torch.cat([vd[ids[u], : min(page, p + 1 - u * page), h] for u in kept])
                w = torch.cat([best[ids[u], : min(page, p + 1 - u * page), h] for u in kept])
                w = w if w.any() else ~w
                if (~w).any():  # the others are behind by far more than fp32's exponents
                    assert d * 5 * 2.0 ** (2 * e - 3) / d ** 0.5 > 1000
                ref, mag = seen[w].mean(0), seen[w].abs().mean(0)
                half = torch.finfo(dt).eps / 2
                # the weights' half step, the sums in fp32 and exp2 (2^-20), the result's half step
                tol = (half + 2.0 ** -20) * mag + half * ref.abs() + 2.0 ** -25
                assert ((got[t, h * (hq // hkv): (h + 1) * (hq // hkv)] - ref).abs() <= tol).all(), (e, t, h)


# f16's P leaves its range from scores of 2^24 on, bf16's from 2^31
EXPS = {torch.float16: [8, 10, 11, 12, 13, 14, 15], torch.bfloat16: [8, 12, 14, 15, 16, 17, 18, 19, 20, 24, 30, 45, 58]}


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("lens,news,hq,hkv,d,page,top", [
    ([700, 65], [1, 1], 8, 2, 128, 64, 8),         # a decode step, split
    ([700, 65], [1, 1], 8, 2, 64, 16, 30),
    ([300, 170], [9, 40], 8, 2, 64, 48, 4),        # tiles of rows
    ([1100], [1010], 32, 8, 64, 64, 2),            # wide tiles
    ([400, 360], [390, 310], 40, 8, 64, 16, 3),
])
def test_large_scores(lens, news, hq, hkv, d, page, top, dt):
    print("case", lens, news, hq, hkv, d, page, top, dt, flush=True)
    exps = EXPS[dt] if max(news) < 300 else EXPS[dt][::3]
    _run(lens, news, hq, hkv, d, page, top, dt, exps)

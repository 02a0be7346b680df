"""Attention over e4m3 caches whose scales change along a sequence, in every width of a tile, within a
wave, over the waves of a workgroup and over the parts of a split tile."""
import pytest
import torch

import yirage_amd.fused as F
from tests.paged_plain import Batch
from tests.test_gpu_tree_edges import DTS, WIDTHS, _check
from tests.tree_plain import E4M3, E8M0, power, random_cache, values

pytestmark = pytest.mark.gpu


def _scales(b, page, hkv, front, back, at):
    """Scale bytes [pool, page, hkv]: `front` before position at[s] of sequence s, `back` from there on."""
    vs = torch.full((b.pool, page, hkv), front, dtype=torch.uint8)
    for s, first in enumerate(at):
        p = torch.arange(first, b.lens[s])
        ids = torch.from_numpy(b.indices[b.kv_ptr[s]:b.kv_ptr[s + 1]]).long()
        vs[ids[p // page], p % page] = back
    return vs


@WIDTHS
@pytest.mark.parametrize("back", [215, 230])
@pytest.mark.parametrize("front", [1, 60, 90])
@pytest.mark.parametrize("kind", ["half", "few", "split"])
def test_scales_that_grow(kind, front, back, news, hq, d):
    """Tokens of V's smallest scales (or zeros) first, then some up to 2^229 above: the first ones' weights stay
    in the sum.  half: every wave has both kinds; few: one block has the large ones; split: parts of one tile.
    (bf16: 16 bits of the other kind do not hold such results.)"""
    dt, hkv, page = torch.bfloat16, 2, 16
    lens = [9000, 700] if kind == "split" else [330, 700]
    at = [(L - n) // 2 if kind == "half" else L - n - 7 for L, n in zip(lens, news)]
    if kind == "split":
        at = [4500, 650]
    print("case", kind, front, back, news, hq, d, flush=True)
    gen = torch.Generator().manual_seed(21)
    b = Batch(lens, news, page, seed=5)
    q = torch.randn((b.rows, hq, d), generator=gen).to(dt)
    kc, vc, ks, _ = random_cache(b.pool, page, hkv, d, gen, 118, 120)
    vs = _scales(b, page, hkv, front, back, at)
    if front == 1:
        vc = torch.where((vs == 1)[..., None], 0, vc.float()).to(E4M3)
    vs = vs.view(E8M0)
    k, v = values(kc, ks), values(vc, vs)
    out = F.gqa_tree_paged(q.cuda(), kc.cuda(), vc.cuda(), *b.args(), qo_indptr=b.qo(), k_scale=ks.cuda(), v_scale=vs.cuda()).cpu()
    assert out.isfinite().all() and (out != 0).any()
    _check(b, q, k, v, out, None, 127)


UNSEEN = pytest.mark.parametrize("news,hq,d", [([3, 2], 8, 128), ([7, 1], 8, 64), ([14, 3], 8, 128), ([40, 70], 8, 64)],
                                 ids=["16", "32", "64", "128"])


@DTS
@UNSEEN
@pytest.mark.parametrize("byte", [160, 215, 254])
def test_scales_of_unseen_tokens(byte, news, hq, d, dt):
    """A token's scale, however large, is nothing to a row that does not see it: neither where no row sees the
    token nor where another row does."""
    print("case", byte, news, hq, d, dt, flush=True)
    gen = torch.Generator().manual_seed(22)
    hkv, page, lens = 2, 16, [330, 700]
    b = Batch(lens, news, page, seed=5)
    q = torch.randn((b.rows, hq, d), generator=gen).to(dt)
    kc, vc, ks, vs = random_cache(b.pool, page, hkv, d, gen, 112, 121)
    mask = torch.rand((b.rows, max(news)), generator=gen) < 0.5
    mask[:, 0] = False
    for s, (L, n) in enumerate(zip(lens, news)):  # each sequence's first new token
        vs.view(torch.uint8)[b.indices[b.kv_ptr[s] + (L - n) // page], (L - n) % page] = byte
    args = (q.cuda(), kc.cuda(), vc.cuda(), *b.args())
    more = dict(qo_indptr=b.qo(), k_scale=ks.cuda(), v_scale=vs.cuda())
    out = F.gqa_tree_paged(*args, tree_mask=mask.cuda(), **more).cpu()
    v = values(vc, vs)
    for s, (L, n) in enumerate(zip(lens, news)):  # (the bound counts the largest value of what is seen)
        v[b.indices[b.kv_ptr[s] + (L - n) // page], (L - n) % page] = 0
    _check(b, q, values(kc, ks), v, out, mask, 16)
    mask[2, 0] = True
    other = F.gqa_tree_paged(*args, tree_mask=mask.cuda(), **more).cpu()
    rest = torch.arange(b.rows) != 2
    assert torch.equal(other[rest], out[rest]) and not torch.equal(other[2], out[2])


@DTS
@WIDTHS
def test_large_scales_with_small_weights(news, hq, d, dt):
    """A token of scale 2^40 whose score leaves it 2^-40 of the others' weight counts beside them."""
    gen = torch.Generator().manual_seed(23)
    hkv, page, lens = 2, 16, [330, 700]
    b = Batch(lens, news, page, seed=5)
    q = (torch.rand((b.rows, hq, d), generator=gen) * 0.1 + 0.95).to(dt)
    kc, vc, ks, vs = random_cache(b.pool, page, hkv, d, gen, 118, 121)
    place = 3 * page + 5
    for s in range(2):
        at = int(b.indices[b.kv_ptr[s] + 3]), 5
        kc[at] = torch.tensor(-28 / d ** 0.5 * 128).to(E4M3)  # the score: -28
        vc[at] = (vc[at].float() / 8).to(E4M3)
        ks.view(torch.uint8)[at], vs.view(torch.uint8)[at] = 120, 167
    k, v, scale = values(kc, ks), values(vc, vs), power(vs)
    out = F.gqa_tree_paged(q.cuda(), kc.cuda(), vc.cuda(), *b.args(), qo_indptr=b.qo(), k_scale=ks.cuda(), v_scale=vs.cuda()).cpu().double()
    G, half, row, moved = hq // hkv, torch.finfo(dt).eps / 2, 0, 0
    for s, (L, n) in enumerate(zip(lens, news)):
        ids = torch.from_numpy(b.indices[b.kv_ptr[s]:b.kv_ptr[s + 1]]).long()
        for i in range(n):
            at = torch.arange(L - n + i + 1)
            others = at != place
            for h in range(hkv):
                qs, kk, vv, ss = q[row, h * G:(h + 1) * G].double(), *(x[ids[at // page], at % page, h] for x in (k, v, scale))
                p = torch.softmax(qs @ kk.t() / d ** 0.5, -1)
                ref, pv = p @ vv, p @ vv.abs()
                a = (qs.abs() @ kk.abs().t()).max().item() / d ** 0.5
                # a weight's and the result's half step, scores of d fp32 products with an exponent of up to 40 among them;
                # f16 weights times scales, the largest at least 2^7, below the normal range: 2^-25 of a code each
                tol = (half + 2 * 2.0 ** -17 * a + 2 * 0.7 * (d / 8) * 2.0 ** -24 * 40 + 2.0 ** -20) * pv + half * ref.abs() + 2.0 ** -25
                tol = tol + len(at) * 2.0 ** -32 * 448 * (p * ss).amax(-1, keepdim=True)
                assert ((out[row, h * G:(h + 1) * G] - ref).abs() <= tol).all(), (row, h)
                moved += int(((p[:, others] @ vv[others] - ref).abs() > 8 * tol).sum())
            row += 1
    assert moved > 100


@DTS
@WIDTHS
@pytest.mark.parametrize("low,high", [(118, 142), (137, 142), (60, 121)])
def test_scales_of_keys(low, high, news, hq, d, dt):
    """Keys beyond what 16 bits of q's type hold, alone and among ordinary ones, and far below."""
    print("case", low, high, news, hq, d, dt, flush=True)
    gen = torch.Generator().manual_seed(24)
    hkv, page, lens = 2, 16, [330, 700]
    b = Batch(lens, news, page, seed=5)
    big = high > 127
    q = (torch.randn((b.rows, hq, d), generator=gen) * (2.0 ** -12 if big else 1)).to(dt)
    kc, vc, _, vs = random_cache(b.pool, page, hkv, d, gen, 118, 122)
    if big:
        kc = (kc.float() / 16).to(E4M3)
    ks = torch.randint(low, high, (b.pool, page, hkv), generator=gen, dtype=torch.uint8).view(E8M0)
    k, v = values(kc, ks), values(vc, vs)
    assert not big or k.abs().max() > 2 * 65504
    out = F.gqa_tree_paged(q.cuda(), kc.cuda(), vc.cuda(), *b.args(), qo_indptr=b.qo(), k_scale=ks.cuda(), v_scale=vs.cuda()).cpu()
    _check(b, q, k, v, out, None, 9)


def test_largest_keys_of_f16():
    """f16's largest keys, appended: their codes stand for 65536, which f16 itself does not hold."""
    gen = torch.Generator().manual_seed(25)
    dt, hq, hkv, d, page, L = torch.float16, 4, 1, 64, 16, 90
    b = Batch([L], [L], page)
    k = torch.where(torch.rand((L, hkv, d), generator=gen) < 0.5, -65504.0, 65504.0).to(dt)
    v = torch.randn((L, hkv, d), generator=gen).to(dt)
    q = (torch.randn((L, hq, d), generator=gen) * 2.0 ** -14).to(dt)
    kc, vc = (torch.zeros((b.pool, page, hkv, d), dtype=torch.uint8, device="cuda").view(E4M3) for _ in range(2))
    ks, vs = (torch.zeros((b.pool, page, hkv), dtype=torch.uint8, device="cuda").view(E8M0) for _ in range(2))
    F.append_kv_paged_fp8(k.cuda(), v.cuda(), kc, vc, ks, vs, *b.args(), qo_indptr=b.qo())
    stored = values(kc.cpu(), ks.cpu())
    assert stored.abs().max() == 65536
    out = F.gqa_tree_paged(q.cuda(), kc, vc, *b.args(), qo_indptr=b.qo(), k_scale=ks, v_scale=vs).cpu()
    _check(b, q, stored, values(vc.cpu(), vs.cpu()), out, None, 9)


def test_reading_beyond_f16():
    """What f16 does not hold reads as infinity of its sign, what rounds to its largest number as that."""
    b = Batch([16], [16], 16)
    codes = torch.linspace(-448, 448, 64).to(E4M3).expand(b.pool, 16, 1, 64).contiguous()
    scales = (torch.arange(16, dtype=torch.uint8) + 130).view(1, 16, 1).expand(b.pool, 16, 1).contiguous().view(E8M0)
    ref = values(codes, scales)[0].half()
    assert ref.isinf().any() and ref.isfinite().any()
    for x in F.read_kv_paged_fp8(codes.cuda(), codes.cuda(), scales.cuda(), scales.cuda(), *b.args(), b.qo(), 16, dtype=torch.float16):
        assert torch.equal(x.cpu(), ref)

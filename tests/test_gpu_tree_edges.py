"""Attention of new rows where it can go wrong beyond the ordinary cases: every width of a tile and
every way the work is cut, scales of V far apart, more new rows than tokens, repeated calls, calls on
two streams, caches of more than 2^32 elements; append with table positions in 16 bits."""
import math

import pytest
import torch

import yirage_amd.fused as F
from tests.paged_plain import Batch, attend, attend_tolerance, tables
from tests.test_gpu_fp8_cache import _check_head
from tests.tree_plain import E4M3, E8M0, power, random_cache, trees, values, visible

pytestmark = pytest.mark.gpu

DTS = pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])


@pytest.fixture(autouse=True)
def give_back():
    yield
    torch.cuda.empty_cache()


def _check(b, q, k, v, out, mask=None, emax=0, least=0.0):
    """out against 64 bits; k, v [pool, page, hkv, d] in 64 bits.  emax: the largest |exponent| of a scale.

    V's scale is added to a score, as e / (log2(e) / sqrt(d)), before its d products are: at most d / 8 roundings of
    sums of that size, half a step of fp32 each, a weight's relative error by ln 2 of that, in the numerator and
    in the sum of the weights.  least: added, for results below 16 bits' normal numbers."""
    (rows, hq, d), hkv, row = q.shape, k.shape[2], 0
    G, dt = hq // hkv, q.dtype
    more = 2 * math.log(2) * (d / 8) * 2.0 ** -24 * emax
    for s, (L, n) in enumerate(zip(b.lens, b.news)):
        ids = torch.from_numpy(b.indices[b.kv_ptr[s]:b.kv_ptr[s + 1]]).long()
        for i in range(n):
            at = torch.tensor(visible(L, n, i, None if mask is None else mask[row]), dtype=torch.long)
            kk, vv = k[ids[at // b.page], at % b.page], v[ids[at // b.page], at % b.page]
            for h in range(hkv):
                qs = q[row, h * G:(h + 1) * G]
                ref, pv, a = attend(qs, kk[:, h], vv[:, h])
                tol = attend_tolerance(ref, pv, a, len(at), vv[:, h].abs().max().item() if len(at) else 0.0, dt) + least
                # (keys below f16's smallest normal number are half its step off)
                small = 2 * 2.0 ** -25 * qs.double().abs().sum(-1).max().item() if emax and dt is torch.float16 else 0.0
                got = out[row, h * G:(h + 1) * G].double()
                assert ((got - ref).abs() <= tol + (more + small) * pv).all(), (row, h, (got - ref).abs().max().item(), len(at))
            row += 1


CASES = [
    # lens, new rows, query heads, kv heads, d, page, max_kv_len, tree
    ([300, 90], [8, 8], 8, 2, 64, 16, None, True),            # 32 columns
    ([90, 700], [8, 8], 8, 2, 128, 64, 700, False),
    ([300, 1400], [16, 16], 4, 1, 128, 32, None, True),       # 64 columns, tiles over several parts
    ([1500, 20], [15, 1], 16, 2, 64, 16, 1500, False),        # a sequence of one row: waves without columns
    ([2000, 3], [120, 2], 8, 2, 128, 64, 2000, True),         # 128 columns
    ([9000, 40], [1, 1], 8, 4, 128, 64, 513, False),          # 4 heads a workgroup, split
    ([9000, 8000], [3, 1], 12, 6, 64, 64, 513, True),         # 2 heads a workgroup
    ([17 + i % 50 for i in range(300)], [1] * 300, 8, 8, 64, 16, 1, False),  # a tile a workgroup of 4 heads
    ([20 + i % 40 for i in range(300)], [i % 4 for i in range(300)], 6, 2, 64, 16, 1, True),
    ([65 + i % 9 for i in range(130)], [33 + i % 5 for i in range(130)], 1, 1, 64, 32, None, True),  # more than 64 sequences, 64 columns
    ([5, 40, 3], [9, 4, 3], 8, 2, 64, 16, None, False),       # more new rows than tokens: the first see nothing
    ([5, 2, 70], [9, 20, 40], 4, 2, 128, 16, None, True),
    ([100001], [2], 8, 1, 64, 128, 100001, False),
]


@DTS
@pytest.mark.parametrize("q8", [False, True], ids=["16", "e4m3"])
@pytest.mark.parametrize("lens,news,hq,hkv,d,page,most,tree", CASES)
def test_rows(lens, news, hq, hkv, d, page, most, tree, q8, dt):
    print("case", len(lens), max(lens), sum(news), hq, hkv, d, page, most, tree, q8, dt, flush=True)
    gen = torch.Generator().manual_seed(d + page)
    b = Batch(lens, news, page, seed=3)
    q = torch.randn((b.rows, hq, d), generator=gen).to(dt)
    if q8:
        kc, vc, ks, vs = random_cache(b.pool, page, hkv, d, gen, 118, 122)
        scales, k, v = dict(k_scale=ks.cuda(), v_scale=vs.cuda()), values(kc, ks), values(vc, vs)
    else:
        kc, vc = (torch.randn((b.pool, page, hkv, d), generator=gen).to(dt) for _ in range(2))
        scales, k, v = {}, kc.double(), vc.double()
    mask = trees(news, seed=4)[2] if tree else None
    args = (q.cuda(), kc.cuda(), vc.cuda(), *b.args())
    more = dict(tree_mask=None if mask is None else mask.cuda(), qo_indptr=b.qo(), max_kv_len=most, **scales)
    out = F.gqa_tree_paged(*args, **more)
    for _ in range(2):
        assert torch.equal(F.gqa_tree_paged(*args, **more), out)  # sums in a fixed order
    _check(b, q, k, v, out.cpu(), mask, 9 if q8 else 0)


WIDTHS = pytest.mark.parametrize("news,hq,d", [([1, 1], 8, 128), ([7, 1], 8, 64), ([14, 3], 8, 128), ([40, 70], 8, 64)],
                                 ids=["16", "32", "64", "128"])


@DTS
@WIDTHS
@pytest.mark.parametrize("kind", ["apart", "zeros", "tiny", "huge"])
def test_scales_of_v(kind, news, hq, d, dt):
    """Scales of V over the range: up to 2^90 and more apart in a row's tokens, heads of zeros (scale
    2^-126) among others and in whole blocks, all of them near either end."""
    if kind == "huge" and dt is torch.float16:
        lo, hi = 127, 134       # (what 16 bits hold)
    else:
        lo, hi = {"apart": (30, 134 if dt is torch.float16 else 180), "zeros": (118, 122), "tiny": (0, 12), "huge": (245, 248)}[kind]
    print("case", kind, news, hq, d, dt, flush=True)
    gen = torch.Generator().manual_seed(11)
    hkv, page, lens = 2, 16, [330, 700]
    b = Batch(lens, news, page, seed=5)
    q = torch.randn((b.rows, hq, d), generator=gen).to(dt)
    kc, vc, ks, _ = random_cache(b.pool, page, hkv, d, gen, 118, 122)
    if kind == "huge":
        vc = (vc.float() / 64).to(E4M3)
    vs = torch.randint(lo, hi, (b.pool, page, hkv), generator=gen, dtype=torch.uint8)
    if kind == "zeros":
        gone = torch.rand((b.pool, page, hkv), generator=gen) < 0.4
        for s in range(2):  # whole blocks at the front
            gone[torch.from_numpy(b.indices[b.kv_ptr[s]:b.kv_ptr[s] + 9]).long()] = True
        vs[gone] = 1
        vc = torch.where(gone[..., None], 0, vc.float()).to(E4M3)
    vs = vs.view(E8M0)
    k, v = values(kc, ks), values(vc, vs)
    out = F.gqa_tree_paged(q.cuda(), kc.cuda(), vc.cuda(), *b.args(), qo_indptr=b.qo(), k_scale=ks.cuda(), v_scale=vs.cuda()).cpu()
    if kind != "tiny":
        assert out.isfinite().all() and (out != 0).any()
        _check(b, q, k, v, out, None, 127)
    elif dt is torch.float16:
        assert (out == 0).all()
    else:  # in units of 2^-120, where the tolerance's own constants mean something; bf16's steps below 2^-126 are 2^-133
        _check(b, q, k, v * 2.0 ** 120, (out.double() * 2.0 ** 120), None, 127, least=2.0 ** -13)


@DTS
@WIDTHS
def test_large_scores_over_8_bits(news, hq, d, dt):
    """Scores beyond 2^20, where V's exponents are lost beside them: the largest of each row takes the weight,
    and its value comes back exactly."""
    gen = torch.Generator().manual_seed(12)
    hkv, page, lens = 2, 16, [330, 700]
    b = Batch(lens, news, page, seed=5)
    q = (torch.randn((b.rows, hq, d), generator=gen) * 2.0 ** 8).to(dt)
    kc, vc, ks, vs = random_cache(b.pool, page, hkv, d, gen, 118, 122)
    top = 134 if dt is torch.float16 else 160  # (keys that f16 holds)
    ks = torch.randint(top - 4, top, ks.shape, generator=gen, dtype=torch.uint8).view(E8M0)
    k, v = values(kc, ks), values(vc, vs)
    out = F.gqa_tree_paged(q.cuda(), kc.cuda(), vc.cuda(), *b.args(), qo_indptr=b.qo(), k_scale=ks.cuda(), v_scale=vs.cuda()).cpu()
    assert out.isfinite().all()
    checked, row, G = 0, 0, hq // hkv
    for s, (L, n) in enumerate(zip(b.lens, b.news)):
        ids = torch.from_numpy(b.indices[b.kv_ptr[s]:b.kv_ptr[s + 1]]).long()
        for i in range(n):
            at = torch.arange(L - n + i + 1)
            for h in range(hkv):
                kk, vv = k[ids[at // page], at % page, h], v[ids[at // page], at % page, h]
                qs = q[row, h * G:(h + 1) * G].double()
                score = qs @ kk.t()
                best = score.topk(2, -1).values
                # sums of d terms in fp32 are at most 2^-17 of their magnitudes off; V's exponents are below 128
                sure = best[:, 0] - best[:, 1] > (2.0 ** -16 * (qs.abs() @ kk.abs().t()).amax(-1) + 128 + 40) * math.sqrt(d)
                for g in sure.nonzero()[:, 0].tolist():
                    checked += 1
                    assert torch.equal(out[row, h * G + g], vv[score[g].argmax()].to(dt))
            row += 1
    assert checked > 3 * b.rows


def test_two_streams_at_once():
    """Calls on two streams have workspaces of their own."""
    gen, dt = torch.Generator().manual_seed(6), torch.bfloat16
    sets = []
    for lens in ([6000, 300], [3000, 2500]):
        b = Batch(lens, [20, 4], 64, seed=6)
        q = torch.randn((b.rows, 16, 128), generator=gen).to(dt).cuda()
        kc, vc, ks, vs = (t.cuda() for t in random_cache(b.pool, 64, 4, 128, gen))
        sets.append(((q, kc, vc, *b.args()), dict(qo_indptr=b.qo(), k_scale=ks, v_scale=vs), torch.cuda.Stream()))
    want = [F.gqa_tree_paged(*args, **more) for args, more, _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (args, more, stream) in enumerate(sets):
            with torch.cuda.stream(stream):
                got[i].append(F.gqa_tree_paged(*args, **more))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(x, w) for x in g)


@DTS
@pytest.mark.parametrize("L,n,norm,d,page", [(1, 1, False, 64, 16), (40, 1, True, 128, 16), (70, 33, True, 64, 16), (300, 200, False, 128, 64)])
def test_append_16_bit_at_positions(L, n, norm, d, page, dt):
    """Positions are the tables' rows: the same as without them on tables whose rows lie at the rows' places."""
    print("case", L, n, norm, d, page, dt, flush=True)
    gen = torch.Generator().manual_seed(7)
    hq, hkv, most = 10, 2, 64
    b = Batch([L], [n], page, seed=7)
    q, k, v = (torch.randn((n, h, d), generator=gen).to(dt).cuda() for h in (hq, hkv, hkv))
    cos, sin = (t.to(dt if norm else torch.float32).cuda() for t in tables(most, d))
    pos = torch.randint(0, most, (n,), generator=gen, dtype=torch.int32).cuda()
    qn, kn = ((1 + 0.2 * torch.randn(d, generator=gen)).to(dt).cuda() if norm else None for _ in range(2))
    cos2, sin2 = (torch.zeros((L, d), dtype=t.dtype, device="cuda") for t in (cos, sin))
    cos2[L - n:], sin2[L - n:] = cos[pos.long()], sin[pos.long()]
    start = [torch.randn((b.pool, page, hkv, d), generator=gen).to(dt).cuda() for _ in range(2)]
    bounds = torch.randn((b.pool, hkv, 2, d), generator=gen).to(dt).cuda()
    state = [[t.clone() for t in (*start, bounds)] for _ in range(3)]
    run = lambda s, c, sn, p: F.append_kv_paged(k, v, s[0], s[1], *b.args(), q=q, cos=c, sin=sn, q_norm=qn, k_norm=kn, qo_indptr=b.qo(),
                                                page_bounds=s[2], positions=p)
    assert torch.equal(run(state[0], cos, sin, pos), run(state[1], cos2, sin2, None))
    for x, y in zip(*state[:2]):
        assert torch.equal(x, y)
    # positions outside the tables: NaN, and the token is not written
    lost = torch.rand(n, generator=gen) < 0.5
    lost[0] = True
    pos[lost.cuda()] = torch.tensor([-1, most, 2 ** 31 - 1], dtype=torch.int32)[torch.arange(int(lost.sum())) % 3].cuda()
    out = run(state[2], cos, sin, pos)
    assert out[lost.cuda()].isnan().all() and out[~lost.cuda()].isfinite().all()
    for new, old, done in zip(state[2][:2], start, state[0][:2]):
        for i in range(n):
            at = (int(b.indices[(L - n + i) // page]), (L - n + i) % page)
            assert torch.equal(new[at], (old if lost[i] else done)[at])


@pytest.mark.parametrize("q8", [False, True], ids=["16", "e4m3"])
@pytest.mark.parametrize("news", [[1, 1], [5, 3], [30, 20]])
def test_caches_beyond_32_bits(news, q8):
    """Caches of more than 2^32 elements, the pages in use at both ends and in between."""
    print("case", news, q8, flush=True)
    dt, hkv, hq, d, page, pool = torch.bfloat16, 8, 16, 128, 1, (1 << 22) + 64
    gen = torch.Generator().manual_seed(8)
    b = Batch([60, 50], news, page, seed=2)
    ids = torch.cat([torch.arange(7), (1 << 21) - 20 + torch.arange(40), pool - 63 + torch.arange(63)])
    b.pool, b.indices = pool, ids[torch.randperm(110, generator=gen)].to(torch.int32).numpy()
    at = torch.from_numpy(b.indices).long().cuda()
    if q8:
        kc, vc = (torch.empty((pool, page, hkv, d), dtype=torch.uint8, device="cuda").view(E4M3) for _ in range(2))
        ks, vs = (torch.empty((pool, page, hkv), dtype=torch.uint8, device="cuda").view(E8M0) for _ in range(2))
        raw = [t.view(torch.uint8) for t in (kc, vc, ks, vs)]
        for t, x in zip(raw, random_cache(110, page, hkv, d, gen)):
            t[at] = x.view(torch.uint8).cuda()
        scales = dict(k_scale=ks, v_scale=vs)
    else:
        kc, vc = (torch.empty((pool, page, hkv, d), dtype=dt, device="cuda") for _ in range(2))
        raw, scales = [kc, vc], {}
        for t in raw:
            t[at] = torch.randn((110, page, hkv, d), generator=gen).to(dt).cuda()
    assert kc.numel() > 1 << 32
    q = torch.randn((b.rows, hq, d), generator=gen).to(dt)
    k, v = (torch.randn((b.rows, hkv, d), generator=gen).to(dt) for _ in range(2))
    cos, sin = torch.ones((4, d), device="cuda"), torch.zeros((4, d), device="cuda")
    pos = torch.zeros(b.rows, dtype=torch.int32, device="cuda")
    if q8:
        F.append_kv_paged_fp8(k.cuda(), v.cuda(), kc, vc, ks, vs, *b.args(), qo_indptr=b.qo())
    else:
        F.append_kv_paged(k.cuda(), v.cuda(), kc, vc, *b.args(), qo_indptr=b.qo(), cos=cos, sin=sin, positions=pos)
    # the pages in use, as a small cache of their own
    small = [t[at].cpu() for t in raw]
    if q8:
        codes, sc = [t.view(E4M3) for t in small[:2]], [t.view(E8M0) for t in small[2:]]
        kv = [values(c, s) for c, s in zip(codes, sc)]
    else:
        kv = [t.double() for t in small]
    for s, (L, n) in enumerate(zip(b.lens, b.news)):
        for i in range(n):
            t, x = int(b.qo_ptr[s]) + i, int(b.kv_ptr[s]) + L - n + i
            for h in range(hkv):
                if q8:
                    for j, src in enumerate((k, v)):
                        _check_head(codes[j][x, 0, h], power(sc[j][x, 0, h]), src[t, h].double(), torch.zeros(d))
                else:
                    assert torch.equal(small[0][x, 0, h], k[t, h]) and torch.equal(small[1][x, 0, h], v[t, h])
    out = F.gqa_tree_paged(q.cuda(), kc, vc, *b.args(), qo_indptr=b.qo(), **scales).cpu()
    near = Batch([60, 50], news, page)
    near.indices = torch.arange(110, dtype=torch.int32).numpy()
    _check(near, q, *kv, out, None, 12 if q8 else 0)
    if q8:
        to = torch.tensor([0, 60, 110], dtype=torch.int32, device="cuda")
        for got, want in zip(F.read_kv_paged_fp8(kc, vc, ks, vs, *b.args(), to, 110), kv):
            assert torch.equal(got.cpu(), want[:, 0].to(dt))
    path = torch.tensor([[0, 2, 4], [1, 2, -1]], dtype=torch.int32, device="cuda")
    lens = F.keep_kv_paged(kc, vc, *b.args(), path, qo_indptr=b.qo(), **scales).tolist()
    for s, (L, n) in enumerate(zip(b.lens, b.news)):
        kept = [p for p in path[s].tolist() if 0 <= p < n]
        assert lens[s] == L - n + len(kept)
        x = int(b.kv_ptr[s]) + L - n
        for j, p in enumerate(kept):
            for t, was in zip(raw, small):
                assert torch.equal(t[at[x + j]].cpu(), was[x + p])

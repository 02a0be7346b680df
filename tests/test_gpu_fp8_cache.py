"""append_kv_paged_fp8 and read_kv_paged_fp8 against 64 bits: ragged batches, page
sizes, norms, table types, tree positions, extreme magnitudes, missing places."""
import math

import pytest
import torch

import yirage_amd.fused as F
from tests.paged_plain import Batch, norm_rotate, tables
from tests.tree_plain import E4M3, E8M0, power, random_cache, trees, values

pytestmark = pytest.mark.gpu

DTS = pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])


def _bytes(t):
    return t.view(torch.uint8)


def _check_head(codes, scale, ref, mag):
    """One head's codes [d] and scale against its value in 64 bits; mag: what the fp32 sums add up."""
    err = 2.0 ** -19 * mag + 2.0 ** -140  # about 20 fp32 roundings
    top, s = ref.abs().max().item(), scale.item()
    slack = err.max().item()
    assert top <= 448 * s + slack, (top, s)
    assert top + slack > 224 * s or s == 2.0 ** -126, (top, s)
    # half a step of e4m3: 2^-4 of the value, 2^-10 of the scale below 2^-6 of it
    tol = torch.maximum(2.0 ** -4 * ref.abs(), torch.full_like(ref, 2.0 ** -10 * s)) + 2 * err
    assert ((codes.float().double() * s - ref).abs() <= tol).all()


@DTS
@pytest.mark.parametrize("lens,news,hq,hkv,d,page,norm,tree", [
    ([1], [1], 4, 4, 64, 16, False, False), ([64], [1], 32, 8, 128, 64, False, False), ([65], [1], 32, 8, 128, 64, True, False),
    ([5, 70, 16, 33], [1, 1, 1, 1], 10, 2, 128, 16, True, False),
    ([5, 70, 16, 33], [5, 1, 0, 20], 14, 2, 64, 16, False, True),
    ([200, 131], [37, 131], 8, 1, 128, 48, True, True),
    ([3, 9], [3, 2], 16, 16, 64, 1, False, False),
    ([40 + i for i in range(70)], [1 + i % 3 for i in range(70)], 5, 1, 128, 32, False, True),
    ([50], [7], 24, 3, 64, 16, True, False),          # rows of q, k and v share a pass
])
def test_append(lens, news, hq, hkv, d, page, norm, tree, dt):
    print("case", len(lens), max(lens), sum(news), hq, hkv, d, page, norm, tree, dt, flush=True)
    gen = torch.Generator().manual_seed(hq + page)
    b = Batch(lens, news, page, seed=page)
    qkv = torch.randn((b.rows, hq + 2 * hkv, d), generator=gen)
    qkv = (qkv * 2.0 ** torch.randint(-6, 7, (b.rows, hq + 2 * hkv, 1), generator=gen)).to(dt)
    q, k, v = qkv.split([hq, hkv, hkv], 1)
    cos, sin = (t.to(dt if norm else torch.float32) for t in tables(max(lens), d))
    qn, kn = ((1 + 0.2 * torch.randn(d, generator=gen)).to(dt) if norm else None for _ in range(2))
    before = random_cache(b.pool, page, hkv, d, gen)
    pos = torch.tensor([p for _, p, _ in b.each_row()], dtype=torch.int32)
    if tree:
        _, depth, _ = trees(news, seed=1)
        firsts = torch.tensor([L - n for L, n in zip(lens, news) for _ in range(n)])
        pos = (firsts + torch.from_numpy(depth)).int()
    dev = lambda t: None if t is None else t.cuda()
    cache = [t.cuda() for t in before]
    dq, dk, dv = qkv.cuda().split([hq, hkv, hkv], 1)
    got = F.append_kv_paged_fp8(dk, dv, *cache, *b.args(), q=dq, cos=dev(cos), sin=dev(sin), q_norm=dev(qn), k_norm=dev(kn),
                                qo_indptr=b.qo(), positions=pos.cuda() if tree else None).cpu()
    kc, vc, ks, vs = (t.cpu() for t in cache)
    want = [_bytes(t).clone() for t in before]
    for t, p, ids in b.each_row():
        c, s = cos[pos[t].item()], sin[pos[t].item()]
        ref, mag = norm_rotate(q[t], qn, c, s, 1e-6)
        tol = torch.finfo(dt).eps / 2 * ref.abs() * (1 + 2.0 ** -8) + 2.0 ** -19 * mag + 2.0 ** -25
        assert ((got[t].double() - ref).abs() <= tol).all(), ("q", t)
        at = (ids[p // page], p % page)
        ref, mag = norm_rotate(k[t], kn, c, s, 1e-6)
        for h in range(hkv):
            _check_head(kc[at][h], power(ks[at][h]), ref[h], mag[h])
            _check_head(vc[at][h], power(vs[at][h]), v[t, h].double(), torch.zeros(d))
        for w, t2 in zip(want, (kc, vc, ks, vs)):
            w[at] = _bytes(t2)[at]
    for w, t2 in zip(want, (kc, vc, ks, vs)):
        assert torch.equal(w, _bytes(t2))  # no other slot changed


@DTS
def test_codes_of_every_magnitude(dt):
    """Without norm and rotation a code is x / scale rounded to nearest even, whatever the magnitude:
    powers of two around the border of a scale, zeros, the type's smallest and largest numbers."""
    gen = torch.Generator().manual_seed(3)
    fi = torch.finfo(dt)
    tops = [0.0, fi.tiny, fi.max, 448.0, 449.0, 450.0, 447.0, 224.0, 225.0, 1.75, 1.76, 1.0, fi.tiny * 1.75, fi.smallest_normal / 4]
    x = torch.rand((len(tops), 1, 128), generator=gen) * 2 - 1
    x[0] = 0
    x = torch.stack([(r * t).to(dt) for r, t in zip(x, tops)])
    for r, t in zip(x, tops):
        r[0, 17] = torch.tensor(t).to(dt)
    b = Batch([len(tops)], [len(tops)], 16)
    cache = [t.cuda() for t in random_cache(b.pool, 16, 1, 128, gen)]
    assert F.append_kv_paged_fp8(x.cuda(), -x.cuda(), *cache, *b.args(), qo_indptr=b.qo()) is None
    pg = b.indices[0]
    for c, s, sign in ((cache[0], cache[2], 1), (cache[1], cache[3], -1)):
        c, s = c.cpu()[pg, :len(tops), 0], s.cpu()[pg, :len(tops), 0]
        for i in range(len(tops)):
            y = sign * x[i, 0].double()
            top = y.abs().max().item()
            e = max(math.ceil(math.log2(top / 448)), -126) if top else -126
            assert _bytes(s)[i] == e + 127, (tops[i], e)
            # (below 2^-126 / 2^-9 nothing is left; the quotient is exact in fp32)
            assert torch.equal(c[i].float(), (y / 2.0 ** e).float().to(E4M3).float()), tops[i]


def test_not_finite():
    """A head with a NaN or an infinity reads as NaN, the others as they are; so does its attention."""
    dt, b = torch.bfloat16, Batch([5], [5], 16)
    k = torch.randn((5, 2, 64), generator=torch.Generator().manual_seed(1)).to(dt)
    v = k.clone()
    k[1, 0, 5], k[2, 1, 63], v[3, 0, 0] = math.nan, math.inf, -math.inf
    cache = [t.cuda() for t in random_cache(b.pool, 16, 2, 64, torch.Generator().manual_seed(2))]
    F.append_kv_paged_fp8(k.cuda(), v.cuda(), *cache, *b.args(), qo_indptr=b.qo())
    rk, rv = F.read_kv_paged_fp8(*cache, *b.args(), b.qo(), 5)
    for x, r in ((k, rk.cpu()), (v, rv.cpu())):
        lost = ~x.isfinite().all(-1)
        assert r[lost].isnan().all() and r[~lost].isfinite().all()


def test_what_has_no_place():
    """Pages outside the cache, a short table, positions behind the tables, padded rows: nothing else is touched."""
    gen = torch.Generator().manual_seed(3)
    dt, d = torch.bfloat16, 64
    b = Batch([40, 40, 40, 25], [10, 10, 10, 10], 16)
    b.rows += 5
    q = torch.randn((b.rows, 2, d), generator=gen).to(dt)
    k, v = (torch.randn((b.rows, 1, d), generator=gen).to(dt) for _ in range(2))
    cos, sin = (t.float() for t in tables(36, d))
    before = random_cache(b.pool, 16, 1, d, gen)
    bad = b.indices.copy()
    bad[b.kv_ptr[0] + 2], bad[b.kv_ptr[1] + 1] = -1, b.pool
    ptr = b.kv_ptr.copy()
    ptr[4] = ptr[3] + 1
    cache = [t.cuda() for t in before]
    out = torch.full((b.rows, 2, d), 3.0, dtype=dt, device="cuda")
    table = (torch.from_numpy(ptr).cuda(), torch.from_numpy(bad).cuda(), b.args()[2])
    F.append_kv_paged_fp8(k.cuda(), v.cuda(), *cache, *table, q=q.cuda(), cos=cos.cuda(), sin=sin.cuda(),
                          qo_indptr=torch.from_numpy(b.qo_ptr).cuda(), out=out)
    after, want, has = [t.cpu() for t in cache], [_bytes(t).clone() for t in before], {}
    for s, (L, n) in enumerate(zip(b.lens, b.news)):
        for p in range(L):
            e = ptr[s] + p // 16
            has[s, p] = e < ptr[s + 1] and 0 <= bad[e] < b.pool
            if p < L - n:
                continue
            t = int(b.qo_ptr[s]) + p - (L - n)
            if p >= 36:
                assert torch.isnan(out[t].float()).all()
            else:
                assert out[t].isfinite().all()
                if has[s, p]:
                    for w, x in zip(want, after):
                        w[bad[e], p % 16] = _bytes(x)[bad[e], p % 16]
    for w, x in zip(want, after):
        assert torch.equal(w, _bytes(x))
    assert (out[40:] == 3).all()
    # read back: what has no place is 0, rows behind the last sequence stay
    ptr_out = torch.tensor([0, 45, 85, 125, 150], dtype=torch.int32, device="cuda")  # 45 rows for 40 tokens
    res = [torch.full((155, 1, d), 7.0, dtype=dt, device="cuda") for _ in range(2)]
    F.read_kv_paged_fp8(*cache, *table, ptr_out, 155, out=res)
    for r, c, s in zip(res, after[:2], after[2:]):
        r, val = r.cpu(), values(c, s)
        for sq, (o, L) in enumerate(zip([0, 45, 85, 125], [45, 40, 40, 25])):
            for p in range(L):
                ref = val[bad[ptr[sq] + p // 16], p % 16].to(dt) if has.get((sq, p)) else torch.zeros(1, d, dtype=dt)
                assert torch.equal(r[o + p], ref), (sq, p)
        assert (r[150:] == 7).all()


@DTS
@pytest.mark.parametrize("lens,hkv,d,page", [([1], 1, 64, 16), ([500], 8, 128, 64), ([0, 3, 77, 16], 2, 64, 16), ([130, 5], 5, 128, 48),
                                             ([9] * 100, 1, 128, 1), ([1000, 333], 16, 64, 128), ([2000], 3, 64, 32)])
def test_read(lens, hkv, d, page, dt):
    print("case", len(lens), max(lens), hkv, d, page, dt, flush=True)
    gen = torch.Generator().manual_seed(d)
    b = Batch(lens, lens, page, seed=1)
    kc, vc, ks, vs = random_cache(b.pool, page, hkv, d, gen, low=96, high=134)  # into f16's subnormal numbers, not beyond its largest
    got = F.read_kv_paged_fp8(kc.cuda(), vc.cuda(), ks.cuda(), vs.cuda(), *b.args(), torch.from_numpy(b.qo_ptr).cuda(), b.rows, dtype=dt)
    for g, c, s in zip(got, (kc, vc), (ks, vs)):
        val = values(c, s).float()  # (exact)
        ref = torch.cat([val[torch.from_numpy(ids).long()].flatten(0, 1)[:L] for L, ids in
                         zip(lens, (b.indices[a:z] for a, z in zip(b.kv_ptr, b.kv_ptr[1:])))])
        assert torch.equal(g.cpu(), ref.to(dt))


def test_scale_bytes():
    """Every scale byte, in bf16: 0 stands for 2^-127, 255 for NaN."""
    b = Batch([256], [256], 256)
    codes = torch.full((b.pool, 256, 1, 64), 1.5).to(E4M3)
    scales = torch.arange(256, dtype=torch.uint8).view(1, 256, 1).expand(b.pool, 256, 1).contiguous().view(E8M0)
    k, v = F.read_kv_paged_fp8(codes.cuda(), codes.cuda(), scales.cuda(), scales.cuda(), *b.args(), b.qo(), 256)
    ref = (1.5 * power(scales[0, :, 0]))
    for x in (k.cpu(), v.cpu()):
        assert x[255].isnan().all() and torch.equal(x[1:255, 0, 0].double(), ref[1:255])
        assert (x[0].double() - ref[0]).abs().max() <= 2.0 ** -127  # (below bf16's normal numbers)

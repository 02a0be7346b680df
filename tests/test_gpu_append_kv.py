"""append_kv_paged against 64 bits: ragged batches, page sizes, partial first and
last pages, norms, table types, sliced projections, missing pages and positions."""
import pytest
import torch

import yirage_amd.fused as F
from tests.paged_plain import Batch, norm_rotate, tables

pytestmark = pytest.mark.gpu

DTS = pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])


def _caches(b, hkv, d, dt, gen):
    k = torch.randn((b.pool, b.page, hkv, d), generator=gen).to(dt)
    v = torch.randn((b.pool, b.page, hkv, d), generator=gen).to(dt)
    bounds = torch.full((b.pool, hkv, 2, d), 7.0).to(dt)
    # pages that hold tokens already have their bounds
    for L, n, p0 in zip(b.lens, b.news, b.kv_ptr):
        old = L - n
        for u in range(-(-old // b.page)):
            seen = k[b.indices[p0 + u], : min(b.page, old - u * b.page)]
            bounds[b.indices[p0 + u], :, 0], bounds[b.indices[p0 + u], :, 1] = seen.amin(0), seen.amax(0)
    return k, v, bounds


def _half_step(ref, mag, dt):
    # one rounding to dt; in fp32 about 20 roundings of the norm and 3 of the rotation (below 2^-19 of what it adds)
    return torch.finfo(dt).eps / 2 * ref.abs() * (1 + 2.0 ** -8) + 2.0 ** -19 * mag + 2.0 ** -25


def _check(b, hq, hkv, d, dt, q, k, v, got_q, before, after, cos, sin, qn, kn, eps=1e-6):
    kc, vc, bd = (t.clone() for t in before)
    got_k, got_v, got_b = after
    for t, p, ids in b.each_row():
        c, s = (None, None) if cos is None else (cos[p], sin[p])
        ref, mag = norm_rotate(q[t], qn, c, s, eps)
        assert ((got_q[t].double() - ref).abs() <= _half_step(ref, mag, dt)).all(), ("q", t)
        at = (ids[p // b.page], p % b.page)
        ref, mag = norm_rotate(k[t], kn, c, s, eps)
        assert ((got_k[at].double() - ref).abs() <= _half_step(ref, mag, dt)).all(), ("k", t)
        kc[at] = got_k[at]
        vc[at] = v[t]
    assert torch.equal(got_k, kc)  # no other slot changed
    assert torch.equal(got_v, vc)
    for L, n, p0 in zip(b.lens, b.news, b.kv_ptr):
        for u in range(max(L - n, 0) // b.page if n else 0, -(-L // b.page) if n else 0):
            seen = kc[b.indices[p0 + u], : min(b.page, L - u * b.page)]
            bd[b.indices[p0 + u], :, 0], bd[b.indices[p0 + u], :, 1] = seen.amin(0), seen.amax(0)
    assert torch.equal(got_b, bd)


@DTS
@pytest.mark.parametrize("lens,news,hq,hkv,d,page,norm", [
    ([1], [1], 4, 4, 64, 16, False), ([64], [1], 32, 8, 128, 64, False), ([65], [1], 32, 8, 128, 64, True),
    ([5, 70, 16, 33], [1, 1, 1, 1], 10, 2, 128, 16, True),
    ([5, 70, 16, 33], [5, 1, 0, 20], 14, 2, 64, 16, False),      # a sequence without new rows
    ([200, 131], [137, 131], 8, 1, 128, 48, True),               # over several pages, odd page size
    ([3, 9], [3, 2], 16, 16, 64, 1, False),                      # one token a page
    ([700] * 3 + [1], [700, 699, 64, 1], 16, 4, 64, 128, True),
    ([40 + i for i in range(70)], [1 + i % 3 for i in range(70)], 5, 1, 128, 32, False),  # many sequences
    ([17] * 300, [1] * 300, 2, 2, 64, 16, False),
])
def test_rows(lens, news, hq, hkv, d, page, norm, dt):
    print("case", len(lens), max(lens), sum(news), hq, hkv, d, page, norm, dt, flush=True)
    gen = torch.Generator().manual_seed(hq + page)
    b = Batch(lens, news, page, seed=page)
    qkv = torch.randn((b.rows, hq + 2 * hkv, d), generator=gen).to(dt)
    q, k, v = qkv.split([hq, hkv, hkv], 1)
    cos, sin = (t.to(dt if norm else torch.float32) for t in tables(max(lens), d))
    qn, kn = ((1 + 0.2 * torch.randn(d, generator=gen)).to(dt) if norm else None for _ in range(2))
    before = _caches(b, hkv, d, dt, gen)
    dev = lambda t: None if t is None else t.cuda()
    kc, vc, bd = (t.cuda() for t in before)
    dq, dk, dv = qkv.cuda().split([hq, hkv, hkv], 1)  # slices, as they come
    for _ in range(2):  # again with the same tokens: nothing changes
        got = F.append_kv_paged(dk, dv, kc, vc, *b.args(), q=dq, cos=dev(cos), sin=dev(sin), q_norm=dev(qn),
                                k_norm=dev(kn), qo_indptr=b.qo(), page_bounds=bd)
        _check(b, hq, hkv, d, dt, q, k, v, got.cpu(), before, (kc.cpu(), vc.cpu(), bd.cpu()), cos, sin, qn, kn)
        before = (kc.cpu(), vc.cpu(), bd.cpu())


@DTS
def test_without_q_tables_and_bounds(dt):
    gen = torch.Generator().manual_seed(1)
    b = Batch([50, 33], [20, 33], 16)
    k, v = (torch.randn((b.rows, 2, 128), generator=gen).to(dt) for _ in range(2))
    before = _caches(b, 2, 128, dt, gen)
    kc, vc = before[0].cuda(), before[1].cuda()
    assert F.append_kv_paged(k.cuda(), v.cuda(), kc, vc, *b.args(), qo_indptr=b.qo()) is None
    kr, vr = before[0].clone(), before[1].clone()
    for t, p, ids in b.each_row():
        kr[ids[p // 16], p % 16], vr[ids[p // 16], p % 16] = k[t], v[t]
    assert torch.equal(kc.cpu(), kr) and torch.equal(vc.cpu(), vr)


@DTS
def test_group_layout_and_in_place(dt):
    """q as [T, Hkv, G, D] inside a projection laid out per kv head (q x G | k | v), and q_out = q."""
    gen = torch.Generator().manual_seed(2)
    G, hkv, d = 4, 2, 128
    b = Batch([30, 7], [9, 7], 16)
    rows = torch.randn((b.rows, hkv, G + 2, d), generator=gen).to(dt)
    cos, sin = (t.float() for t in tables(30, d))
    before = _caches(b, hkv, d, dt, gen)
    kc, vc, bd = (t.cuda() for t in before)
    dr = rows.cuda()
    got = F.append_kv_paged(dr[:, :, G], dr[:, :, G + 1], kc, vc, *b.args(), q=dr[:, :, :G], cos=cos.cuda(),
                            sin=sin.cuda(), qo_indptr=b.qo(), page_bounds=bd)
    q = rows[:, :, :G].reshape(b.rows, hkv * G, d)
    _check(b, hkv * G, hkv, d, dt, q, rows[:, :, G], rows[:, :, G + 1], got.cpu(), before,
           (kc.cpu(), vc.cpu(), bd.cpu()), cos, sin, None, None)
    dq = q.cuda()
    same = F.append_kv_paged(dr[:, :, G], dr[:, :, G + 1], kc, vc, *b.args(), q=dq, cos=cos.cuda(), sin=sin.cuda(),
                             qo_indptr=b.qo(), page_bounds=bd, out=dq)
    assert same is dq and torch.equal(dq, got)


def test_what_has_no_place():
    """Pages outside the cache, a table that is too short, positions behind the tables, rows
    behind the last sequence: not written, and nothing else is touched."""
    gen = torch.Generator().manual_seed(3)
    dt, d = torch.bfloat16, 64
    b = Batch([40, 40, 40, 25], [10, 10, 10, 10], 16)
    b.rows += 5  # padded rows
    q = torch.randn((b.rows, 2, d), generator=gen).to(dt)
    k, v = (torch.randn((b.rows, 1, d), generator=gen).to(dt) for _ in range(2))
    cos, sin = (t.float() for t in tables(36, d))  # positions 36 .. 39 have no angle
    before = _caches(b, 1, d, dt, gen)
    bad = b.indices.copy()
    bad[b.kv_ptr[0] + 2] = -1            # sequence 0: tokens 32 ..
    bad[b.kv_ptr[1] + 1] = b.pool        # sequence 1: tokens 16 .. 31
    ptr = b.kv_ptr.copy()
    ptr[4] = ptr[3] + 1                  # sequence 3 owns 16 tokens' pages and has 25
    kc, vc, bd = (t.cuda() for t in before)
    out = torch.full((b.rows, 2, d), 3.0, dtype=dt, device="cuda")
    qo = torch.from_numpy(b.qo_ptr).cuda()
    F.append_kv_paged(k.cuda(), v.cuda(), kc, vc, torch.from_numpy(ptr).cuda(), torch.from_numpy(bad).cuda(),
                      b.args()[2], q=q.cuda(), cos=cos.cuda(), sin=sin.cuda(), qo_indptr=qo, page_bounds=bd, out=out)
    kr, vr, written = before[0].clone(), before[1].clone(), set()
    got_k = kc.cpu()
    for s, (L, n) in enumerate(zip(b.lens, b.news)):
        for i in range(n):
            p, t = L - n + i, int(b.qo_ptr[s]) + i
            e = ptr[s] + p // 16
            has = e < ptr[s + 1] and 0 <= bad[e] < b.pool and p < 36
            if p >= 36:
                assert torch.isnan(out[t].float()).all()
            else:
                ref, mag = norm_rotate(q[t], None, cos[p], sin[p], 0)
                assert ((out[t].cpu().double() - ref).abs() <= _half_step(ref, mag, dt)).all()
            if has:
                written.add(int(bad[e]))
                kr[bad[e], p % 16] = got_k[bad[e], p % 16]
                vr[bad[e], p % 16] = v[t]
    assert torch.equal(got_k, kr) and torch.equal(vc.cpu(), vr)
    assert (out[40:] == 3).all()
    for pg in set(range(b.pool)) - written:
        assert torch.equal(bd[pg].cpu(), before[2][pg])


@DTS
def test_bounds_of_infinite_and_nan_keys(dt):
    """Bounds leave NaN out and take infinities as they are; without rotation keys pass unchanged."""
    b = Batch([16], [16], 16)
    k = torch.randn((16, 1, 64), generator=torch.Generator().manual_seed(4)).to(dt)
    k[3, 0, :8], k[5, 0, 4:12], k[:, 0, 20] = float("nan"), float("inf"), float("-inf")
    kc, vc = (torch.zeros((b.pool, 16, 1, 64), dtype=dt, device="cuda") for _ in range(2))
    bd = torch.zeros((b.pool, 1, 2, 64), dtype=dt, device="cuda")
    F.append_kv_paged(k.cuda(), k.cuda(), kc, vc, *b.args(), qo_indptr=b.qo(), page_bounds=bd)
    pg = b.indices[0]
    assert torch.equal(kc[pg, :, 0].cpu().view(torch.int16), k[:, 0].view(torch.int16))
    lo = torch.where(k.isnan(), float("inf"), k.float()).amin(0)[0]
    hi = torch.where(k.isnan(), -float("inf"), k.float()).amax(0)[0]
    assert torch.equal(bd[pg, 0, 0].float().cpu(), lo) and torch.equal(bd[pg, 0, 1].float().cpu(), hi)

"""Plain 64-bit forms (on the CPU) of drafting over a paged cache: e4m3 codes with a
power of two per token and head, trees of drafted tokens, their accepted paths."""
import math

import numpy as np
import torch

from tests.paged_plain import attend, attend_tolerance

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def power(scale):
    """e8m0 -> 64 bits (255: NaN)"""
    b = scale.view(torch.uint8).int()
    return torch.where(b == 255, math.nan, torch.ldexp(torch.ones(b.shape, dtype=torch.float64), b - 127))


def values(codes, scale):
    """What codes [..., hkv, d] and scales [..., hkv] stand for, in 64 bits."""
    return codes.float().double() * power(scale)[..., None]


def random_cache(pool, page, hkv, d, gen, low=115, high=122):
    """k, v codes and scales of random exponents"""
    codes = [(torch.randn((pool, page, hkv, d), generator=gen) * 120).clamp(-448, 448).to(E4M3) for _ in range(2)]
    scales = [torch.randint(low, high, (pool, page, hkv), generator=gen, dtype=torch.uint8).view(E8M0) for _ in range(2)]
    return (*codes, *scales)


def trees(news, seed=0, width=5):
    """Parents of each sequence's nodes (-1: a root), each node's depth, and the mask [rows, most]."""
    rng = np.random.default_rng(seed)
    rows, most = int(sum(news)), max(int(max(news)), 1)
    parents, depth, mask, row = [], np.zeros(rows, dtype=np.int64), np.zeros((rows, most), dtype=bool), 0
    for n in news:
        up = [-1 if i == 0 else int(max(i - rng.integers(1, width + 1), 0)) for i in range(n)]
        for i in range(n):
            if i:
                depth[row + i] = depth[row + up[i]] + 1
                mask[row + i] = mask[row + up[i]]
            mask[row + i, i] = True
        parents.append(up)
        row += n
    return parents, depth, torch.from_numpy(mask)


def visible(L, n, i, mask_row=None):
    """Positions that row i of a sequence's n new rows sees (L tokens with the new ones)."""
    first = L - n
    seen = [p for p in range(L) if p < first]
    if mask_row is None:
        return seen + [p for p in range(max(first, 0), min(L, first + i + 1))]
    return seen + [first + j for j in range(min(n, len(mask_row))) if mask_row[j] and first + j >= 0]


def check_attention(b, hq, hkv, q, k, v, out, mask=None, dtype_p=None, skip=()):
    """out [rows, hq, d] of batch b against 64 bits; k, v [pool, page, hkv, d] in 64 bits.  dtype_p: what the
    weights are rounded to.  skip: pages that count as missing."""
    G, dt, row = hq // hkv, q.dtype, 0
    for s, (L, n) in enumerate(zip(b.lens, b.news)):
        ids = b.indices[b.kv_ptr[s]:b.kv_ptr[s + 1]]
        for i in range(n):
            seen = [p for p in visible(L, n, i, None if mask is None else mask[row]) if p // b.page < len(ids)]
            at = [(ids[p // b.page], p % b.page) for p in seen if ids[p // b.page] not in skip]
            pg, sl = torch.tensor([x[0] for x in at], dtype=torch.long), torch.tensor([x[1] for x in at], dtype=torch.long)
            for h in range(hkv):
                qs = q[row, h * G:(h + 1) * G]
                kk, vv = k[pg, sl, h], v[pg, sl, h]
                ref, pv, a = attend(qs, kk, vv)
                tol = attend_tolerance(ref, pv, a, len(at), vv.abs().max().item() if len(at) else 0.0, dt)
                if dtype_p is not None and len(at):
                    # weights in another type, keys below f16's smallest normal number, half its step off
                    tol = tol + (torch.finfo(dtype_p).eps / 2 + 2 * 2.0 ** -25 * qs.double().abs().sum(-1).max().item()) * pv
                got = out[row, h * G:(h + 1) * G].double()
                bad = (got - ref).abs() > tol
                assert not bad.any() and not got.isnan().any(), (row, h, (got - ref).abs().max().item(), len(at))
            row += 1

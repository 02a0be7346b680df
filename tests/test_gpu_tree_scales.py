"""Attention over e4m3 caches whose scales change along a sequence, in every width of a tile, within a
wave, over the waves of a workgroup and over the parts of a split tile."""
import pytest
import torch

import yirage_amd.fused as F
from tests.paged_plain import Batch
from tests.test_gpu_tree_edges import DTS, WIDTHS, _check
from tests.tree_plain import E4M3, E8M0, random_cache, values

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

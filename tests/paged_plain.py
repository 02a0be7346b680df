"""Plain 64-bit forms (on the CPU) of the operators around a paged cache, row by
row from their definitions, and ragged batches to test them on."""
import math

import numpy as np
import torch


class Batch:
    """lens: tokens of each sequence, its new rows included; news: new rows; pages in
    a shuffled table over a pool with a few spare pages."""

    def __init__(self, lens, news, page, seed=0):
        self.lens, self.news, self.page = list(lens), list(news), page
        npg = [-(-n // page) for n in lens]
        self.pool = sum(npg) + 3
        rng = np.random.default_rng(seed)
        self.indices = rng.permutation(self.pool)[: sum(npg)].astype(np.int32)
        self.kv_ptr = np.concatenate([[0], np.cumsum(npg)]).astype(np.int32)
        self.qo_ptr = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        self.rows = int(sum(news))

    def args(self, device="cuda"):
        dev = lambda a: torch.from_numpy(np.asarray(a, dtype=np.int32)).to(device)
        return dev(self.kv_ptr), dev(self.indices), dev(self.lens)

    def qo(self, device="cuda"):
        """None for one row a sequence, as a decode step passes it."""
        if all(n == 1 for n in self.news):
            return None
        return torch.from_numpy(self.qo_ptr).to(device)

    def each_row(self):
        """(row, position, page ids of its sequence)"""
        for b, (L, n) in enumerate(zip(self.lens, self.news)):
            ids = self.indices[self.kv_ptr[b]:self.kv_ptr[b + 1]]
            for i in range(n):
                yield int(self.qo_ptr[b]) + i, L - n + i, ids


def tables(positions, d, theta=10000.0):
    inv = theta ** (-np.arange(0, d, 2) / d)
    ang = np.outer(np.arange(positions), np.concatenate([inv, inv]))
    return torch.from_numpy(np.cos(ang)), torch.from_numpy(np.sin(ang))


def norm_rotate(x, w, cos, sin, eps):
    """x [heads, d] in 64 bits; also the magnitude of what the rotation adds up."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    if cos is None:
        return x, x.abs()
    h = x.shape[-1] // 2
    turned = torch.cat([-x[:, h:], x[:, :h]], -1)
    return x * cos.double() + turned * sin.double(), (x * cos.double()).abs() + (turned * sin.double()).abs()


def score(q, lo, hi):
    """q [G, d], lo / hi [pages, d] -> [pages]; for finite lo <= hi the sum over heads and
    channels of max(q lo, q hi)."""
    q = q.double()
    return (q.clamp(min=0).sum(0) * hi.double() + q.clamp(max=0).sum(0) * lo.double()).sum(-1)


def select(scores, n, top, first, last):
    """Ascending pages of a row with n visible pages; NaN ranks last."""
    f = min(first, n)
    l = min(last, n - f)
    forced = list(range(f)) + list(range(n - l, n))
    rest = sorted(range(f, n - l), key=lambda u: (-math.inf if math.isnan(scores[u]) else scores[u], -u), reverse=True)
    nans = [u for u in rest if math.isnan(scores[u])]
    rest = [u for u in rest if not math.isnan(scores[u])] + sorted(nans)
    return sorted(forced + rest[: max(top - len(forced), 0)])


def attend(q, k, v):
    """q [G, d], k / v [tokens, d] -> out [G, d] and an error bound's parts: sum p |v|, the largest sum |q k| / sqrt(d)."""
    if k.shape[0] == 0:
        z = torch.zeros(q.shape, dtype=torch.float64)
        return z, z, 0.0
    q, k, v = q.double(), k.double(), v.double()
    p = torch.softmax(q @ k.t() / math.sqrt(q.shape[1]), -1)
    return p @ v, p @ v.abs(), (q.abs() @ k.abs().t()).max().item() / math.sqrt(q.shape[1])


def attend_tolerance(out, pv, a, n, vmax, dtype):
    """16-bit weights (half a step each), the result's own half step, scores of 128
    fp32 products, f16 weights below their normal range."""
    half = torch.finfo(dtype).eps / 2
    return (half + 2 * 2.0 ** -17 * a + 2.0 ** -20) * pv + half * out.abs() + n * 2.0 ** -31 * vmax + 2.0 ** -25

"""A step of drafting as it is put together: projection, append of the trees' tokens, attention over
the cache and the trees, projection, next tokens, the accepted paths kept; prompts first, trees of new
sizes after, in 16 and in 8 bits; eager, on other streams and as replayed graphs."""
import pytest
import torch

import yirage_amd.fused as F
from tests.paged_plain import Batch, norm_rotate
from tests.test_gpu_fp8_cache import _check_head
from tests.test_gpu_serving_step import COLUMNS, HIDDEN, HKV, HQ, PAGE, VOCAB, Server
from tests.test_gpu_tree_edges import _check as check_attention
from tests.tree_plain import E4M3, E8M0, power, trees, values

pytestmark = pytest.mark.gpu

I32 = dict(dtype=torch.int32, device="cuda")
Q8 = pytest.mark.parametrize("q8", [False, True], ids=["16", "e4m3"])


class Drafter(Server):
    def __init__(self, seqs, most, q8, dtype=torch.bfloat16, seed=0, d=64):
        super().__init__(seqs, most, dtype, seed, d)
        self.scales = {}
        if q8:
            gen = torch.Generator().manual_seed(seed)
            byte = lambda *s: torch.randint(0, 256, s, generator=gen, dtype=torch.uint8).cuda()  # (whatever was there before)
            self.kc, self.vc = (byte(self.pool, PAGE, HKV, d).view(E4M3) for _ in range(2))
            self.ks, self.vs = (byte(self.pool, PAGE, HKV).view(E8M0) for _ in range(2))
            self.scales, self.bounds = dict(k_scale=self.ks, v_scale=self.vs), None
        self.caches = [self.kc, self.vc, *self.scales.values()] + ([] if self.bounds is None else [self.bounds])

    def draft(self, tokens, kv_len, qo=None, positions=None, mask=None, path=None):
        """tokens [T], kv_len with them -> (parts for checks, the new lengths)"""
        table, T = (self.kv_indptr, self.kv_indices, kv_len), len(tokens)
        x = self.embed[tokens]
        qkv = F.linear(x, self.wqkv).view(T, HQ + 2 * HKV, self.d)
        q, k, v = qkv.split([HQ, HKV, HKV], 1)
        more = dict(q=q, cos=self.cos, sin=self.sin, q_norm=self.q_norm, k_norm=self.k_norm, qo_indptr=qo, positions=positions)
        if self.scales:
            q = F.append_kv_paged_fp8(k, v, self.kc, self.vc, self.ks, self.vs, *table, **more)
        else:
            q = F.append_kv_paged(k, v, self.kc, self.vc, *table, page_bounds=self.bounds, **more)
        att = F.gqa_tree_paged(q, self.kc, self.vc, *table, tree_mask=mask, qo_indptr=qo, max_kv_len=self.most, **self.scales)
        logits = F.linear(F.linear(att.view(T, HQ * self.d), self.wo, residual=x), self.head)
        nxt = F.argmax(logits, VOCAB).view(-1)
        lp = F.token_logprobs(logits, nxt.long(), n_valid=VOCAB).logprob
        lens = kv_len.clone() if path is None else F.keep_kv_paged(self.kc, self.vc, *table, path, qo_indptr=qo, page_bounds=self.bounds,
                                                                   **self.scales)
        return (qkv, q, att, logits, nxt, lp), lens


def _plan(news, seed, lens):
    """Trees of `news` nodes behind `lens` tokens: qo_indptr, positions, mask and a random path from a root down."""
    parents, depth, mask = trees(news, seed)
    gen = torch.Generator().manual_seed(seed)
    qo = torch.tensor([0] + torch.tensor(news).cumsum(0).tolist(), dtype=torch.int32)
    pos = torch.from_numpy(depth).int() + torch.tensor(lens, dtype=torch.int32).repeat_interleave(torch.tensor(news))
    path = torch.full((len(news), max(news)), -1, dtype=torch.int32)
    for s, up in enumerate(parents):
        if up:
            node, chain = int(torch.randint(0, len(up), (1,), generator=gen)), []
            while node >= 0:
                chain.append(node)
                node = up[node]
            path[s, :len(chain)] = torch.tensor(chain[::-1], dtype=torch.int32)
    return qo, pos, mask, path


def _prompts(s, lens, seed):
    gen = torch.Generator().manual_seed(seed)
    qo = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), **I32)
    return s.draft(torch.randint(0, VOCAB, (sum(lens),), generator=gen).cuda(), torch.tensor(lens, **I32), qo)[0]


def _batch(s, lens, news):
    b = Batch(lens, news, PAGE)
    b.pool, b.indices = s.pool, s.kv_indices.cpu().numpy()
    b.kv_ptr = s.kv_indptr.cpu().numpy()
    return b


def _check_step(s, parts, before, after, lens, news, pos, mask):
    """before: the caches once the tokens are in, after: once the paths are kept"""
    qkv, q, att = (t.cpu() for t in parts[:3])
    cos, sin, b = s.cos.cpu(), s.sin.cpu(), _batch(s, lens, news)
    if s.scales:
        k, v = values(before[0], before[2]), values(before[1], before[3])
    else:
        k, v = before[0].double(), before[1].double()
    half = torch.finfo(q.dtype).eps / 2
    for t, place, ids in b.each_row():
        at, p = (int(ids[place // PAGE]), place % PAGE), int(pos[t])
        ref, mag = norm_rotate(qkv[t, :HQ], s.q_norm.cpu(), cos[p], sin[p], 1e-6)
        err = (s.d / 8 + 8) * 2.0 ** -24 * (1 + half)  # the norm's sum, root and products and the rotation in fp32
        assert ((q[t].double() - ref).abs() <= half * ref.abs() + err * mag + 1e-30).all()
        ref, mag = norm_rotate(qkv[t, HQ:HQ + HKV], s.k_norm.cpu(), cos[p], sin[p], 1e-6)
        if s.scales:
            for h in range(HKV):
                _check_head(before[0][at][h], power(before[2][at][h]), ref[h], mag[h])
                _check_head(before[1][at][h], power(before[3][at][h]), qkv[t, HQ + HKV + h].double(), torch.zeros(s.d))
        else:
            assert ((k[at] - ref).abs() <= half * ref.abs() + err * mag + 1e-30).all()
            assert torch.equal(before[1][at], qkv[t, HQ + HKV:])
    # (what was there before may hold NaN behind the sequences, where 64 bits do not look either)
    check_attention(b, q, k, v, att, mask, 20 if s.scales else 0)


def _moved(s, before, after, lens, news, path, got):
    ids, ptr = s.kv_indices.cpu().tolist(), s.kv_indptr.cpu().tolist()
    for b, (L, n) in enumerate(zip(lens, news)):
        kept = [p for p in path[b].tolist() if p >= 0]
        assert got[b] == L - n + len(kept)
        where = lambda p: (ids[ptr[b] + p // PAGE], p % PAGE)
        for j, p in enumerate(kept):
            for x, y in zip(before, after):
                assert torch.equal(y[where(L - n + j)], x[where(L - n + p)])


def _bytes(ts):
    return [t.cpu().view(torch.uint8) if t.dtype in (E4M3, E8M0) else t.cpu() for t in ts]


@Q8
@pytest.mark.parametrize("dtype,d", [(torch.float16, 64), (torch.bfloat16, 128)], ids=["f16", "bf16"])
def test_prompts_then_trees(dtype, d, q8):
    print("case", dtype, d, q8, flush=True)
    lens, most = [97, 1, 33, 160], 400
    s = Drafter(4, most, q8, dtype, d=d)
    parts = _prompts(s, lens, 3)
    now = [t.cpu() for t in s.caches]
    _check_step(s, parts, now, now, lens, lens, torch.cat([torch.arange(n) for n in lens]), None)
    gen = torch.Generator().manual_seed(4)
    for i, news in enumerate(([5, 1, 0, 9], [1, 1, 1, 1], [20, 33, 40, 7], [3, 3, 3, 3])):
        qo, pos, mask, path = _plan(news, i, lens)
        full = [a + n for a, n in zip(lens, news)]
        one = all(n == 1 for n in news)
        args = (torch.randint(0, VOCAB, (sum(news),), generator=gen).cuda(), torch.tensor(full, **I32), None if one else qo.cuda())
        more = dict(positions=pos.cuda(), mask=mask.cuda())
        parts, _ = s.draft(*args, **more)
        before = [t.cpu() for t in s.caches]
        again, got = s.draft(*args, path=path.cuda(), **more)  # the same tokens to the same places
        for x, y in zip(parts, again):
            assert torch.equal(x, y)
        _check_step(s, parts, before, None, full, news, pos, mask)
        _moved(s, _bytes(before)[:4 if q8 else 2], _bytes(s.caches), full, news, path, got.tolist())
        if not q8:  # each page's bounds hold its keys
            kc, bd = s.kc.cpu().float(), s.bounds.cpu().float()
            for b, L in enumerate(got.tolist()):
                ids = s.kv_indices.cpu()[int(s.kv_indptr[b]):].long()
                for p in range(L):
                    key, (lo, hi) = kc[ids[p // PAGE], p % PAGE], bd[ids[p // PAGE]].unbind(1)
                    assert (lo <= key).all() and (key <= hi).all()
        lens = got.tolist()


def test_a_tree_is_its_paths():
    """A path's nodes, appended token by token to another cache, leave what the tree's append and the keeping
    of that path leave, and their results are off by roundings alone (each is held to 64 bits)."""
    lens, news = [60, 200], [12, 12]
    s, alone = Drafter(2, 300, True, seed=5), Drafter(2, 300, True, seed=5)
    for x in (s, alone):
        _prompts(x, lens, 5)
    qo, pos, mask, path = _plan(news, 3, lens)
    deep = int((path >= 0).sum(1).min())
    assert deep >= 3
    path[:, deep:] = -1
    full = torch.tensor([72, 212], **I32)
    qkv = torch.randn((24, HQ + 2 * HKV, s.d), generator=torch.Generator().manual_seed(5)).bfloat16().cuda()

    def step(x, rows, kv_len, **tree):
        q, k, v = qkv[rows].split([HQ, HKV, HKV], 1)
        table, news = (x.kv_indptr, x.kv_indices, kv_len), tree.pop("mask", None)
        q = F.append_kv_paged_fp8(k, v, x.kc, x.vc, x.ks, x.vs, *table, q=q, cos=x.cos, sin=x.sin, q_norm=x.q_norm, k_norm=x.k_norm, **tree)
        return q, F.gqa_tree_paged(q, x.kc, x.vc, *table, tree_mask=news, qo_indptr=tree.get("qo_indptr"), **x.scales)

    q, att = step(s, torch.arange(24).cuda(), full, qo_indptr=qo.cuda(), positions=pos.cuda(), mask=mask.cuda())
    kv = [values(c.cpu(), e.cpu()) for c, e in ((s.kc, s.ks), (s.vc, s.vs))]
    check_attention(_batch(s, full.tolist(), news), q.cpu(), *kv, att.cpu(), mask, 20)
    kept = F.keep_kv_paged(s.kc, s.vc, s.kv_indptr, s.kv_indices, full, path.cuda(), qo_indptr=qo.cuda(), **s.scales)
    kv_len = torch.tensor(lens, **I32)
    for j in range(deep):
        kv_len += 1
        rows = (path[:, j].long() + torch.tensor([0, 12])).cuda()
        q1, a1 = step(alone, rows, kv_len)
        assert torch.equal(q1, q[rows])
        kv = [values(c.cpu(), e.cpu()) for c, e in ((alone.kc, alone.ks), (alone.vc, alone.vs))]
        check_attention(_batch(alone, kv_len.tolist(), [1, 1]), q1.cpu(), *kv, a1.cpu(), None, 20)
        check_attention(_batch(alone, kv_len.tolist(), [1, 1]), q1.cpu(), *kv, att[rows].cpu(), None, 20)
    assert torch.equal(kept, kv_len)
    for x, y in zip(_bytes(s.caches), _bytes(alone.caches)):
        for b, L in enumerate(kv_len.tolist()):
            ids = s.kv_indices.cpu()[int(s.kv_indptr[b]):].long()
            for p in range(L):
                assert torch.equal(x[ids[p // PAGE], p % PAGE], y[ids[p // PAGE], p % PAGE])


class Captured:
    """A step as a graph: fixed sizes, the trees' tokens, masks, positions and paths in tensors that are set
    between replays; its lengths go on by themselves."""

    def __init__(self, q8, lens, news, seed):
        self.s, self.news, self.lens = Drafter(len(lens), 500, q8, seed=seed), news, list(lens)
        _prompts(self.s, lens, seed)
        qo, pos, mask, path = _plan(news, 0, lens)
        self.qo, self.pos, self.mask, self.path = qo.cuda(), pos.cuda(), mask.cuda(), path.cuda()
        self.tokens, self.kept, self.new = torch.zeros(sum(news), dtype=torch.long, device="cuda"), torch.tensor(lens, **I32), torch.tensor(news, **I32)
        self.stream, self.graph, self.parts = torch.cuda.Stream(), None, None

    def set(self, i):
        qo, pos, mask, path = _plan(self.news, i, self.kept.tolist())
        for t, x in ((self.pos, pos), (self.mask, mask), (self.path, path)):
            t.copy_(x)
        self.tokens.copy_(torch.randint(0, VOCAB, self.tokens.shape, generator=torch.Generator().manual_seed(i)))

    def run(self):
        parts, kept = self.s.draft(self.tokens, self.kept + self.new, self.qo, self.pos, self.mask, self.path)
        self.kept.copy_(kept)
        return parts

    def capture(self):
        state = [t.clone() for t in (self.kept, *self.s.caches)]
        self.run()  # library calls' first time
        torch.cuda.synchronize()
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph, stream=self.stream):
            self.parts = self.run()
        for t, old in zip((self.kept, *self.s.caches), state):
            t.copy_(old)
        torch.cuda.synchronize()
        return self


def _eager(q8, lens, news, seed, steps):
    s, out = Captured(q8, lens, news, seed), []
    for i in range(steps):
        s.set(i)
        out.append([t.clone() for t in s.run()] + [s.kept.clone()])
    return s, out


@Q8
def test_replayed_step(q8):
    lens, news = [300, 61, 20], [14, 9, 30]
    eager, want = _eager(q8, lens, news, 1, 5)
    g = Captured(q8, lens, news, 1).capture()
    other = Captured(q8, [200, 100], [5, 40], 2)
    for i in range(5):
        g.set(i)
        g.graph.replay()
        other.set(i)
        other.run()  # eager work between the replays, on the same workspaces
        torch.cuda.synchronize()
        for x, y in zip([*g.parts, g.kept], want[i]):
            assert torch.equal(x, y), i
    for x, y in zip(_bytes(g.s.caches), _bytes(eager.s.caches)):
        assert torch.equal(x, y)


@Q8
def test_two_graphs_and_an_eager_stream_at_once(q8):
    lens, news = [400, 61], [20, 17]
    want = [_eager(q8, lens, news, seed, 4)[1] for seed in (1, 2, 3)]
    graphs = [Captured(q8, lens, news, seed).capture() for seed in (1, 2)]
    s, stream = Captured(q8, lens, news, 3), torch.cuda.Stream()
    for i in range(4):
        for g in (*graphs, s):
            g.set(i)
        torch.cuda.synchronize()
        for g in graphs:
            with torch.cuda.stream(g.stream):
                g.graph.replay()
        with torch.cuda.stream(stream):
            mine = s.run()
        torch.cuda.synchronize()
        for parts, g, w in ((graphs[0].parts, graphs[0], want[0]), (graphs[1].parts, graphs[1], want[1]), (mine, s, want[2])):
            for x, y in zip([*parts, g.kept], w[i]):
                assert torch.equal(x, y), i

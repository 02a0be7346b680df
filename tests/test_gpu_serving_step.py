"""A serving step as it is put together: projection, append, page selection, sparse
attention, projection, log probabilities; prompts and then single tokens, eager,
on other streams and as replayed graphs."""
import math

import pytest
import torch

import paged_plain as P
import yirage_amd.fused as F
from test_gpu_logprobs import _check as check_logprobs

pytestmark = pytest.mark.gpu

HIDDEN, HQ, HKV, PAGE = 256, 8, 2, 16
VOCAB, COLUMNS = 1031, 1032  # the products' columns are multiples of 8
TOP = 4


class Server:
    """One layer's weights and caches, with room for `most` tokens a sequence."""

    def __init__(self, seqs, most, dtype=torch.bfloat16, seed=0, d=64):
        self.d = d
        gen = torch.Generator().manual_seed(seed)
        rnd = lambda *s, std=1.0: (std * torch.randn(s, generator=gen)).to(dtype).cuda()
        self.embed = rnd(VOCAB, HIDDEN)
        self.wqkv = rnd((HQ + 2 * HKV) * d, HIDDEN, std=HIDDEN ** -0.5)
        self.wo = rnd(HIDDEN, HQ * d, std=(HQ * d) ** -0.5)
        self.head = rnd(COLUMNS, HIDDEN, std=2 * HIDDEN ** -0.5)
        self.q_norm, self.k_norm = 1 + rnd(d, std=0.1), 1 + rnd(d, std=0.1)
        cos, sin = P.tables(most, d)
        self.cos, self.sin = cos.float().cuda(), sin.float().cuda()
        npg = -(-most // PAGE)
        self.most, self.pool = most, seqs * npg + 2
        self.kc, self.vc = rnd(self.pool, PAGE, HKV, d), rnd(self.pool, PAGE, HKV, d)  # (whatever was there before)
        self.bounds = rnd(self.pool, HKV, 2, d)
        order = torch.randperm(self.pool, generator=gen)[: seqs * npg]
        self.kv_indices = order.to(torch.int32).cuda()
        self.kv_indptr = (torch.arange(seqs + 1, dtype=torch.int32) * npg).cuda()

    def step(self, tokens, kv_len, qo_indptr=None, top=TOP):
        """tokens [T] -> (their rows' parts in order, for checks)"""
        table = (self.kv_indptr, self.kv_indices, kv_len)
        x = self.embed[tokens]
        qkv = F.linear(x, self.wqkv).view(len(tokens), HQ + 2 * HKV, self.d)
        k, v = qkv[:, HQ: HQ + HKV], qkv[:, HQ + HKV:]
        q = F.append_kv_paged(k, v, self.kc, self.vc, *table, q=qkv[:, :HQ], cos=self.cos, sin=self.sin, q_norm=self.q_norm,
                              k_norm=self.k_norm, qo_indptr=qo_indptr, page_bounds=self.bounds)
        pages = F.select_pages(q, self.bounds, *table, page_size=PAGE, top_pages=top, qo_indptr=qo_indptr, max_kv_len=self.most)
        att = F.gqa_sparse_paged(q, self.kc, self.vc, *table, pages, qo_indptr=qo_indptr)
        logits = F.linear(F.linear(att.view(len(tokens), HQ * self.d), self.wo, residual=x), self.head)
        nxt = F.argmax(logits, VOCAB).view(-1)
        lp = F.token_logprobs(logits, nxt.long(), top_n=3, n_valid=VOCAB)
        return qkv, q, pages, att, logits, nxt, lp


def _check_step(s, parts, lens, news, top=TOP):
    """Each operator's result against 64 bits, from what the one before it gave."""
    qkv, q, pages, att, logits, nxt, lp = (t.cpu() if torch.is_tensor(t) else t for t in parts)
    kc, vc, bounds = s.kc.cpu(), s.vc.cpu(), s.bounds.cpu()
    cos, sin = s.cos.cpu(), s.sin.cpu()
    ids_all, ptr = s.kv_indices.cpu().tolist(), s.kv_indptr.cpu().tolist()
    half, eps = torch.finfo(q.dtype).eps / 2, 1e-6
    row, g = 0, HQ // HKV
    for b, (L, n) in enumerate(zip(lens, news)):
        ids = ids_all[ptr[b]: ptr[b + 1]]
        for u in range(max(L - n, 0) // PAGE, -(-L // PAGE)):  # the pages that the step touched
            keys = kc[ids[u], : min(L - u * PAGE, PAGE)].float()
            assert torch.equal(bounds[ids[u], :, 0].float(), keys.amin(0)) and torch.equal(bounds[ids[u], :, 1].float(), keys.amax(0))
        for i in range(n):
            p = L - n + i
            at = (ids[p // PAGE], p % PAGE)
            for got, raw, w in [(q[row], qkv[row, :HQ], s.q_norm), (kc[at], qkv[row, HQ: HQ + HKV], s.k_norm)]:
                ref, mag = P.norm_rotate(raw, w.cpu(), cos[p], sin[p], eps)
                # half a step of the result; the norm's sum, root and products and the rotation in fp32
                assert ((got.double() - ref).abs() <= half * ref.abs() + (s.d / 8 + 8) * 2.0 ** -24 * mag * (1 + half) + 1e-30).all()
            assert torch.equal(vc[at], qkv[row, HQ + HKV:])
            seen = p // PAGE + 1
            lo, hi = (bounds[ids[:seen]][:, :, j] for j in (0, 1))
            for h in range(HKV):
                want = P.select(P.score(q[row, h * g: (h + 1) * g], lo[:, h], hi[:, h]).tolist(), seen, top, 1, 1)
                assert pages[row, h].tolist() == want + [-1] * (top - len(want)), (b, i, h)
                k = torch.cat([kc[ids[u], :, h][: p + 1 - u * PAGE] for u in want])
                v = torch.cat([vc[ids[u], :, h][: p + 1 - u * PAGE] for u in want])
                ref, pv, a = P.attend(q[row, h * g: (h + 1) * g], k, v)
                tol = P.attend_tolerance(ref, pv, a, len(k), v.double().abs().max().item(), q.dtype)
                assert ((att[row, h * g: (h + 1) * g].double() - ref).abs() <= tol).all(), (b, i, h)
            row += 1
    check_logprobs(logits, nxt, 3, lp, VOCAB)
    assert torch.equal(lp.top_token[:, 0].cpu(), nxt.long())  # the greedy choice is the likeliest


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
def test_prompts_then_tokens(dtype):
    print("case", dtype, flush=True)
    lens, most = [97, 1, 33, 160], 200
    s = Server(len(lens), most, dtype)
    gen = torch.Generator().manual_seed(3)
    kv_len = torch.tensor(lens, dtype=torch.int32).cuda()
    qo = torch.tensor([0, 97, 98, 131, 291], dtype=torch.int32).cuda()
    parts = s.step(torch.randint(0, VOCAB, (sum(lens),), generator=gen).cuda(), kv_len, qo)
    _check_step(s, parts, lens, lens)
    tokens = parts[5][(qo[1:] - 1).long()].long()
    for i in range(20):  # over the ends of pages
        kv_len += 1
        lens = [n + 1 for n in lens]
        parts = s.step(tokens, kv_len)
        if i % 5 == 0 or i > 17:
            _check_step(s, parts, lens, [1] * 4)
        tokens = parts[5].long()
    # three drafted tokens a sequence at once
    kv_len += 3
    lens = [n + 3 for n in lens]
    parts = s.step(tokens.repeat_interleave(3), kv_len, torch.arange(0, 13, 3, dtype=torch.int32).cuda())
    _check_step(s, parts, lens, [3] * 4)


def test_all_pages_selected_is_dense_attention():
    lens, most = [190, 64, 5], 200
    s = Server(3, most, d=128)
    gen = torch.Generator().manual_seed(4)
    kv_len = torch.tensor(lens, dtype=torch.int32).cuda()
    qo = torch.tensor([0, 190, 254, 259], dtype=torch.int32).cuda()
    s.step(torch.randint(0, VOCAB, (sum(lens),), generator=gen).cuda(), kv_len, qo)
    kv_len += 1
    parts = s.step(torch.tensor([3, 4, 5]).cuda(), kv_len, top=13)
    dense = F.gqa_decode_paged(parts[1], s.kc, s.vc, s.kv_indptr, s.kv_indices, kv_len, most)
    # each is off by its 16-bit weights and result: a step of the sums of |v| and of the result
    eps = torch.finfo(dense.dtype).eps
    vmax = s.vc.abs().max().item()
    assert ((parts[3].float() - dense.float()).abs() <= eps * dense.float().abs() + 1.25 * eps * vmax).all()


def _same(a, b):
    for x, y in zip(a, b):
        assert all(torch.equal(i, j) for i, j in zip(x, y)) if isinstance(x, tuple) else torch.equal(x, y)


def _copy(parts):
    return [tuple(t.clone() for t in p) if isinstance(p, tuple) else p.clone() for p in parts]


def _prefill(s, lens, seed):
    gen = torch.Generator().manual_seed(seed)
    kv_len = torch.tensor(lens, dtype=torch.int32).cuda()
    qo = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32).cuda()
    parts = s.step(torch.randint(0, VOCAB, (sum(lens),), generator=gen).cuda(), kv_len, qo)
    return kv_len, parts[5][(qo[1:] - 1).long()].long()


class Captured:
    """A decode step as a graph that takes its own tokens and lengths forward."""

    def __init__(self, seqs, most, lens, seed):
        self.s = Server(seqs, most, seed=seed)
        self.kv_len, self.tokens = _prefill(self.s, lens, seed)
        self.stream = torch.cuda.Stream()
        state = (self.kv_len.clone(), self.tokens.clone(), self.s.kc.clone(), self.s.vc.clone(), self.s.bounds.clone())
        self.run()  # library calls' first time
        torch.cuda.synchronize()
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph, stream=self.stream):
            self.parts = self.run()
        for t, old in zip((self.kv_len, self.tokens, self.s.kc, self.s.vc, self.s.bounds), state):
            t.copy_(old)
        torch.cuda.synchronize()

    def run(self):
        self.kv_len.add_(1)
        parts = self.s.step(self.tokens, self.kv_len)
        self.tokens.copy_(parts[5])
        return parts


def test_replayed_step():
    lens = [700, 61, 350]
    eager = Server(3, 800, seed=1)
    kv_len, tokens = _prefill(eager, lens, 1)
    g = Captured(3, 800, lens, 1)
    other = Server(2, 300, seed=2)  # eager work between the replays, on the same workspaces
    other_len, other_tokens = _prefill(other, [200, 100], 2)
    for i in range(6):
        g.graph.replay()
        kv_len += 1
        parts = eager.step(tokens, kv_len)
        tokens = parts[5].long()
        other_len += 1
        other_tokens = other.step(other_tokens, other_len)[5].long()
        torch.cuda.synchronize()
        _same(g.parts, parts)
        assert torch.equal(g.s.kc, eager.kc) and torch.equal(g.s.bounds, eager.bounds)
    _check_step(g.s, g.parts, [n + 6 for n in lens], [1] * 3)


def test_two_graphs_and_an_eager_stream_at_once():
    lens = [600, 61, 350]
    want = []
    for seed in (1, 2, 3):
        s = Server(3, 700, seed=seed)
        kv_len, tokens = _prefill(s, lens, seed)
        steps = []
        for _ in range(4):
            kv_len += 1
            parts = s.step(tokens, kv_len)
            tokens = parts[5].long()
            steps.append(_copy(parts))
        want.append(steps)
    graphs = [Captured(3, 700, lens, seed) for seed in (1, 2)]
    s, stream = Server(3, 700, seed=3), torch.cuda.Stream()
    kv_len, tokens = _prefill(s, lens, 3)
    torch.cuda.synchronize()
    for i in range(4):
        for g in graphs:
            with torch.cuda.stream(g.stream):
                g.graph.replay()
        with torch.cuda.stream(stream):
            kv_len += 1
            parts = s.step(tokens, kv_len)
            tokens = parts[5].long()
        torch.cuda.synchronize()
        _same(parts, want[2][i])
        for g, w in zip(graphs, want):
            _same(g.parts, w[i])

"""The operators of a serving step around a paged key-value cache, as measurable
cases: appending rotated keys and values (with each page's key bounds),
selecting pages by those bounds, attention over the selected pages, and token
log probabilities.

Sizes are those of a Llama-3-8B-shaped model (32 / 8 heads of 128, vocabulary
128256, pages of 64) and generic ones around them; draw() spreads lengths, page
sizes, head counts, head dims and types.

Layouts: caches [pages, page, kv heads, d], bounds [pages, kv heads, 2, d]
(smallest, largest key per channel), rows of a ragged batch back to back
(sequence b: rows qo_indptr[b] .. qo_indptr[b + 1]), page table and lengths
int32 as for the paged decode.
"""
import math

import numpy as np
import torch

own = False  # True: run() calls this package's operators; False: their plain forms

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
VOCAB = 128256
THETA = 500000.0
EPS = 1e-6
DEVICE = "cuda"


def listed():
    return [
        # one token of one conversation: the smallest call, latency only
        {"name": "append_step_b1", "op": "append", "seqs": 1, "new": 1, "kv": 4096, "hq": 32, "hkv": 8, "d": 128,
         "page": 64, "norm": False, "dtype": "bf16"},
        # a serving batch's decode step, sequences of different lengths, q / k normalised per head
        {"name": "append_step_b64", "op": "append", "seqs": 64, "new": 1, "kv": 2048, "hq": 32, "hkv": 8, "d": 128,
         "page": 16, "norm": True, "dtype": "f16"},
        # a batch of prompts of up to 2048 tokens, the largest append
        {"name": "append_prompts_b8", "op": "append", "seqs": 8, "new": 2048, "kv": 2048, "hq": 32, "hkv": 8, "d": 128,
         "page": 64, "norm": False, "dtype": "bf16"},
        # one conversation 128 K tokens in: 2048 pages to choose from
        {"name": "select_step_b1", "op": "select", "seqs": 1, "new": 1, "kv": 131072, "hq": 32, "hkv": 8, "d": 128,
         "page": 64, "top": 64, "dtype": "bf16"},
        # a decode batch of long conversations, small pages
        {"name": "select_step_b32", "op": "select", "seqs": 32, "new": 1, "kv": 16384, "hq": 32, "hkv": 8, "d": 128,
         "page": 16, "top": 128, "dtype": "f16"},
        # a chunk of a long prompt: every row chooses for itself
        {"name": "select_chunk_512", "op": "select", "seqs": 1, "new": 512, "kv": 32768, "hq": 32, "hkv": 8, "d": 128,
         "page": 64, "top": 32, "dtype": "bf16"},
        # one conversation, 2048 of 32 K tokens read
        {"name": "sparse_step_b1", "op": "sparse", "seqs": 1, "new": 1, "kv": 32768, "hq": 32, "hkv": 8, "d": 128,
         "page": 64, "top": 32, "dtype": "bf16"},
        # a decode batch, 16-token pages, 8 query heads a kv head of 64
        {"name": "sparse_step_b32", "op": "sparse", "seqs": 32, "new": 1, "kv": 8191, "hq": 64, "hkv": 8, "d": 64,
         "page": 16, "top": 128, "dtype": "f16"},
        # a chunk of a prompt of no round length after 15 K tokens
        {"name": "sparse_chunk_777", "op": "sparse", "seqs": 1, "new": 777, "kv": 16000, "hq": 32, "hkv": 8, "d": 128,
         "page": 64, "top": 16, "dtype": "bf16"},
        # the next token's probabilities with 20 alternatives, one conversation
        {"name": "logprobs_b1", "op": "logprobs", "rows": 1, "n": VOCAB, "top": 20, "masked": False, "dtype": "bf16"},
        # a decode batch under a grammar: most tokens masked out, a vocabulary of odd size
        {"name": "logprobs_b64", "op": "logprobs", "rows": 64, "n": 50001, "top": 5, "masked": True, "dtype": "f32"},
        # scoring a 2048-token prompt
        {"name": "logprobs_prompt_2048", "op": "logprobs", "rows": 2048, "n": VOCAB, "top": 5, "masked": False,
         "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "select", "sparse", "logprobs"])
    if op == "logprobs":
        n, dtype = _log(rng, 1000, 152000), rng.choice(["f16", "bf16", "f32"])
        rows = 2048 * VOCAB // (2 * n if dtype == "f32" else n)
        return {"op": op, "rows": _log(rng, 1, min(2048, rows)), "n": n, "top": rng.choice([0, 1, 5, 20]),
                "masked": rng.random() < 0.3, "dtype": dtype}
    hkv, group, d = rng.choice([(1, 8, 128), (2, 4, 128), (2, 7, 64), (2, 7, 128), (4, 1, 64), (4, 1, 128), (4, 5, 128),
                                (4, 16, 128), (8, 1, 64), (8, 2, 64), (8, 4, 128), (8, 8, 64), (8, 8, 128)])
    case = {"op": op, "hq": hkv * group, "hkv": hkv, "d": d,
            "page": rng.choice([16, 32, 64, 128]), "dtype": rng.choice(["f16", "bf16"])}
    if op == "append":
        seqs = _log(rng, 1, 64)
        most = 12288 * 48 * 128 // ((case["hq"] + 2 * hkv) * d * seqs)
        new = 1 if rng.random() < 0.5 else _log(rng, 2, max(2, min(2048, most)))
        return {**case, "seqs": seqs, "new": new, "kv": new + _log(rng, 1, 2048), "norm": rng.random() < 0.5}
    top = rng.choice([4, 8, 16, 32])
    # select: enough pages for a choice; attention: short sequences too
    least, most = (4 * top * case["page"], 131072) if op == "select" else (64, 32768)
    if rng.random() < 0.6:  # a decode step
        most_seqs = 64 if op == "select" else 32 * 2048 * 8 * 64 // (top * case["page"] * hkv * d)
        seqs, new = _log(rng, 1, max(1, min(64, most_seqs))), 1
        kv = _log(rng, least, max(least, min(most, 262144 // seqs)))
    else:  # new rows after a long prefix: a verified draft, a chunk of a prompt
        seqs = _log(rng, 1, 4)
        kv = _log(rng, least, max(least, most // 4))
        new = _log(rng, 2, max(2, min(128, 700000 // (seqs * (top * case["page"] if op == "sparse" else kv // case["page"])))))
        kv += new
    return {**case, "seqs": seqs, "new": new, "kv": kv, "top": top}


# ------------------------------------------------------------------ inputs
def _normal(gen, shape, std, dtype):
    return torch.empty(shape, dtype=dtype, device=DEVICE).normal_(0.0, std, generator=gen)


def _lengths(case):
    """Lengths and new rows of a batch in service: the first sequence has kv tokens
    and the most new rows, the others half to all of that. The case alone decides."""
    rng = np.random.default_rng([case["seqs"], case["new"], case["kv"]])
    news = rng.integers((case["new"] + 1) // 2, case["new"] + 1, size=case["seqs"])
    lens = rng.integers((case["kv"] + 1) // 2, case["kv"] + 1, size=case["seqs"])
    news[0], lens[0] = case["new"], case["kv"]
    return np.maximum(lens, news), news


def _batch(case, seed):
    """Lengths, new rows and a shuffled page table."""
    lens, news = _lengths(case)
    npg = -(-lens // case["page"])
    pool = int(npg.sum()) + 2

    def dev(a):
        return torch.from_numpy(np.asarray(a, dtype=np.int32)).to(DEVICE)

    return {"lens": lens, "news": news, "pool": pool, "kv_len": dev(lens),
            "kv_indptr": dev(np.concatenate([[0], np.cumsum(npg)])),
            "kv_indices": dev(np.random.default_rng(seed).permutation(pool)[: int(npg.sum())]),
            "qo_indptr": dev(np.concatenate([[0], np.cumsum(news)])) if case["new"] > 1 else None}


def _keys(case, gen, pool):
    """Keys of a page have something in common, as those of a passage do."""
    shape = (pool, case["page"], case["hkv"], case["d"])
    k = _normal(gen, shape, 1.0, DTYPES[case["dtype"]])
    return k.add_(_normal(gen, (pool, 1, case["hkv"], case["d"]), 0.5, k.dtype))


def _queries(case, gen, rows):
    """Queries of neighbouring rows resemble each other: half of each is shared by 64 rows."""
    q = _normal(gen, (rows, case["hq"], case["d"]), 0.7, DTYPES[case["dtype"]])
    shared = _normal(gen, (-(-rows // 64), case["hq"], case["d"]), 0.7, q.dtype)
    return q.add_(shared.repeat_interleave(64, 0)[:rows])


def _tables(case, seed):
    """cos / sin rows of the rotate-half rotation, [positions, d] in 32 bits."""
    d = case["d"]
    inv = THETA ** (-np.arange(0, d, 2, dtype=np.float64) / d)
    ang = np.outer(np.arange(case["kv"], dtype=np.float64), np.concatenate([inv, inv]))
    return tuple(torch.from_numpy(f(ang).astype(np.float32)).to(DEVICE) for f in (np.cos, np.sin))


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    if case["op"] == "logprobs":
        # a few likely tokens stand apart from the rest
        x = _normal(gen, (case["rows"], case["n"]), 2.0, dt)
        x[:, ::257] += 4.0
        if case["masked"]:
            x.masked_fill_(torch.rand(x.shape, device=DEVICE, generator=gen) < 0.9, -math.inf)
        rows = torch.arange(case["rows"], device=DEVICE)
        tokens = torch.randint(0, case["n"], (case["rows"],), device=DEVICE, generator=gen)
        x[rows, tokens] = _normal(gen, (case["rows"],), 2.0, dt)  # the given tokens are allowed ones
        return {"case": case, "logits": x, "tokens": tokens}
    s = {"case": case, **_batch(case, seed)}
    rows, B = int(s["news"].sum()), case["seqs"]
    if case["op"] == "append":
        # k and v are slices of one projection's output, as programs have them
        qkv = _normal(gen, (rows, case["hq"] + 2 * case["hkv"], case["d"]), 1.0, dt)
        s["q"], s["k"], s["v"] = qkv.split([case["hq"], case["hkv"], case["hkv"]], 1)
        s["cos"], s["sin"] = _tables(case, seed)
        s["q_norm"] = s["k_norm"] = None
        if case["norm"]:
            s["q_norm"], s["k_norm"] = (1 + _normal(gen, (2, case["d"]), 0.1, dt)).unbind(0)
        s["k_cache"] = _keys(case, gen, s["pool"])
        s["v_cache"] = _normal(gen, s["k_cache"].shape, 1.0, dt)
        # what the pages held before: the tokens in front of the new ones
        old = torch.zeros((s["pool"], case["page"]), dtype=torch.bool, device=DEVICE)
        for b, pages in enumerate(_pages_of(s)):
            n = int(s["lens"][b] - s["news"][b])
            old[pages] = (torch.arange(pages.numel() * case["page"], device=DEVICE) < n).view(-1, case["page"])
        k, hidden = s["k_cache"], ~old[:, :, None, None]
        s["bounds"] = torch.stack([k.masked_fill(hidden, math.inf).amin(1), k.masked_fill(hidden, -math.inf).amax(1)], 2)
        s["bounds"][~old.any(1)] = 0  # an empty page's bounds mean nothing
        return s
    s["q"] = _queries(case, gen, rows)
    k = _keys(case, gen, s["pool"]) if case["op"] == "sparse" else None
    if k is None:
        # bounds alone: centre and half width of a page's keys
        shape = (s["pool"], case["hkv"], case["d"])
        mid = _normal(gen, shape, 0.5, torch.float32)
        half = 1.8 + _normal(gen, shape, 0.3, torch.float32).abs()
        s["bounds"] = torch.stack([mid - half, mid + half], 2).to(dt)
        return s
    s["k_cache"], s["v_cache"] = k, _normal(gen, k.shape, 1.0, dt)
    s["bounds"] = torch.stack([k.amin(1), k.amax(1)], 2)
    s["pages"] = _select(s)
    return s


def _pages_of(s):
    """Page ids of each sequence."""
    ptr = [0] + np.cumsum(-(-s["lens"] // s["case"]["page"])).tolist()
    return [s["kv_indices"][a:b].long() for a, b in zip(ptr, ptr[1:])]


# ------------------------------------------------------------------ plain forms
def _rows(s):
    """Sequence and position of every row."""
    lens = s["kv_len"].long()
    if s["qo_indptr"] is None:
        return torch.arange(lens.numel(), device=DEVICE), lens - 1
    ptr = s["qo_indptr"].long()
    row = torch.arange(s["q"].shape[0], device=DEVICE)
    seq = torch.searchsorted(ptr[1:].contiguous(), row, right=True)
    return seq, lens[seq] - (ptr[seq + 1] - row)


def _rotate(x, weight, cos, sin):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    half = x.shape[-1] // 2
    return x * cos[:, None] + torch.cat([-x[..., half:], x[..., :half]], -1) * sin[:, None]


def _append(s):
    dt, page = s["k"].dtype, s["case"]["page"]
    seq, pos = _rows(s)
    cos, sin = s["cos"][pos], s["sin"][pos]
    k = _rotate(s["k"], s["k_norm"], cos, sin).to(dt)
    q = _rotate(s["q"], s["q_norm"], cos, sin).to(dt)
    ids, slot = s["kv_indices"].long()[s["kv_indptr"].long()[seq] + pos // page], pos % page
    s["k_cache"][ids, slot] = k
    s["v_cache"][ids, slot] = s["v"]
    lo, hi = s["bounds"].float().unbind(2)
    lo[ids[slot == 0]], hi[ids[slot == 0]] = math.inf, -math.inf
    to = ids[:, None, None].expand(k.shape)
    lo.scatter_reduce_(0, to, k.float(), "amin")
    hi.scatter_reduce_(0, to, k.float(), "amax")
    s["bounds"].copy_(torch.stack([lo, hi], 2))
    return q, s["k_cache"], s["v_cache"], s["bounds"]


def _select(s):
    """Page numbers within the sequence, ascending, -1 behind: the first page, the
    last visible one and the best bounds. Scores in 64 bits, since the border
    between the last taken and the first left page can be narrow."""
    c = s["case"]
    hkv, page, top = c["hkv"], c["page"], c["top"]
    seq, pos = _rows(s)
    q = s["q"].double().unflatten(1, (hkv, -1))
    up, down = q.clamp(min=0).sum(2), q.clamp(max=0).sum(2)
    out = torch.full((q.shape[0], hkv, top), -1, dtype=torch.int32, device=DEVICE)
    row = 0
    for pages, n in zip(_pages_of(s), s["news"].tolist()):
        r = slice(row, row + n)
        row += n
        lo, hi = s["bounds"][pages].double().permute(2, 1, 3, 0)
        score = (up[r].transpose(0, 1) @ hi + down[r].transpose(0, 1) @ lo).transpose(0, 1)  # [rows, kv heads, pages]
        last = (pos[r] // page)[:, None, None]
        u = torch.arange(pages.numel(), device=DEVICE)
        score = torch.where((u == 0) | (u == last), math.inf, score)
        score = torch.where(u <= last, score, -math.inf)
        best = torch.sort(score, dim=-1, descending=True, stable=True)
        take = min(top, pages.numel())
        kept = torch.where(best.indices <= last, best.indices, 2 ** 31 - 1)[..., :take].sort(-1).values
        out[r, :, :take] = torch.where(kept == 2 ** 31 - 1, -1, kept).int()
    return out


def _sparse(s):
    c = s["case"]
    hkv, page, d = c["hkv"], c["page"], c["d"]
    seq, pos = _rows(s)
    q = s["q"].float().unflatten(1, (hkv, -1))
    k, v = s["k_cache"].transpose(1, 2), s["v_cache"].transpose(1, 2)
    heads = torch.arange(hkv, device=DEVICE)[None, :, None]
    out = []
    for r in range(0, q.shape[0], 64):
        p = s["pages"][r:r + 64].long()
        ids = s["kv_indices"].long()[s["kv_indptr"].long()[seq[r:r + 64]][:, None, None] + p.clamp(min=0)]
        token = p[..., None] * page + torch.arange(page, device=DEVICE)
        seen = ((p[..., None] >= 0) & (token <= pos[r:r + 64][:, None, None, None])).flatten(2)
        kf, vf = (x[ids, heads].float().flatten(2, 3) for x in (k, v))
        a = (q[r:r + 64] @ kf.transpose(2, 3).contiguous()) / math.sqrt(d)
        a = torch.where(seen[:, :, None], a, -math.inf)
        e = torch.exp(a - a.amax(-1, keepdim=True))
        out.append((e / e.sum(-1, keepdim=True)) @ vf)
    return torch.cat(out).flatten(1, 2).to(s["q"].dtype)


def _logprobs(s):
    c, tokens = s["case"], s["tokens"][:, None]
    parts = []
    for x, t in zip(s["logits"].split(256), tokens.split(256)):
        x = x.float()
        y = x - x.amax(-1, keepdim=True)
        e = torch.exp(y)
        # 64 bits: a nearly certain token leaves sums next to 1
        z = e.sum(-1, keepdim=True, dtype=torch.float64)
        log_z = torch.log(z)
        entropy = log_z[:, 0] - torch.where(e > 0, e * y, 0.0).sum(-1, dtype=torch.float64) / z[:, 0]
        # whole-number keys: larger values first, the lowest token first among equals
        bits = x.view(torch.int32).long()
        order = torch.where(bits < 0, -(bits & 0x7fffffff), bits) * 2 ** 20 + (2 ** 20 - 1 - torch.arange(c["n"], device=DEVICE))
        ids = torch.topk(order, c["top"], -1).indices
        parts.append(((y.gather(1, t) - log_z)[:, 0].float(), entropy.float(), (y.gather(1, ids) - log_z).float(), ids))
    return tuple(torch.cat(p) for p in zip(*parts))


def run(s):
    c = s["case"]
    op = c["op"]
    if not own:
        return {"append": _append, "select": _select, "sparse": _sparse, "logprobs": _logprobs}[op](s)
    from yirage_amd import fused

    if op == "logprobs":
        return tuple(fused.token_logprobs(s["logits"], s["tokens"], top_n=c["top"]))
    table = (s["kv_indptr"], s["kv_indices"], s["kv_len"])
    if op == "append":
        q = fused.append_kv_paged(s["k"], s["v"], s["k_cache"], s["v_cache"], *table, q=s["q"], cos=s["cos"], sin=s["sin"],
                                  q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS, qo_indptr=s["qo_indptr"],
                                  page_bounds=s["bounds"])
        return q, s["k_cache"], s["v_cache"], s["bounds"]
    if op == "select":
        return fused.select_pages(s["q"], s["bounds"], *table, page_size=c["page"], top_pages=c["top"],
                                  qo_indptr=s["qo_indptr"], max_kv_len=c["kv"])
    return fused.gqa_sparse_paged(s["q"], s["k_cache"], s["v_cache"], *table, s["pages"], qo_indptr=s["qo_indptr"])


def work(case):
    if case["op"] == "logprobs":
        size = 4 if case["dtype"] == "f32" else 2
        cells = case["rows"] * case["n"]
        return {"bytes": size * cells + case["rows"] * (16 + 12 * case["top"]), "flops": 5 * cells}
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    lens, news = _lengths(case)
    rows, pages = int(news.sum()), -(-lens // page)
    if case["op"] == "append":
        touched = int((pages - (lens - news) // page).sum())
        move = 4 * rows * (hq + 2 * hkv) * d + 8 * int(news.max()) * d + touched * 8 * hkv * d
        return {"bytes": move, "flops": 3 * rows * (hq + hkv) * d}
    if case["op"] == "select":
        return {"bytes": int(pages.sum()) * hkv * 4 * d + 2 * rows * hq * d + 4 * rows * hkv * case["top"],
                "flops": 4 * int((news * pages).sum()) * hkv * d}
    # one row's pages at least; rows of a sequence share what they have in common
    read = np.minimum(lens, case["top"] * page)
    return {"bytes": 4 * int(read.sum()) * hkv * d + 4 * rows * hq * d + 4 * rows * hkv * case["top"],
            "flops": 4 * int((news * read).sum()) * hq * d}


# ------------------------------------------------------------------ 64 bits
def _exact_rotate(x, weight, cos, sin):
    """Pair (i, i + d / 2) turned as a complex number, the two halves with their own angle rows."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + EPS) * weight.double()
    a, b = x.chunk(2, -1)
    (ca, cb), (sa, sb) = (t.double()[:, None].chunk(2, -1) for t in (cos, sin))
    return torch.cat([a * ca - b * sa, b * cb + a * sb], -1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        out = []
        for x, t in zip(s["logits"].split(128), s["tokens"].split(128)):
            lp = torch.log_softmax(x.double(), -1)
            ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :case["top"]]
            h = -torch.where(lp == -math.inf, 0.0, lp.exp() * lp).sum(-1)
            out.append((lp[torch.arange(len(t), device=DEVICE), t], h, lp.gather(1, ids), ids))
        return tuple(torch.cat(p) for p in zip(*out))
    hkv, d, page = case["hkv"], case["d"], case["page"]
    pages = _pages_of(s)
    starts = np.concatenate([[0], np.cumsum(s["news"])]).tolist()
    if case["op"] == "append":
        q = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
        kc, vc, bounds = s["k_cache"].double(), s["v_cache"].double(), s["bounds"].double()
        for b, ids in enumerate(pages):
            L, n, r = int(s["lens"][b]), int(s["news"][b]), slice(starts[b], starts[b + 1])
            cos, sin = s["cos"][L - n:L], s["sin"][L - n:L]
            q[r] = _exact_rotate(s["q"][r], s["q_norm"], cos, sin)
            flat_k, flat_v = kc[ids].flatten(0, 1), vc[ids].flatten(0, 1)
            flat_k[L - n:L] = _exact_rotate(s["k"][r], s["k_norm"], cos, sin)
            flat_v[L - n:L] = s["v"][r].double()
            kc[ids], vc[ids] = flat_k.view(-1, page, hkv, d), flat_v.view(-1, page, hkv, d)
            for u in range((L - n) // page, (L - 1) // page + 1):
                seen = flat_k[u * page:min(L, (u + 1) * page)]
                bounds[ids[u], :, 0], bounds[ids[u], :, 1] = seen.amin(0), seen.amax(0)
        return q, kc, vc, bounds
    if case["op"] == "select":
        out = torch.full((s["q"].shape[0], hkv, case["top"]), -1, dtype=torch.int32, device=DEVICE)
        for b, ids in enumerate(pages):
            lo, hi = s["bounds"][ids].double().unbind(2)
            first = int(s["lens"][b] - s["news"][b])
            for h in range(hkv):
                q = s["q"][starts[b]:starts[b + 1]].double().unflatten(1, (hkv, -1))[:, h]
                score = torch.cat([torch.maximum(x[:, :, None] * lo[:, h], x[:, :, None] * hi[:, h]).sum((1, 3))
                                   for x in q.split(16)])
                n = ids.numel()
                here = (first + torch.arange(len(q), device=DEVICE)) // page
                score[:, 0] = math.inf
                score[torch.arange(len(q), device=DEVICE), here] = math.inf
                hidden = torch.arange(n, device=DEVICE)[None] > here[:, None]
                rank = score.masked_fill(hidden, -math.inf).argsort(dim=-1, descending=True, stable=True).argsort(dim=-1)
                chosen = (rank < case["top"]) & ~hidden
                at = chosen.cumsum(-1) - 1
                rows, cols = chosen.nonzero(as_tuple=True)
                out[starts[b] + rows, h, at[rows, cols]] = cols.int()
        return out
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE).unflatten(1, (hkv, -1))
    for b, ids in enumerate(pages):
        n, first = int(s["news"][b]), int(s["lens"][b] - s["news"][b])
        token = torch.arange(ids.numel() * page, device=DEVICE)
        for h in range(hkv):
            k, v = (s[x][ids][:, :, h].flatten(0, 1).double() for x in ("k_cache", "v_cache"))
            for r in range(0, n, 256):
                m = min(256, n - r)
                at = slice(starts[b] + r, starts[b] + r + m)
                chosen = torch.zeros((m, ids.numel() + 1), dtype=torch.bool, device=DEVICE)
                listed_pages = s["pages"][at, h].long()
                chosen.scatter_(1, torch.where(listed_pages < 0, ids.numel(), listed_pages), True)
                seen = chosen[:, :-1].repeat_interleave(page, 1)
                seen &= token <= (first + r + torch.arange(m, device=DEVICE))[:, None]
                q = s["q"][at].double().unflatten(1, (hkv, -1))[:, h]
                a = (q.reshape(-1, d) @ k.t() / math.sqrt(d)).view(m, -1, token.numel())
                out[at, h] = (torch.softmax(a.masked_fill(~seen[:, None], -math.inf), -1).reshape(-1, token.numel()) @ v).view(m, -1, d)
    return out.flatten(1, 2)

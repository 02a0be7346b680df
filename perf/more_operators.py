"""Drafting over a paged key-value cache in 8 bits, as measurable cases: appending
rotated keys and values as e4m3 with a power of two per token and head (codes that
float lose nothing to a scale without a fraction), attention of single tokens, trees
of drafted tokens and chunks of prompts over such a cache (or one in 16 bits), reading
the cache back, and keeping the accepted path of a tree.

Sizes are those of a Llama-3-8B-shaped model (32 / 8 heads of 128, pages of 64) and
generic ones around them; draw() spreads lengths, page sizes, head counts, head dims
and types.

Layouts: caches [pages, page, kv heads, d], scales [pages, page, kv heads] in e8m0,
rows of a ragged batch back to back (sequence b: rows qo_indptr[b] .. qo_indptr[b + 1],
which are the last of its kv_len[b] tokens), page table and lengths int32 as for the
paged decode.  tree_mask[row, j]: whether a row sees new token j of its sequence;
tokens before the new ones are always seen.
"""
import math

import numpy as np
import torch

own = False  # True: run() calls this package's operators; False: their plain forms

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
LARGEST = 448.0  # of e4m3: 0.875 * 2^9
LEAST = -126  # the smallest scale's exponent
THETA = 500000.0
EPS = 1e-6
DEVICE = "cuda"


def listed():
    return [
        # one token of one conversation: the smallest call, latency only
        {"name": "append_step_b1", "op": "append", "seqs": 1, "new": 1, "kv": 4096, "hq": 32, "hkv": 8, "d": 128,
         "page": 64, "norm": False, "tree": False, "dtype": "bf16"},
        # a batch with a tree of up to 32 drafted tokens each, q / k normalised per head
        {"name": "append_trees_b32", "op": "append", "seqs": 32, "new": 32, "kv": 2048, "hq": 32, "hkv": 8, "d": 128,
         "page": 16, "norm": True, "tree": True, "dtype": "f16"},
        # a batch of prompts of up to 2048 tokens, the largest append
        {"name": "append_prompts_b8", "op": "append", "seqs": 8, "new": 2048, "kv": 2048, "hq": 32, "hkv": 8, "d": 128,
         "page": 64, "norm": False, "tree": False, "dtype": "bf16"},
        # the next token of one long conversation
        {"name": "attend_step_b1", "op": "attend", "seqs": 1, "new": 1, "kv": 32768, "hq": 32, "hkv": 8, "d": 128,
         "page": 64, "tree": False, "cache": "e4m3", "dtype": "bf16"},
        # a decode batch, sequences of different lengths
        {"name": "attend_step_b32", "op": "attend", "seqs": 32, "new": 1, "kv": 8192, "hq": 32, "hkv": 8, "d": 128,
         "page": 64, "tree": False, "cache": "e4m3", "dtype": "bf16"},
        # small trees of a batch, 16-token pages, 8 query heads a kv head of 64, an odd length
        {"name": "attend_trees_b16", "op": "attend", "seqs": 16, "new": 15, "kv": 4093, "hq": 64, "hkv": 8, "d": 64,
         "page": 16, "tree": True, "cache": "e4m3", "dtype": "f16"},
        # trees of up to 64 tokens over a cache in 16 bits
        {"name": "attend_trees_16bit_b8", "op": "attend", "seqs": 8, "new": 64, "kv": 8192, "hq": 32, "hkv": 8, "d": 128,
         "page": 64, "tree": True, "cache": "16", "dtype": "bf16"},
        # a chunk of a long prompt after 14 K tokens, the most products
        {"name": "attend_chunk_2048", "op": "attend", "seqs": 1, "new": 2048, "kv": 16000, "hq": 32, "hkv": 8, "d": 128,
         "page": 64, "tree": False, "cache": "e4m3", "dtype": "bf16"},
        # one short prompt read back
        {"name": "read_b1", "op": "read", "seqs": 1, "kv": 500, "hkv": 8, "d": 128, "page": 64, "dtype": "f16"},
        # a batch of long prefixes read back
        {"name": "read_b8", "op": "read", "seqs": 8, "kv": 16384, "hkv": 8, "d": 128, "page": 64, "dtype": "bf16"},
        # the accepted path of one tree, a cache in 16 bits with its page bounds
        {"name": "keep_b1", "op": "keep", "seqs": 1, "new": 16, "kv": 200, "depth": 5, "hkv": 8, "d": 128, "page": 64,
         "cache": "16", "dtype": "bf16"},
        # the accepted paths of a batch, 8 bits
        {"name": "keep_b64", "op": "keep", "seqs": 64, "new": 32, "kv": 300, "depth": 8, "hkv": 8, "d": 128, "page": 16,
         "cache": "e4m3", "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "read", "keep"])
    hkv, group, d = rng.choice([(1, 8, 128), (2, 4, 128), (2, 7, 64), (2, 7, 128), (4, 1, 64), (4, 1, 128), (4, 5, 128),
                                (4, 16, 128), (8, 1, 64), (8, 2, 64), (8, 4, 128), (8, 8, 64), (8, 8, 128)])
    case = {"op": op, "hkv": hkv, "d": d, "page": rng.choice([16, 32, 64, 128]), "dtype": rng.choice(["f16", "bf16"])}
    if op == "read":
        seqs = _log(rng, 1, 64)
        return {**case, "seqs": seqs, "kv": _log(rng, 16, 8 * 16384 * 1024 // (seqs * hkv * d))}
    if op == "keep":
        new = _log(rng, 2, 64)
        return {**case, "seqs": _log(rng, 1, 64), "new": new, "kv": new + _log(rng, 1, 300), "depth": _log(rng, 1, min(new, 12)),
                "cache": rng.choice(["e4m3", "16"])}
    case["hq"] = hq = hkv * group
    if op == "append":
        seqs = _log(rng, 1, 64)
        most = 12288 * 48 * 128 // ((hq + 2 * hkv) * d * seqs)
        tree = rng.random() < 0.4
        new = 1 if not tree and rng.random() < 0.4 else _log(rng, 2, max(2, min(64 if tree else 2048, most)))
        return {**case, "seqs": seqs, "new": new, "kv": new + _log(rng, 1, 2048), "norm": rng.random() < 0.5, "tree": tree}
    case["cache"] = rng.choice(["e4m3", "e4m3", "16"])
    kind = rng.choice(["step", "tree", "chunk"])
    seqs = _log(rng, 1, {"step": 64, "tree": 32, "chunk": 4}[kind])
    cells = 32 * 8192 * 1024 // (seqs * hkv * d)  # of a head's cache, over the batch
    products = 2048 * 16000 * 32 * 128 // (seqs * hq * d)  # new rows x tokens
    new = {"step": 1, "tree": _log(rng, 2, 128), "chunk": _log(rng, 64, 2048)}[kind]
    kv = new + _log(rng, 1, max(1, min(131072, cells // 2, products // new) - new))
    return {**case, "seqs": seqs, "new": new, "kv": kv, "tree": kind == "tree"}


# ------------------------------------------------------------------ inputs
def _normal(gen, shape, std, dtype):
    return torch.empty(shape, dtype=dtype, device=DEVICE).normal_(0.0, std, generator=gen)


def _lengths(case):
    """Lengths and new rows of a batch in service: the first sequence has kv tokens
    and the most new rows, the others half to all of that. The case alone decides."""
    new = case.get("new", 1)
    rng = np.random.default_rng([case["seqs"], new, case["kv"]])
    news = rng.integers((new + 1) // 2, new + 1, size=case["seqs"])
    lens = rng.integers((case["kv"] + 1) // 2, case["kv"] + 1, size=case["seqs"])
    news[0], lens[0] = new, case["kv"]
    return np.maximum(lens, news), news


def _dev(a, dtype=np.int32):
    return torch.from_numpy(np.asarray(a, dtype=dtype)).to(DEVICE)


def _batch(case, seed):
    """Lengths, new rows and a shuffled page table."""
    lens, news = _lengths(case)
    npg = -(-lens // case["page"])
    pool = int(npg.sum()) + 2
    return {"lens": lens, "news": news, "pool": pool, "kv_len": _dev(lens),
            "kv_indptr": _dev(np.concatenate([[0], np.cumsum(npg)])),
            "kv_indices": _dev(np.random.default_rng(seed).permutation(pool)[: int(npg.sum())]),
            "qo_indptr": _dev(np.concatenate([[0], np.cumsum(news)])) if case.get("new", 1) > 1 else None}


def _trees(news, seed):
    """Parents (-1: the root), depths and masks of a tree for each sequence: a drafted
    token follows one of the few before it."""
    rng = np.random.default_rng([seed, 7])
    parents, depths, mask, row = [], np.zeros(int(news.sum()), dtype=np.int64), np.zeros((int(news.sum()), int(news.max())), dtype=bool), 0
    for n in news:
        up = np.maximum(np.arange(n) - rng.integers(1, 7, size=n), 0)
        up[0] = -1
        for i in range(n):
            if i:
                depths[row + i] = depths[row + up[i]] + 1
                mask[row + i] = mask[row + up[i]]
            mask[row + i, i] = True
        parents.append(up)
        row += n
    return parents, depths, mask


def _paths(parents, depth, seed):
    """From the root to one node of each tree, at most `depth` tokens, -1 behind them."""
    rng = np.random.default_rng([seed, 8])
    out = np.full((len(parents), depth), -1, dtype=np.int32)
    for b, up in enumerate(parents):
        node, path = int(rng.integers(0, len(up))), []
        while node >= 0:
            path.append(node)
            node = int(up[node])
        path = path[::-1][:depth]
        out[b, :len(path)] = path
    return out


def _codes(gen, shape):
    """Codes of a cache in 8 bits, as tokens of normal channels have them: the largest near 448."""
    return _normal(gen, shape, 150.0, torch.float16).clamp_(-LARGEST, LARGEST).to(E4M3)


def _scales(gen, shape):
    return torch.randint(118, 121, shape[:3], dtype=torch.uint8, device=DEVICE, generator=gen).view(E8M0)


def _tables(case):
    """cos / sin rows of the rotate-half rotation, [positions, d] in 32 bits."""
    d = case["d"]
    inv = THETA ** (-np.arange(0, d, 2, dtype=np.float64) / d)
    ang = np.outer(np.arange(case["kv"], dtype=np.float64), np.concatenate([inv, inv]))
    return tuple(torch.from_numpy(f(ang).astype(np.float32)).to(DEVICE) for f in (np.cos, np.sin))


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    s = {"case": case, **_batch(case, seed)}
    rows, news, first = int(s["news"].sum()), s["news"], s["lens"] - s["news"]
    shape = (s["pool"], case["page"], case["hkv"], case["d"])
    if case.get("cache") == "16":
        s["k_cache"], s["v_cache"] = _normal(gen, shape, 1.0, dt), _normal(gen, shape, 1.0, dt)
        s["k_scale"] = s["v_scale"] = None
    else:
        s["k_cache"], s["v_cache"] = _codes(gen, shape), _codes(gen, shape)
        s["k_scale"], s["v_scale"] = _scales(gen, shape), _scales(gen, shape)
    parents = depths = mask = None
    if case.get("tree") or case["op"] == "keep":
        parents, depths, mask = _trees(news, seed)
    if case["op"] == "append":
        # k and v are slices of one projection's output, as programs have them
        qkv = _normal(gen, (rows, case["hq"] + 2 * case["hkv"], case["d"]), 1.0, dt)
        s["q"], s["k"], s["v"] = qkv.split([case["hq"], case["hkv"], case["hkv"]], 1)
        s["cos"], s["sin"] = _tables(case)
        s["q_norm"] = s["k_norm"] = None
        if case["norm"]:
            s["q_norm"], s["k_norm"] = (1 + _normal(gen, (2, case["d"]), 0.1, dt)).unbind(0)
        # a drafted token's position is its depth in the tree
        s["positions"] = _dev(np.repeat(first, news) + depths) if case["tree"] else None
    elif case["op"] == "attend":
        s["q"] = _normal(gen, (rows, case["hq"], case["d"]), 1.0, dt)
        s["tree_mask"] = _dev(mask, dtype=bool) if case["tree"] else None
    elif case["op"] == "read":
        s["out_indptr"] = _dev(np.concatenate([[0], np.cumsum(s["lens"])]))
        s["total"] = int(s["lens"].sum())
    else:
        s["path"] = _dev(_paths(parents, case["depth"], seed))
        s["bounds"] = None
        if case["cache"] == "16":
            s["bounds"] = torch.stack([s["k_cache"].amin(1), s["k_cache"].amax(1)], 2) * 0.5  # (of some tokens)
    return s


# ------------------------------------------------------------------ plain forms
def _slot(s, seq, pos):
    """Page and slot of a sequence's token."""
    page = s["case"]["page"]
    return s["kv_indices"].long()[s["kv_indptr"].long()[seq] + pos // page], pos % page


def _row_tokens(ptr, lens, rows):
    """Sequence of each row and the token that it is, where row i of n is token len - n + i."""
    if ptr is None:
        return torch.arange(lens.numel(), device=DEVICE), lens.long() - 1
    ptr, row = ptr.long(), torch.arange(rows, device=DEVICE)
    seq = torch.searchsorted(ptr[1:].contiguous(), row, right=True)
    return seq, lens.long()[seq] - (ptr[seq + 1] - row)


def _rotate(x, weight, cos, sin):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    half = x.shape[-1] // 2
    return x * cos[:, None] + torch.cat([-x[..., half:], x[..., :half]], -1) * sin[:, None]


def _quantise(x):
    """Codes, and the smallest power of two that leaves none beyond the largest."""
    m, e = torch.frexp(x.abs().amax(-1))  # m * 2^e, m in [0.5, 1) or 0
    e = torch.where(m == 0, LEAST, (e - 9 + (m > 0.875)).clamp(min=LEAST))
    return (x * _power((127 - e).to(torch.uint8))[..., None]).to(E4M3), (e + 127).to(torch.uint8)


def _power(scale):
    """The power of two that a scale in e8m0 (or its bits) stands for."""
    return (scale.view(torch.uint8).int() << 23).view(torch.float32)


def _append(s):
    seq, pos = _row_tokens(s["qo_indptr"], s["kv_len"], s["q"].shape[0])
    at = pos if s["positions"] is None else s["positions"].long()
    cos, sin = s["cos"][at], s["sin"][at]
    k, ks = _quantise(_rotate(s["k"], s["k_norm"], cos, sin))
    v, vs = _quantise(s["v"].float())
    ids, slot = _slot(s, seq, pos)
    s["k_cache"].view(torch.uint8)[ids, slot] = k.view(torch.uint8)
    s["v_cache"].view(torch.uint8)[ids, slot] = v.view(torch.uint8)
    s["k_scale"].view(torch.uint8)[ids, slot], s["v_scale"].view(torch.uint8)[ids, slot] = ks, vs
    return _rotate(s["q"], s["q_norm"], cos, sin).to(s["q"].dtype), s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]


def _padded(s, name):
    """A cache's tokens by sequence, in 32 bits: [sequences, kv heads, most tokens, d]."""
    ptr, ids = s["kv_indptr"].long(), s["kv_indices"].long()
    most = int(-(-s["lens"].max() // s["case"]["page"]))
    ids = ids[(ptr[:-1, None] + torch.arange(most, device=DEVICE)).clamp(max=ids.numel() - 1)]
    x = s[name + "_cache"]
    if x.dtype == E4M3:
        x = x.view(torch.uint8)[ids].view(E4M3).float() * _power(s[name + "_scale"])[ids][..., None]
    else:
        x = x[ids].float()
    return x.flatten(1, 2).transpose(1, 2).contiguous()


def _attend(s):
    c, q, lens = s["case"], s["q"], s["kv_len"].long()
    B, hkv, d = c["seqs"], c["hkv"], c["d"]
    ptr = torch.arange(B + 1, device=DEVICE) if s["qo_indptr"] is None else s["qo_indptr"].long()
    news, most = ptr[1:] - ptr[:-1], int(s["news"].max())
    k, v = _padded(s, "k"), _padded(s, "v")
    i = torch.arange(most, device=DEVICE)
    rows = (ptr[:-1, None] + i).clamp(max=q.shape[0] - 1)
    qp = q[rows].float().unflatten(2, (hkv, -1)).permute(0, 2, 3, 1, 4).flatten(2, 3).contiguous()  # [B, hkv, group x rows, d]
    token = torch.arange(k.shape[2], device=DEVICE)
    j = token - (lens - news)[:, None]  # new token's number, negative in front
    if s["tree_mask"] is None:
        seen = j[:, None] <= i[:, None]
    else:
        width = s["tree_mask"].shape[1]
        seen = s["tree_mask"][rows].gather(2, j.clamp(0, width - 1)[:, None].expand(B, most, -1)) | (j < 0)[:, None]
    seen &= (token < lens[:, None])[:, None]
    a = (qp @ k.transpose(2, 3).contiguous()).unflatten(2, (-1, most)) / math.sqrt(d)  # [B, hkv, group, rows, tokens]
    a = a.masked_fill_(~seen[:, None, None], -math.inf)
    a = torch.exp(a - a.amax(-1, keepdim=True))
    out = ((a / a.sum(-1, keepdim=True)).flatten(2, 3) @ v).unflatten(2, (-1, most)).permute(0, 3, 1, 2, 4).flatten(2, 3)
    return out[i < news[:, None]].to(q.dtype)


def _read(s):
    row = torch.arange(s["total"], device=DEVICE)
    seq = torch.searchsorted(s["out_indptr"][1:].long(), row, right=True)
    ids, slot = _slot(s, seq, row - s["out_indptr"].long()[seq])
    dt = DTYPES[s["case"]["dtype"]]
    return tuple((s[n + "_cache"].view(torch.uint8)[ids, slot].view(E4M3).float() * _power(s[n + "_scale"])[ids, slot][..., None]).to(dt)
                 for n in ("k", "v"))


def _keep(s):
    path, lens = s["path"].long(), s["kv_len"].long()
    first = lens - (s["qo_indptr"][1:] - s["qo_indptr"][:-1]).long()
    seq, to = (path >= 0).nonzero(as_tuple=True)
    src, dst = _slot(s, seq, first[seq] + path[seq, to]), _slot(s, seq, first[seq] + to)
    for n in ("k_cache", "v_cache", "k_scale", "v_scale"):
        if s[n] is not None:
            x = s[n].view(torch.uint8) if s[n].itemsize == 1 else s[n]
            x[dst] = x[src]
    if s["bounds"] is not None:
        k = s["k_cache"][dst]
        at = dst[0][:, None, None].expand(k.shape)
        lo, hi = s["bounds"].float().unbind(2)
        s["bounds"].copy_(torch.stack([lo.scatter_reduce(0, at, k.float(), "amin"), hi.scatter_reduce(0, at, k.float(), "amax")], 2))
    return (first + (path >= 0).sum(1)).int()


def run(s):
    c = s["case"]
    op = c["op"]
    table = (s["kv_indptr"], s["kv_indices"], s["kv_len"])
    if op == "append":
        if not own:
            return _append(s)
        from yirage_amd import fused

        q = fused.append_kv_paged_fp8(s["k"], s["v"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], *table, q=s["q"],
                                      cos=s["cos"], sin=s["sin"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS,
                                      qo_indptr=s["qo_indptr"], positions=s["positions"])
        return q, s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]
    if op == "attend":
        if not own:
            return _attend(s)
        from yirage_amd import fused

        return fused.gqa_tree_paged(s["q"], s["k_cache"], s["v_cache"], *table, tree_mask=s["tree_mask"], qo_indptr=s["qo_indptr"],
                                    k_scale=s["k_scale"], v_scale=s["v_scale"], max_kv_len=c["kv"])
    if op == "read":
        if not own:
            return _read(s)
        from yirage_amd import fused

        return fused.read_kv_paged_fp8(s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], *table, s["out_indptr"], s["total"],
                                       dtype=DTYPES[c["dtype"]])
    if not own:
        lens = _keep(s)
    else:
        from yirage_amd import fused

        lens = fused.keep_kv_paged(s["k_cache"], s["v_cache"], *table, s["path"], qo_indptr=s["qo_indptr"], k_scale=s["k_scale"],
                                   v_scale=s["v_scale"], page_bounds=s["bounds"])
    return lens, s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["bounds"]


def work(case):
    hkv, d = case["hkv"], case["d"]
    lens, news = _lengths(case)
    size = 2 * d if case.get("cache") == "16" else d + 1  # of a token's head in the cache, its scale included
    if case["op"] == "read":
        return {"bytes": int(lens.sum()) * 2 * hkv * (size + 2 * d), "flops": 2 * int(lens.sum()) * hkv * d}
    if case["op"] == "keep":
        # the longest paths that the case allows, read and written
        moved = int(np.minimum(news, case["depth"]).sum())
        return {"bytes": moved * 4 * hkv * size + 12 * case["seqs"], "flops": 0}
    rows, hq = int(news.sum()), case["hq"]
    if case["op"] == "append":
        move = rows * (4 * hq * d + 2 * hkv * (2 * d + size)) + 8 * int(news.max()) * d
        return {"bytes": move, "flops": rows * (3 * hq + 7 * hkv) * d}
    seen = news * (lens - news) + news * (news + 1) // 2
    return {"bytes": 2 * int(lens.sum()) * hkv * size + 4 * rows * hq * d, "flops": 4 * int(seen.sum()) * hq * d}


# ------------------------------------------------------------------ 64 bits
def _exact_rotate(x, weight, cos, sin):
    """Pair (i, i + d / 2) turned as a complex number, the two halves with their own angle rows."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + EPS) * weight.double()
    a, b = x.chunk(2, -1)
    (ca, cb), (sa, sb) = (t.double()[:, None].chunk(2, -1) for t in (cos, sin))
    return torch.cat([a * ca - b * sa, b * cb + a * sb], -1)


def _values(s, name, ids):
    """Values of a sequence's tokens, [tokens, kv heads, d]."""
    x = s[name + "_cache"]
    if x.dtype != E4M3:
        return x[ids].double().flatten(0, 1)
    codes = x.view(torch.uint8)[ids].view(E4M3).double()
    return (codes * s[name + "_scale"].double()[ids][..., None]).flatten(0, 1)


def exact(case, seed):
    s = prepare(case, seed)
    hkv, d, page = case["hkv"], case["d"], case["page"]
    lens, news = s["lens"].tolist(), s["news"].tolist()
    starts = np.concatenate([[0], np.cumsum(news)]).tolist()
    tables = np.concatenate([[0], np.cumsum(-(-s["lens"] // page))]).tolist()
    pages = [s["kv_indices"][a:b].long() for a, b in zip(tables, tables[1:])]
    if case["op"] == "append":
        # the codes before their rounding to 8 bits
        q = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
        caches = [s[n].float().double() for n in ("k_cache", "v_cache", "k_scale", "v_scale")]
        for b, ids in enumerate(pages):
            r, token = slice(starts[b], starts[b + 1]), torch.arange(lens[b] - news[b], lens[b], device=DEVICE)
            at = token if s["positions"] is None else s["positions"][r].long()
            q[r] = _exact_rotate(s["q"][r], s["q_norm"], s["cos"][at], s["sin"][at])
            new = (_exact_rotate(s["k"][r], s["k_norm"], s["cos"][at], s["sin"][at]), s["v"][r].double())
            for x, cache, scale in zip(new, caches[:2], caches[2:]):
                step = torch.exp2(torch.ceil(torch.log2(torch.maximum(x.amax(-1), -x.amin(-1)) / LARGEST)).clamp(min=LEAST))
                cache[ids[token // page], token % page] = x / step[..., None]
                scale[ids[token // page], token % page] = step
        return q, *caches
    if case["op"] == "read":
        return tuple(torch.cat([_values(s, n, ids)[:m] for ids, m in zip(pages, lens)]) for n in ("k", "v"))
    if case["op"] == "keep":
        out = [s[n].float().double() if s[n] is not None else None for n in ("k_cache", "v_cache", "k_scale", "v_scale", "bounds")]
        kept = []
        for b, (ids, path) in enumerate(zip(pages, s["path"].tolist())):
            base = lens[b] - news[b]
            path = [p for p in path if p >= 0]
            for to, frm in enumerate(path):
                (u, i), (w, j) = divmod(base + frm, page), divmod(base + to, page)
                for x in out[:4]:
                    if x is not None:
                        x[ids[w], j] = x[ids[u], i]
                if out[4] is not None:
                    key = out[0][ids[w], j]
                    out[4][ids[w]] = torch.stack([torch.minimum(out[4][ids[w], :, 0], key), torch.maximum(out[4][ids[w], :, 1], key)], 1)
            kept.append(base + len(path))
        return (_dev(kept), *out)
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE).unflatten(1, (hkv, -1))
    for b, ids in enumerate(pages):
        n, base = news[b], lens[b] - news[b]
        k, v = (_values(s, x, ids)[:lens[b]].transpose(0, 1).contiguous() for x in ("k", "v"))
        for r in range(0, n, 64):
            m = min(64, n - r)
            at = slice(starts[b] + r, starts[b] + r + m)
            hidden = torch.zeros((m, lens[b]), dtype=torch.bool, device=DEVICE)
            if s["tree_mask"] is None:
                hidden[:, base:] = torch.ones((n, n), dtype=torch.bool, device=DEVICE).triu(1)[r:r + m]
            else:
                hidden[:, base:] = ~s["tree_mask"][at, :n]
            q = s["q"][at].double().unflatten(1, (hkv, -1)).permute(1, 2, 0, 3)
            a = (q.flatten(1, 2) @ k.transpose(1, 2).contiguous() / math.sqrt(d)).unflatten(1, (-1, m))
            p = torch.softmax(a.masked_fill_(hidden, -math.inf), -1)
            out[at] = (p.flatten(1, 2) @ v).unflatten(1, (-1, m)).permute(2, 0, 1, 3)
    return out.flatten(1, 2)

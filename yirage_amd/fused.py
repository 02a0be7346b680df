"""Torch-tensor front end of the fused HIP operators.

PyTorch supplies device memory and the current stream only; every operator
runs a hand-written gfx950 kernel through the C ABI.  Outputs are allocated
here (the reference allocates them in Python from the generated program's
output directives, python/yirage/kernel.py:393-402), workspaces come from a
per-device cache that is zero-filled once at allocation.
"""
from __future__ import annotations

import ctypes
import struct
from typing import NamedTuple

import torch

from . import _lib
from ._lib import check, lib

_TORCH_DT = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}
_ws_cache: dict = {}


def dtype_code(t: torch.dtype) -> int:
    try:
        return _TORCH_DT[t]
    except KeyError:
        raise _lib.YirageHipError(f"hip backend: unsupported dtype {t} (float16/bfloat16 only)")


def _ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream(device) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def workspace(nbytes: int, device) -> torch.Tensor | None:
    """Zero-filled scratch shared by the fused operators on one device/stream.
    The kernels return it to all-zero tickets when they finish."""
    if nbytes == 0:
        return None
    key = (torch.device(device).index, torch.cuda.current_stream(device).cuda_stream)
    ws = _ws_cache.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = torch.zeros(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
        _ws_cache[key] = ws
    return ws


def _check_cuda(*ts):
    for t in ts:
        if t is not None:
            if not t.is_cuda:
                raise _lib.YirageHipError("hip backend: tensors must live on the GPU")
            if not t.is_contiguous():
                raise _lib.YirageHipError("hip backend: tensors must be contiguous (row-major)")


def _same_dtype(x, *others):
    """Every 16-bit operand must share x's dtype (the kernels read them all
    as x's element type)."""
    for t in others:
        if t is not None and t.dtype != x.dtype:
            raise _lib.YirageHipError(f"hip backend: operand dtype {t.dtype} differs from x's {x.dtype}")


def _w_layout_and_n(w: torch.Tensor, k: int, layout: int | None):
    if layout is None:
        layout = _lib.W_KN
    if layout == _lib.W_KN:
        if w.shape[0] != k:
            raise _lib.YirageHipError(f"W shape {tuple(w.shape)} does not match K={k} (KN layout)")
        return layout, w.shape[1]
    if w.shape[1] != k:
        raise _lib.YirageHipError(f"W shape {tuple(w.shape)} does not match K={k} (NK layout)")
    return layout, w.shape[0]


def rmsnorm_linear(x, gamma, w, eps: float = 1e-6, w_layout: int | None = None, out=None):
    """out = (x * rsqrt(mean(x^2) + eps) * gamma) @ W  (fp32 accumulate)."""
    _check_cuda(x, gamma, w)
    _same_dtype(x, gamma, w)
    B, K = x.shape
    layout, N = _w_layout_and_n(w, K, w_layout)
    dt = dtype_code(x.dtype)
    if out is None:
        out = torch.empty((B, N), dtype=x.dtype, device=x.device)
    nb = lib().yr_hip_rmsnorm_linear_workspace(B, K, N, dt, layout)
    ws = workspace(nb, x.device)
    check(lib().yr_hip_rmsnorm_linear(_ptr(x), _ptr(gamma), _ptr(w), _ptr(out), B, K, N, dt, layout, eps,
                                      _ptr(ws), nb, _stream(x.device)), "rmsnorm_linear")
    return out


def gated_mlp(x, w1, w3, w_layout: int | None = None, out=None):
    """out = silu(x @ W1) * (x @ W3)."""
    _check_cuda(x, w1, w3)
    _same_dtype(x, w1, w3)
    B, K = x.shape
    layout, N = _w_layout_and_n(w1, K, w_layout)
    if w3.shape != w1.shape:
        raise _lib.YirageHipError("W1 and W3 shapes differ")
    dt = dtype_code(x.dtype)
    if out is None:
        out = torch.empty((B, N), dtype=x.dtype, device=x.device)
    nb = lib().yr_hip_gated_mlp_workspace(B, K, N, dt, layout)
    ws = workspace(nb, x.device)
    check(lib().yr_hip_gated_mlp(_ptr(x), _ptr(w1), _ptr(w3), _ptr(out), B, K, N, dt, layout,
                                 _ptr(ws), nb, _stream(x.device)), "gated_mlp")
    return out


def linear(x, w, residual=None, w_layout: int | None = _lib.W_NK, out=None):
    """out = x @ W^T (NK layout, torch Linear.weight) or x @ W (KN) (+ residual)."""
    _check_cuda(x, w, residual)
    _same_dtype(x, w, residual)
    B, K = x.shape
    layout, N = _w_layout_and_n(w, K, w_layout)
    dt = dtype_code(x.dtype)
    if out is None:
        out = torch.empty((B, N), dtype=x.dtype, device=x.device)
    nb = lib().yr_hip_linear_workspace(B, K, N, dt, layout)
    ws = workspace(nb, x.device)
    check(lib().yr_hip_linear(_ptr(x), _ptr(w), _ptr(residual), _ptr(out), B, K, N, dt, layout,
                              _ptr(ws), nb, _stream(x.device)), "linear")
    return out


def gqa_decode_paged(q, k_cache, v_cache, kv_indptr, kv_indices, kv_len, max_kv_len: int | None = None, out=None):
    """Paged GQA decode: q[B,Hq,D], caches [P,page,Hkv,D], int32 page table."""
    _check_cuda(q, k_cache, v_cache, kv_indptr, kv_indices, kv_len)
    _same_dtype(q, k_cache, v_cache)
    B, Hq, D = q.shape
    P, page, Hkv, D2 = k_cache.shape
    if D2 != D or v_cache.shape != k_cache.shape:
        raise _lib.YirageHipError("cache shape mismatch")
    for t in (kv_indptr, kv_indices, kv_len):
        if t.dtype != torch.int32:
            raise _lib.YirageHipError("page table tensors must be int32")
    if max_kv_len is None:
        max_kv_len = int(kv_len.max().item())
    dt = dtype_code(q.dtype)
    if out is None:
        out = torch.empty_like(q)
    nb = lib().yr_hip_gqa_decode_workspace(B, Hq, Hkv, D, max_kv_len, page)
    ws = workspace(nb, q.device)
    check(lib().yr_hip_gqa_decode_paged(_ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(kv_indptr), _ptr(kv_indices),
                                        _ptr(kv_len), _ptr(out), B, Hq, Hkv, D, page, max_kv_len, dt,
                                        _ptr(ws), nb, _stream(q.device)), "gqa_decode_paged")
    return out


def gqa_prefill(q, k, v, causal: bool = True, out=None):
    """Prefill attention q[B,S,Hq,D], k/v[B,S,Hkv,D]."""
    _check_cuda(q, k, v)
    _same_dtype(q, k, v)
    B, S, Hq, D = q.shape
    Hkv = k.shape[2]
    dt = dtype_code(q.dtype)
    if out is None:
        out = torch.empty_like(q)
    check(lib().yr_hip_gqa_prefill(_ptr(q), _ptr(k), _ptr(v), _ptr(out), B, S, Hq, Hkv, D, int(causal), dt,
                                   _stream(q.device)), "gqa_prefill")
    return out


def argmax(x, n_valid: int | None = None, out=None):
    """Row-wise argmax (lowest index on ties) of a 2-D f16/bf16 tensor -> int64."""
    _check_cuda(x)
    rows, n = x.shape
    if out is None:
        out = torch.empty(rows, dtype=torch.int64, device=x.device)
    check(lib().yr_hip_argmax(_ptr(x), _ptr(out), rows, n, n if n_valid is None else n_valid,
                              dtype_code(x.dtype), _stream(x.device)), "argmax")
    return out


# ---------------------------------------------------------------- serving step around a paged cache
# Operators on a ragged batch: sequence b owns the rows qo_indptr[b] ..
# qo_indptr[b + 1) of the new tokens (qo_indptr None: one row each), the pages
# kv_indices[kv_indptr[b] .. kv_indptr[b + 1]) and kv_len[b] tokens, the new ones
# last.  Their kernels run on the tensors' device and its current stream.  A
# decode step's calls are as short as their host side, so the checks below read
# each property once.
_TICKET_BYTES = 65536  # what a workspace has zeroed at rest
_scratch_cache: dict = {}
_DTYPE_ALL = {**_TORCH_DT, torch.float32: _lib.DTYPE_F32}
_pack7 = struct.Struct("7q").pack  # seven int64 in memory, as a pointer argument takes them


def _fail(msg: str):
    raise _lib.YirageHipError(f"hip backend: {msg}")


def _one_device(*ts) -> int:
    """Index of the one GPU that the tensors (or None) live on."""
    index = ts[0].get_device()
    for t in ts:
        if t is not None and t.get_device() != index:
            _fail(f"tensors on different devices ({t.device}, {ts[0].device})")
    if index < 0:
        _fail("tensors must live on the GPU")
    return index


def _dense(*ts):
    for t in ts:
        if t is not None and not t.is_contiguous():
            _fail(f"caches, tables and inputs of shape {tuple(t.shape)} must be contiguous (row-major)")


def _launch(index: int, fn, what: str, *args):
    """fn(*args) with the tensors' device current."""
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args)
    else:
        with torch.cuda.device(index):
            rc = fn(*args)
    if rc != _lib.YR_OK:
        check(rc, what)


def _scratch(nbytes: int, device, stream: int):
    """Zero-filled scratch of one device and stream.  It is not workspace()'s: these calls ask
    for much more, and an entry that they replaced there could be one that a captured
    graph of the other operators has the address of.  A captured call owns its scratch: the
    graph's pool keeps it, tickets are cleared at every replay, and no two graphs meet in
    it.  The caller holds the tensor until its launch has returned: another thread's larger
    call on the same stream may replace the cache's entry at any time, and a block that
    nothing holds is the allocator's again."""
    if nbytes == 0:
        return None
    if torch.cuda.is_current_stream_capturing():
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
        ws[:_TICKET_BYTES].zero_()
        return ws
    key = (device.index, stream)
    ws = _scratch_cache.get(key)
    if ws is None or ws.numel() < nbytes:
        with torch.cuda.device(device):  # (allocated and cleared on its stream)
            ws = _scratch_cache[key] = torch.zeros(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
    return ws


def _at(t):
    return None if t is None else t.data_ptr()


def _page_table(rows, kv_indptr, kv_indices, kv_len, qo_indptr):
    """Checks of a ragged batch's tables -> batch size."""
    i32 = torch.int32
    if kv_indptr.dtype is not i32 or kv_indices.dtype is not i32 or kv_len.dtype is not i32:
        _fail("page table tensors must be int32")
    batch = kv_len.numel()
    if kv_indptr.numel() != batch + 1:
        _fail(f"kv_indptr must have {batch + 1} entries (kv_len has {batch})")
    if qo_indptr is None:
        if rows != batch:
            _fail(f"without qo_indptr every sequence has one row ({rows} rows, {batch} sequences)")
    elif qo_indptr.dtype is not i32 or qo_indptr.numel() != batch + 1:
        _fail(f"qo_indptr must be int32 with {batch + 1} entries (kv_len has {batch})")
    _dense(kv_indptr, kv_indices, kv_len, qo_indptr)
    return batch


def _output(out, shape, like):
    """A result of like's dtype, or the caller's."""
    if out is None:
        return like.new_empty(shape)
    if tuple(out.shape) != tuple(shape) or out.dtype is not like.dtype:
        _fail(f"out must be {tuple(shape)} {like.dtype}, got {tuple(out.shape)} {out.dtype}")
    _dense(out)
    return out


def append_kv_paged(k, v, k_cache, v_cache, kv_indptr, kv_indices, kv_len, q=None, cos=None, sin=None, q_norm=None,
                    k_norm=None, eps: float = 1e-6, qo_indptr=None, page_bounds=None, out=None):
    """Writes new tokens k, v [T, Hkv, D] into the paged caches [P, page, Hkv, D]; returns q as the
    attention reads it, [T, Hq, D] (None without q).

    kv_len counts the new tokens, so row i of a sequence's n rows has position kv_len - n + i.
    Keys and q are normalised per head (q_norm / k_norm [D]) and rotated (rotate-half, cos / sin
    [positions, D], fp32 or k's dtype), in fp32 with one rounding; a q row whose position lies
    outside the tables is NaN and its key is not written.  page_bounds [P, Hkv, 2, D] keeps each
    page's smallest and largest key per channel, NaN left out (what select_pages reads).  q is [T, Hq, D] or
    [T, Hkv, Hq / Hkv, D]; q, k and v may be slices of one projection (last dim contiguous, 16-byte
    aligned).  out may be q itself where that is contiguous.  D is 64 or 128."""
    dtype = k.dtype
    dt = dtype_code(dtype)
    for t in (v, q):
        if t is not None and t.dtype is not dtype:
            _fail(f"operand dtype {t.dtype} differs from k's {dtype}")
    for t in (k_cache, v_cache, page_bounds, q_norm, k_norm):
        if t is not None and (t.dtype is not dtype or not t.is_contiguous()):
            if t.dtype is not dtype:
                _fail(f"operand dtype {t.dtype} differs from k's {dtype}")
            _dense(t)
    kshape, cshape = k.shape, k_cache.shape
    if len(kshape) != 3 or v.shape != kshape or len(cshape) != 4 or v_cache.shape != cshape:
        _fail("k and v must be [T, Hkv, D], the caches [P, page, Hkv, D]")
    T, hkv, D = kshape
    P, page, h2, d2 = cshape
    if h2 != hkv or d2 != D:
        _fail(f"cache heads {(h2, d2)} differ from k's {(hkv, D)}")
    batch = _page_table(T, kv_indptr, kv_indices, kv_len, qo_indptr)
    if page_bounds is not None and page_bounds.shape != (P, hkv, 2, D):
        _fail(f"page_bounds must be {(P, hkv, 2, D)}")
    for w in (q_norm, k_norm):
        if w is not None and w.shape != (D,):
            _fail(f"norm weights must be [{D}]")
    tdt, npos = 0, 0
    if cos is not None or sin is not None:
        if cos is None or sin is None:
            _fail("cos and sin come together")
        tshape, ttype = cos.shape, cos.dtype
        if len(tshape) != 2 or tshape[1] != D or sin.shape != tshape or sin.dtype is not ttype:
            _fail(f"cos and sin must be [positions, {D}] of one dtype")
        if ttype is not dtype and ttype is not torch.float32:
            _fail(f"tables must be float32 or {dtype}, got {ttype}")
        _dense(cos, sin)
        tdt, npos = _DTYPE_ALL[ttype], tshape[0]
    hq, qs = 0, (0, 0, 0)
    ks, vs = k.stride(), v.stride()
    if q is not None:
        qs, qshape = q.stride(), q.shape
        if len(qshape) == 4:
            if qshape[0] != T or qshape[1] != hkv or qshape[3] != D:
                _fail(f"q must be [{T}, {hkv}, heads, {D}]")
            hq = hkv * qshape[2]
        else:
            if len(qshape) != 3 or qshape[0] != T or qshape[2] != D or qshape[1] % hkv:
                _fail(f"q must be [{T}, heads, {D}] with a multiple of {hkv} heads")
            hq = qshape[1]
            qs = (qs[0], qs[1] * (hq // hkv), qs[1], qs[2])
        if qs[3] != 1 and q.numel():
            _fail("the last dim of q must be contiguous")
    elif out is not None or q_norm is not None:
        _fail("out and q_norm need q")
    if (ks[2] != 1 or vs[2] != 1) and T:
        _fail("the last dim of k and v must be contiguous")
    if q is not None:
        out = q.new_empty((T, hq, D)) if out is None else _output(out, (T, hq, D), q)
    index = _one_device(k, v, k_cache, v_cache, kv_indptr, kv_indices, kv_len, q, cos, sin, q_norm, k_norm, qo_indptr,
                        page_bounds, out)
    if T == 0:
        return out
    _launch(index, lib().yr_hip_append_kv_paged, "append_kv_paged", None if q is None else q.data_ptr(), k.data_ptr(),
            v.data_ptr(), None if q is None else out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
            None if page_bounds is None else page_bounds.data_ptr(), None if cos is None else cos.data_ptr(),
            None if cos is None else sin.data_ptr(), tdt, npos, None if q_norm is None else q_norm.data_ptr(),
            None if k_norm is None else k_norm.data_ptr(), eps, None if qo_indptr is None else qo_indptr.data_ptr(),
            kv_indptr.data_ptr(), kv_indices.data_ptr(), kv_indices.numel(), kv_len.data_ptr(), T, batch, hq, hkv, D, page,
            P, _pack7(qs[0], qs[1], qs[2], ks[0], ks[1], vs[0], vs[1]), dt, torch._C._cuda_getCurrentRawStream(index))
    return out


def select_pages(q, page_bounds, kv_indptr, kv_indices, kv_len, page_size: int, top_pages: int, qo_indptr=None,
                 first_pages: int = 1, last_pages: int = 1, max_kv_len: int | None = None, out=None):
    """Pages that each row of q [T, Hq, D] attends to, per kv head: int32 [T, Hkv, top_pages], page
    numbers within the sequence, ascending, -1 behind.

    The first first_pages pages, the last last_pages (>= 1) visible ones, and the best of the others
    by an upper bound of their scores from page_bounds [P, Hkv, 2, D] (append_kv_paged keeps it),
    summed over the group's heads in 64 bits; ties take the lower page.  max_kv_len bounds kv_len
    (None: its maximum, read on the host)."""
    if page_bounds.dtype is not q.dtype:
        _fail(f"page_bounds' dtype {page_bounds.dtype} differs from q's {q.dtype}")
    dt = dtype_code(q.dtype)
    _dense(q, page_bounds)
    qshape, bshape = q.shape, page_bounds.shape
    if len(qshape) != 3 or len(bshape) != 4 or bshape[2] != 2 or bshape[3] != qshape[2]:
        _fail("q must be [T, Hq, D], page_bounds [P, Hkv, 2, D]")
    T, hq, D = qshape
    P, hkv, _, _ = bshape
    batch = _page_table(T, kv_indptr, kv_indices, kv_len, qo_indptr)
    if top_pages < 1:
        _fail("top_pages must be positive")
    if out is None:
        out = kv_len.new_empty((T, hkv, top_pages))  # (int32, q's device: checked here and below)
    elif tuple(out.shape) != (T, hkv, top_pages) or out.dtype is not torch.int32 or not out.is_contiguous():
        _fail(f"out must be contiguous int32 {(T, hkv, top_pages)}")
    index = _one_device(q, page_bounds, kv_indptr, kv_indices, kv_len, qo_indptr, out)
    if T == 0:
        return out
    if max_kv_len is None:
        max_kv_len = max(int(kv_len.max().item()), 1)
    stream = torch._C._cuda_getCurrentRawStream(index)
    nb = lib().yr_hip_select_pages_workspace(T, hkv, page_size, max_kv_len)
    ws = _scratch(nb, q.device, stream)
    _launch(index, lib().yr_hip_select_pages, "select_pages", q.data_ptr(), page_bounds.data_ptr(), _at(qo_indptr),
            kv_indptr.data_ptr(), kv_indices.data_ptr(), kv_indices.numel(), kv_len.data_ptr(), out.data_ptr(), T, batch,
            hq, hkv, D, page_size, P, max_kv_len, top_pages, first_pages, last_pages, dt,
            _at(ws), nb, stream)
    return out


def gqa_sparse_paged(q, k_cache, v_cache, kv_indptr, kv_indices, kv_len, pages, qo_indptr=None, out=None):
    """Paged GQA attention over selected pages: row t of q [T, Hq, D] attends to the tokens at or
    before its position in pages[t, h // (Hq / Hkv)] (int32 [T, Hkv, n], as select_pages gives them;
    any order, negative, invisible and repeated entries count for nothing).  A row without a token, or
    whose scores are all -inf, is 0.  Lists of up to 256 pages are the fast ones."""
    if k_cache.dtype is not q.dtype or v_cache.dtype is not q.dtype:
        _fail(f"cache dtypes {k_cache.dtype}, {v_cache.dtype} differ from q's {q.dtype}")
    dt = dtype_code(q.dtype)
    _dense(q, k_cache, v_cache, pages)
    qshape, cshape, pshape = q.shape, k_cache.shape, pages.shape
    if len(qshape) != 3 or len(cshape) != 4 or v_cache.shape != cshape or cshape[3] != qshape[2]:
        _fail("q must be [T, Hq, D], the caches [P, page, Hkv, D]")
    T, hq, D = qshape
    P, page, hkv, _ = cshape
    batch = _page_table(T, kv_indptr, kv_indices, kv_len, qo_indptr)
    if pages.dtype is not torch.int32 or len(pshape) != 3 or pshape[0] != T or pshape[1] != hkv:
        _fail(f"pages must be int32 [{T}, {hkv}, n]")
    top = pshape[2]
    out = torch.empty_like(q) if out is None else _output(out, qshape, q)
    index = _one_device(q, k_cache, v_cache, kv_indptr, kv_indices, kv_len, pages, qo_indptr, out)
    if T == 0:
        return out
    stream = torch._C._cuda_getCurrentRawStream(index)
    nb = lib().yr_hip_gqa_sparse_workspace(T, batch, qo_indptr is not None, hq, hkv, D, page, top)
    ws = _scratch(nb, q.device, stream)
    _launch(index, lib().yr_hip_gqa_sparse_paged, "gqa_sparse_paged", q.data_ptr(), k_cache.data_ptr(),
            v_cache.data_ptr(), _at(qo_indptr), kv_indptr.data_ptr(), kv_indices.data_ptr(), kv_indices.numel(),
            kv_len.data_ptr(), pages.data_ptr(), out.data_ptr(), T, batch, hq, hkv, D, page, P, top, dt,
            _at(ws), nb, stream)
    return out


class LogProbs(NamedTuple):
    logprob: torch.Tensor      # [rows] fp32, of the given tokens
    entropy: torch.Tensor      # [rows] fp32, nats
    top_logprob: torch.Tensor  # [rows, top_n] fp32, descending
    top_token: torch.Tensor    # [rows, top_n] int64, lowest first among equals


def token_logprobs(logits, tokens, top_n: int = 0, n_valid: int | None = None) -> LogProbs:
    """Log probabilities of tokens [rows] (int64) under softmax(logits[:, :n_valid]) (f16, bf16 or
    fp32, rows contiguous), the rows' entropy, and the top_n (<= 64) most likely tokens.  A token outside
    [0, n_valid) has NaN; NaN logits and rows of -inf alone give NaN numbers."""
    dt = _DTYPE_ALL.get(logits.dtype)
    if dt is None:
        _fail(f"unsupported logits dtype {logits.dtype}")
    if logits.dim() != 2 or (logits.stride(1) != 1 and logits.shape[1] > 1):
        _fail("logits must be [rows, n] with contiguous rows")
    rows, n = logits.shape
    if tokens.dtype is not torch.int64 or tokens.dim() != 1 or tokens.shape[0] != rows or not tokens.is_contiguous():
        _fail(f"tokens must be contiguous int64 [{rows}]")
    index = _one_device(logits, tokens)
    n_valid, top_n = n if n_valid is None else n_valid, int(top_n)
    # one allocation: the ids first (8 bytes each), then the three fp32 results
    cut = rows * max(top_n, 0)
    if logits.dtype is torch.float32:
        flat = logits.new_empty(3 * cut + 2 * rows)
    else:
        flat = torch.empty(3 * cut + 2 * rows, dtype=torch.float32, device=logits.device)
    ids, tops, lp, ent = flat.split_with_sizes((2 * cut, cut, rows, rows))
    if cut:
        res = LogProbs(lp, ent, tops.view(rows, top_n), ids.view(torch.int64).view(rows, top_n))
    else:
        res = LogProbs(lp, ent, tops.view(rows, 0), tokens.new_empty((rows, 0)))
    if rows == 0:
        return res
    stream = torch._C._cuda_getCurrentRawStream(index)
    nb = lib().yr_hip_token_logprobs_workspace(rows, n_valid, top_n, dt)
    ws = _scratch(nb, logits.device, stream)
    at = flat.data_ptr()
    _launch(index, lib().yr_hip_token_logprobs, "token_logprobs", logits.data_ptr(), tokens.data_ptr(), at + 12 * cut,
            at + 12 * cut + 4 * rows, at + 8 * cut, at, rows, n, n_valid, logits.stride(0) if rows > 1 else n, top_n, dt,
            _at(ws), nb, stream)
    return res


def synth_fill(t: torch.Tensor, seed: int, std: float, offset: int = 0) -> torch.Tensor:
    """Deterministic ~N(0, std) fill on the device (bit-identical to the CPU generator)."""
    _check_cuda(t)
    check(lib().yr_hip_synth_fill(_ptr(t), t.numel(), dtype_code(t.dtype), seed, offset, std,
                                  _stream(t.device)), "synth_fill")
    return t


def float_bits(x: float) -> int:
    return struct.unpack("<i", struct.pack("<f", x))[0]

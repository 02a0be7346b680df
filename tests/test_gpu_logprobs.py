"""token_logprobs against 64 bits: types, odd and strided rows, ties, masked
rows, NaN and infinities, nearly certain and even distributions."""
import math

import pytest
import torch

import yirage_amd.fused as F

pytestmark = pytest.mark.gpu

DTS = pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32], ids=["f16", "bf16", "f32"])


def _check(x, tokens, top, got, n_valid=None):
    """x on the CPU."""
    n = x.shape[1] if n_valid is None else n_valid
    lp, h, tlp, tid = (t.cpu() for t in got)
    for r in range(x.shape[0]):
        row = x[r, :n]
        order = torch.sort(torch.where(row.isnan(), -math.inf, row.double()), descending=True, stable=True).indices
        order = [i for i in order.tolist() if not math.isnan(row[i])][:top]
        assert tid[r].tolist() == order + [-1] * (top - len(order)), r
        assert (tlp[r, len(order):] == -math.inf).all()
        m = row[~row.isnan()].max().double().item() if (~row.isnan()).any() else math.nan
        t = int(tokens[r])
        if row.isnan().any() or not math.isfinite(m):
            assert lp[r].isnan() and h[r].isnan() and tlp[r, : len(order)].isnan().all()
            continue
        y = row.double() - m
        p = torch.softmax(y, 0)
        ls = torch.logsumexp(y, 0)
        py = torch.where(p > 0, p * y.clamp(min=-1e30), 0.0)
        ref_h = (ls - py.sum()).item()
        ty = py.abs().sum().item()
        ty2 = torch.where(p > 0, p * y.clamp(min=-1e30) ** 2, 0.0).sum().item()
        # exp of an fp32 argument: its rounding (y 2^-23 with the base change) and the function's, 2^-22
        rel = 2.0 ** -22 + 2.0 ** -23 * ty
        assert abs(h[r].item() - ref_h) <= rel + ty * (rel + 2.0 ** -22) + 2.0 ** -23 * ty2 + 2.0 ** -24 * ref_h, r

        def same(g, i):
            ref = (y[i] - ls).item()
            if ref == -math.inf:
                return g == -math.inf
            return abs(g - ref) <= rel + 2.0 ** -23 * (abs(y[i].item()) + abs(ref))  # the difference, the result

        if 0 <= t < n:
            assert same(lp[r].item(), t), (r, lp[r].item(), (y[t] - ls).item())
        else:
            assert lp[r].isnan()
        for j, i in enumerate(order):
            assert same(tlp[r, j].item(), i), (r, j)


@DTS
@pytest.mark.parametrize("rows,n,top", [(1, 1, 1), (1, 1, 0), (3, 7, 7), (5, 9, 3), (4, 63, 64 - 1), (2, 1000, 20), (9, 2051, 5),
                                        (3, 8193, 64), (2, 32771, 20), (1, 128256, 20), (33, 128251, 1), (300, 5003, 2),
                                        (600, 1024, 0)])
def test_rows(rows, n, top, dt):
    print("case", rows, n, top, dt, flush=True)
    gen = torch.Generator().manual_seed(rows + n)
    x = (2 * torch.randn((rows, n), generator=gen)).to(dt)  # many ties in 16 bits
    tok = torch.randint(0, n, (rows,), generator=gen)
    got = F.token_logprobs(x.cuda(), tok.cuda(), top_n=top)
    assert [tuple(t.shape) for t in got] == [(rows,), (rows,), (rows, top), (rows, top)]
    _check(x, tok, top, got)
    again = F.token_logprobs(x.cuda(), tok.cuda(), top_n=top)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@DTS
@pytest.mark.parametrize("n,n_valid,extra", [(130, 127, 3), (4097, 4000, 0), (20000, 19999, 13), (1000, 1, 24)])
def test_strided_rows_and_columns_never_looked_at(n, n_valid, extra, dt):
    gen = torch.Generator().manual_seed(n)
    full = torch.randn((6, n + extra), generator=gen).to(dt)
    full[:, n_valid:] = float("nan")
    x = full.cuda()[:, extra // 2: extra // 2 + n] if extra else full.cuda()
    host = full[:, extra // 2: extra // 2 + n] if extra else full
    if extra:
        full[:, extra // 2: extra // 2 + n_valid] = torch.randn((6, n_valid), generator=gen).to(dt)
        x = full.cuda()[:, extra // 2: extra // 2 + n]
    tok = torch.tensor([0, n_valid - 1, n_valid, n_valid // 2, -1, n_valid])  # the last ones name no token
    _check(host, tok, min(4, n_valid), F.token_logprobs(x, tok.cuda(), top_n=min(4, n_valid), n_valid=n_valid), n_valid)


@DTS
def test_masked_and_special_rows(dt):
    n = 5001
    gen = torch.Generator().manual_seed(7)
    x = torch.randn((14, n), generator=gen).to(dt)
    low = torch.finfo(dt).min
    x[0] = -math.inf                                   # nothing left: NaN
    x[1, torch.randperm(n, generator=gen)[:4990]] = -math.inf
    x[2] = -math.inf
    x[2, 4000] = 1.5                                   # certain
    x[3] = low                                         # even
    x[4, :4999] = low
    x[5, 17] = math.inf
    x[6, 4500] = math.nan
    x[7] = math.nan
    x[8] = 0.0                                         # even, all tied
    x[9, 3] = 60.0                                     # nearly certain
    x[10] = torch.arange(n).to(dt)                     # ascending: every value a new maximum (ties in 16 bits)
    x[11] = -torch.arange(n).to(dt)
    x[12, ::2] = -0.0
    x[12, 1::2] = 0.0                                  # zeros of both signs tie
    x[13] = torch.finfo(dt).max / 2
    x[13, 100] = low
    for tok in (4000, 17, 4999):
        t = torch.full((14,), tok)
        _check(x, t, 20, F.token_logprobs(x.cuda(), t.cuda(), top_n=20))


@DTS
def test_small_entropies_and_probabilities(dt):
    """One logit far above the rest: log s = log1p of little."""
    x = torch.zeros((5, 40000)).to(dt)
    for r, gap in enumerate([12, 16, 20, 24, 28]):
        x[r, 31111] = gap
    tok = torch.full((5,), 31111)
    got = F.token_logprobs(x.cuda(), tok.cuda(), top_n=2)
    _check(x, tok, 2, got)
    p1 = torch.log1p(39999 * torch.exp(-x[:, 31111].double()))
    assert ((got.logprob.cpu().double() + p1).abs() <= 2.0 ** -20 * p1 + 2.0 ** -24 * 40).all()


@DTS
def test_top_64_of_a_row_over_64_workgroups(dt):
    """Parts of a row that hold fewer numbers than are asked for."""
    gen = torch.Generator().manual_seed(5)
    x = torch.randn((3, 140001), generator=gen).to(dt)
    x[1, 70:] = -math.inf
    x[2, : 139990] = math.nan
    tok = torch.tensor([7, 69, 139999])
    for r in range(3):  # a row a call, so that each is split as far as it goes
        _check(x[r: r + 1], tok[r: r + 1], 64, F.token_logprobs(x[r: r + 1].cuda(), tok[r: r + 1].cuda(), top_n=64))

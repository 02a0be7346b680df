"""token_logprobs where logits are large: finite masks of every size in front of,
behind and between the allowed tokens, whole rows of them, and rows whose
numbers are large themselves.  A wave meets its part of a row in tiles of 2048
values, so masked stretches of several thousand make its first maximum a mask."""
import math

import pytest
import torch

import yirage_amd.fused as F

pytestmark = pytest.mark.gpu

DTS = pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32], ids=["f16", "bf16", "f32"])
WIDE = pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])


def _check(x, tok, top, got):
    """x and tok on the CPU; all rows at once. Rows with a NaN have NaN numbers."""
    lp, h, tlp, tid = (t.cpu() for t in got)
    nan = x.isnan()
    assert torch.equal(lp.isnan(), nan.any(1)) and torch.equal(h.isnan(), nan.any(1))
    order = torch.sort(torch.where(nan, -math.inf, x.double()), descending=True, stable=True, dim=1).indices[:, :top]
    assert torch.equal(tid, order)
    ok = ~nan.any(1)
    x, tok, order, lp, h, tlp = x[ok].double(), tok[ok, None], order[ok], lp[ok].double(), h[ok].double(), tlp[ok].double()
    y = x - x.amax(1, keepdim=True)
    ls = torch.logsumexp(y, 1, keepdim=True)
    p = torch.softmax(y, 1)
    py, py2 = (torch.where(p > 0, p * y ** k, 0.0) for k in (1, 2))
    ref, ty, ty2 = (ls - py.sum(1, keepdim=True))[:, 0], py.abs().sum(1), py2.sum(1)
    # exp of an fp32 argument: its rounding (y 2^-23 with the base change) and the function's, 2^-22
    rel = 2.0 ** -22 + 2.0 ** -23 * ty
    assert ((h - ref).abs() <= rel + ty * (rel + 2.0 ** -22) + 2.0 ** -23 * ty2 + 2.0 ** -24 * ref).all()
    for g, i in ((lp[:, None], tok), (tlp, order)):
        yi = y.gather(1, i)
        ref = yi - ls
        beyond = ref < -torch.finfo(torch.float32).max  # (the difference of two halves of fp32's range)
        assert (g[beyond] == -math.inf).all()
        tol = rel[:, None] + 2.0 ** -23 * (yi.abs() + ref.abs())  # the difference, the result
        assert ((g - ref).abs() <= tol)[~beyond].all()


def _run(x, tok, top, each=False):
    """All rows in a call, or (each) a row a call, split over workgroups as far as it goes."""
    print("rows", tuple(x.shape), x.dtype, "top", top, "each" if each else "", flush=True)
    if not each:
        _check(x, tok, top, F.token_logprobs(x.cuda(), tok.cuda(), top_n=top))
        return
    for r in range(x.shape[0]):
        _check(x[r: r + 1], tok[r: r + 1], top, F.token_logprobs(x[r: r + 1].cuda(), tok[r: r + 1].cuda(), top_n=top))


@DTS
@pytest.mark.parametrize("mask", [-1e4, -1e6, -1e9, -3e9, -1e10, -1e12, -1e20, -1e30, -1e38, -3.3e38])
def test_masks(mask, dt):
    """Allowed tokens nowhere, at the end, at the start, in the middle, one in 97."""
    if mask < torch.finfo(dt).min:
        mask = torch.finfo(dt).min
    print("case", mask, dt, flush=True)
    n = 40009
    gen = torch.Generator().manual_seed(11)
    base = (2 * torch.randn((6, n), generator=gen)).to(dt)
    x = torch.full((6, n), mask).to(dt)
    for r, allowed in enumerate([slice(0, 0), slice(n - 30, n), slice(0, 40), slice(20000, 20600), slice(0, n, 97), slice(9000, n)]):
        x[r, allowed] = base[r, allowed]
    tok = torch.tensor([5, n - 3, 7, 20300, 970, 30000])
    for top in (0, 5):
        _run(x, tok, top)
        _run(x, tok, top, each=True)


@WIDE
@pytest.mark.parametrize("size", [1e5, 1e6, 1.1e6, 3e7, 1e9, 1e10, 1e13, 1e25, 3e38])
def test_large_numbers(size, dt):
    """Even rows, a few equal maxima, neighbouring values, of both signs."""
    print("case", size, dt, flush=True)
    n = 9001
    gen = torch.Generator().manual_seed(12)
    for sign in (1.0, -1.0):
        one = torch.tensor(sign * size).to(dt)
        x = one.expand(5, n).clone()
        other = one * (1 - sign * 2 * torch.finfo(dt).eps)  # below it
        x[1] = torch.where(torch.rand(n, generator=gen) < 0.001, one, other)
        x[2, ::3] = other
        x[3] = torch.where(torch.rand(n, generator=gen) < 0.5, other, other * (1 - sign * 4 * torch.finfo(dt).eps))
        x[3, 8000] = one
        x[4] = (sign * size * (1 + torch.randn(n, generator=gen) / 8).clamp(max=1.1)).clamp(torch.finfo(dt).min, torch.finfo(dt).max).to(dt)
        tok = torch.tensor([4, int(x[1].argmax()), 0, 8000, int(x[4].argmax())])
        _run(x, tok, 3)
        _run(x, tok, 3, each=True)


def test_ascending_through_the_change_of_form():
    """Maxima that rise by a little from tile to tile, from numbers where one fma an exponent does
    not do to those where it does and back, with what came before still counting."""
    n = 60000
    i = torch.arange(n)
    x = torch.stack([-(2.0 ** 20) - 40 + i / 2048 * 4,      # -1048616 .. -1048498
                     2.0 ** 20 - 60 + i / 2048 * 4,         # 1048516 .. 1048633
                     -(2.0 ** 21) + i / 2048 * 0.5,
                     -(2.0 ** 20) - 5000 + i / 2048 * 200,  # steps beyond which nothing counts
                     -(2.0 ** 20) - 250 + i / 2048 * 256.0]).float()
    tok = torch.tensor([n - 1, n - 1, n - 5, n - 1, n - 1])
    _run(x, tok, 4)
    _run(x, tok, 4, each=True)
    _run(x.flip(1).contiguous(), n - 1 - tok, 4)


@WIDE
@pytest.mark.parametrize("mask", [-1e9, -1e10, -1e30])
def test_nan_among_masked_tokens(mask, dt):
    n = 30000
    x = torch.full((3, n), mask).to(dt)
    x[:, 25000:] = torch.randn((3, 5000), generator=torch.Generator().manual_seed(13)).to(dt)
    x[0, 3] = x[1, 9000] = x[2, 29999] = math.nan
    _run(x, torch.tensor([26000, 26000, 26000]), 3)
    _run(x, torch.tensor([26000, 26000, 26000]), 3, each=True)


@pytest.mark.parametrize("mask", [-1e9, -1e10, -1e30])
def test_masked_rows_in_a_workgroup_each(mask):
    n, rows = 20001, 1040
    x = torch.full((rows, n), mask).bfloat16()
    gen = torch.Generator().manual_seed(14)
    x[::2, 12000:12100] = torch.randn((rows // 2, 100), generator=gen).bfloat16()
    x[1::4, 19000:] = torch.randn((rows // 4, n - 19000), generator=gen).bfloat16()
    x[3::4] = torch.randn((rows // 4, n), generator=gen).bfloat16()
    x[7] = mask
    _run(x, torch.full((rows,), 12050), 3)

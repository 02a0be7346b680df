"""Results that the caller gives read_kv_paged_fp8: two tensors, apart from each other; nothing here reaches a GPU."""
import pytest
import torch

import yirage_amd.fused as F
from yirage_amd import YirageHipError

BF = torch.bfloat16


def _read(out, total=2):
    cache = torch.zeros((4, 16, 2, 64), dtype=torch.float8_e4m3fn)
    scale = torch.zeros((4, 16, 2), dtype=torch.uint8).view(torch.float8_e8m0fnu)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)
    return F.read_kv_paged_fp8(cache, cache, scale, scale, i32(0, 1, 2), i32(0, 1), i32(3, 4), i32(0, 1, total), total, out=out)


both = torch.zeros((5, 2, 64), dtype=BF)


@pytest.mark.parametrize("out,text", [
    ((both[:2],), "two"), ((both[:2], both[2:4], both[:2]), "two"), (both[0], "two"), ((both[:2], both[:2]), "apart"),
    ((both[:2], both[1:3]), "apart"), ((both[3:], both[2:4]), "apart"), ((both[:2], both[2:4]), "GPU"), (torch.zeros((2, 2, 2, 64), dtype=BF), "GPU"),
])
def test_out(out, text):
    with pytest.raises(YirageHipError, match=text):
        _read(out)

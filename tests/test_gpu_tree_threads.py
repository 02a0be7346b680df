"""Two host threads on one stream: attention of new rows beside itself and beside the other operators
that have scratch there."""
import threading

import pytest
import torch

import yirage_amd.fused as F
from tests.paged_plain import Batch

pytestmark = pytest.mark.gpu


def _call(lens, news, hq, hkv, d, seed):
    gen = torch.Generator().manual_seed(seed)
    b = Batch(lens, news, 16, seed=seed)
    q = torch.randn((b.rows, hq, d), generator=gen).to(torch.bfloat16).cuda()
    k, v = (torch.randn((b.pool, 16, hkv, d), generator=gen).to(torch.bfloat16).cuda() for _ in range(2))
    args, qo = b.args(), b.qo()
    return lambda: F.gqa_tree_paged(q, k, v, *args, qo_indptr=qo)


def _logprobs(seed):
    gen = torch.Generator().manual_seed(seed)
    logits = torch.randn((3, 50000), generator=gen).cuda()
    tokens = torch.arange(3).cuda()
    return lambda: F.token_logprobs(logits, tokens, top_n=3)[0]


def test_threads_on_one_stream():
    calls = [_call([9000, 300], [3, 2], 8, 2, 64, 1), _call([4000], [70], 8, 2, 128, 2), _logprobs(3)]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    wrong, start = [], threading.Barrier(len(calls))

    def run(i):
        try:
            start.wait()
            for _ in range(200):
                if not torch.equal(calls[i](), want[i]):
                    wrong.append(i)
        except Exception as e:  # (a thread's own error)
            wrong.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong

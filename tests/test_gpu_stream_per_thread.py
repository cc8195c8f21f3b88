"""hipStreamPerThread, one handle that is another stream in every thread:
calls of several threads without a workspace do not share one."""
import threading

import numpy as np
import pytest
import torch

from _paged import attend, gather, i32, norm_tol, pool, tables
from rusty_whisper_amd import _abi as A

pytestmark = pytest.mark.gpu

PER_THREAD = 2  # ((hipStream_t)2)


def in_threads(n, work):
    errors = []

    def guarded(i):
        try:
            A.init(0)
            work(i)
            torch.cuda.synchronize()
        except Exception as e:  # reported by the main thread
            errors.append(e)

    ts = [threading.Thread(target=guarded, args=(i,)) for i in range(n)]
    [t.start() for t in ts], [t.join() for t in ts]
    assert not errors, errors


@pytest.fixture(scope="module", autouse=True)
def _device():
    A.init(0)
    torch.cuda.init()


def test_paged_attention():
    page, dim, heads, n, threads = 64, 64, 2, 5000, 4
    P = A.KvPages(*pool("bf16", 1, 80, heads, page, dim, seed=22))
    table = tables([n], page, 80, seed=22)
    td, ld = i32(table), i32([n])
    assert A.paged_attention_workspace_size(P, 1, heads, n) > 0
    qs = [torch.randn(1, heads * dim, device="cuda") for _ in range(threads)]
    outs = [torch.empty_like(x) for x in qs]
    K, V = gather(P.k, P.v, 0, table[0], n)
    for _ in range(2):  # the second time with threads that follow ended ones
        [o.fill_(float("nan")) for o in outs]
        torch.cuda.synchronize()

        def work(i):
            for _ in range(50):
                A.paged_attention_dev(P, 0, qs[i], 1, heads, td, ld, n, outs[i], stream=PER_THREAD)

        in_threads(threads, work)
        for q, out in zip(qs, outs):
            want, tol = attend(q[0].double().cpu().numpy().reshape(heads, dim), K, V)
            got = out[0].double().cpu().numpy().reshape(heads, dim)
            assert np.all(np.abs(got - want) <= tol)
            assert np.linalg.norm(got - want) <= norm_tol(1.0, dim, n) * np.linalg.norm(want)


def test_token_logprobs():
    rows, n, k, threads = 3, 51866, 5, 4
    xs = [torch.randn(rows, n, device="cuda") * 3 for _ in range(threads)]
    tok = torch.arange(rows, dtype=torch.int32, device="cuda")[:, None].contiguous()
    assert A.token_logprobs_workspace_size(rows, n, k) > 0

    def arrays():
        return (torch.empty(rows, 1, device="cuda"), torch.empty(rows, device="cuda"),
                torch.empty(rows, k, dtype=torch.int32, device="cuda"), torch.empty(rows, k, device="cuda"))

    def call(x, a, stream):
        A.token_logprobs_dev(x, rows, n, tok, 1, a[0], entropy=a[1], k=k, top_ids=a[2], top_logprobs=a[3], stream=stream)

    got, want = [arrays() for _ in xs], [arrays() for _ in xs]
    torch.cuda.synchronize()
    in_threads(threads, lambda i: [call(xs[i], got[i], PER_THREAD) for _ in range(50)])
    for x, a, b in zip(xs, got, want):
        call(x, b, None)
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(a, b))

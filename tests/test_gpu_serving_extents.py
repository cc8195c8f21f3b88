"""The serving kernels at the most parts a launch has."""
import numpy as np
import pytest
import torch

from _paged import attend, gather, i32, norm_tol, pool, tables
from rusty_whisper_amd import _abi as A

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def _device():
    A.init(0)
    torch.cuda.init()


@pytest.mark.parametrize("n", [65530, 70001])
def test_attention_over_the_most_chunks(n):
    """512 chunks of 128 keys (and the next length, chunks of 256)."""
    page, dim = 256, 128
    n_pages = -(-n // page)
    P = A.KvPages(*pool("f32", 1, n_pages, 1, page, dim, seed=18))
    assert A.paged_attention_workspace_size(P, 1, 1, n) == 512 * (dim + 2) * 4
    table = tables([n], page, n_pages, seed=18)
    q, out = torch.randn(1, dim, device="cuda"), torch.empty(1, dim, device="cuda")
    A.paged_attention_dev(P, 0, q, 1, 1, i32(table), i32([n]), n, out)
    torch.cuda.synchronize()
    want, tol = attend(q.double().cpu().numpy(), *gather(P.k, P.v, 0, table[0], n))
    got = out.double().cpu().numpy()
    assert np.all(np.abs(got - want) <= tol)
    assert np.linalg.norm(got - want) <= norm_tol(1.0, dim, n) * np.linalg.norm(want)


def test_scores_of_64_parts_of_more_than_64_steps():
    """8.65 million logits: 64 parts of 135168, of which each of two wavefronts
    takes 66 steps of 1024.  Tolerances: at most 66 x 16 + 200 terms are summed
    one after the other, the rest as in test_gpu_token_logprobs.py."""
    n, k = 8_650_000, 32
    x = torch.randn(2, n, device="cuda") * 2
    x[1, -5:] = 20.0  # equal, in the last part
    # a part's sums are 16 bytes, its k best 8 k
    assert A.token_logprobs_workspace_size(2, n, k) == 2 * 64 * (16 + 8 * k)
    tokens = np.array([[0, n - 1], [n // 2, n]])
    lp, ent = torch.empty(2, 2, device="cuda"), torch.empty(2, device="cuda")
    ids, top = torch.empty(2, k, dtype=torch.int32, device="cuda"), torch.empty(2, k, device="cuda")
    A.token_logprobs_dev(x, 2, n, i32(tokens), 2, lp, entropy=ent, k=k, top_ids=ids, top_logprobs=top)
    torch.cuda.synchronize()
    for r in range(2):
        d = x[r].double().cpu().numpy()
        order = np.lexsort((np.arange(n), -d))[:k]
        d -= d.max()
        e = np.exp(d)
        S, T = e.sum(), (d * e).sum()
        share = (66 * 16 + 284) * U + 2 * U * abs(T) / S
        tol = share + U * np.abs(d) + 3 * U * (np.log(S) + 1)
        assert ids[r].tolist() == order.tolist()
        assert np.all(np.abs(top[r].double().cpu().numpy() - (d[order] - np.log(S))) <= tol[order])
        for i, t in enumerate(tokens[r]):
            got = float(lp[r, i])
            assert np.isnan(got) if t >= n else abs(got - (d[t] - np.log(S))) <= tol[t]
        H = np.log(S) - T / S
        assert abs(float(ent[r]) - H) <= 2 * share * (1 + abs(T) / S) + 3 * U * (np.log(S) + abs(T) / S)


def test_a_write_of_more_rows_than_one_launch_takes():
    """2^21 + 33 rows of 8192 values (2^23 + 256 tiles), few of which have a
    place: around the end of the first launch and at both ends."""
    heads, dim, page, rows = 64, 128, 16, 2**21 + 33
    n = heads * dim
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 69 GB for the rows")
    x = torch.empty(rows, n, device="cuda")
    at = [0, 1, 31, 32, 2**21 - 32, 2**21 - 1, 2**21, 2**21 + 1, 2**21 + 31, 2**21 + 32]
    k, v = pool("f32", 1, 1, heads, page, dim, seed=0, fill=-3.0)
    pos = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    for i, r in enumerate(at):
        x[r] = torch.arange(n, device="cuda") + i * 2**-8
        pos[r] = i
    A.kv_write_dev(A.KvPages(k, v), 0, x, x, rows, i32([[0]]), pos, seq=torch.zeros_like(pos))
    torch.cuda.synchronize()
    for i, r in enumerate(at):
        want = x[r].reshape(heads, dim)
        assert torch.equal(k[0, 0, :, i], want) and torch.equal(v[0, 0, :, :, i], want), r
    assert torch.all(k[0, 0, :, len(at):] == -3) and torch.all(v[0, 0, :, :, len(at):] == -3)
    del x
    torch.cuda.empty_cache()

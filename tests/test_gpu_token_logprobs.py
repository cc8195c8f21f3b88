"""Log-probs of given tokens, entropy and top alternatives on the GPU against
the definitions in 64 bits.

Tolerances (u = 2^-24, half a step of f32; M the row's maximum, S = sum
e^(x - M), T = sum (x - M) e^(x - M)): the sums run over at most n / 256 + 80
terms one after the other, each term's exponential is off by 4 u and, through
its argument, by 2 u |x - M|.  So S is off by (n / 256 + 84) u + 2 u |T| / S of
itself, a log-prob by that, by u |x - M| and by 3 u of its own parts' sizes,
and the entropy, ln S + |T| / S, by twice S's share of (1 + |T| / S) and 3 u of
its parts."""
import numpy as np
import pytest
import torch

from rusty_whisper_amd import _abi as A

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24
NONE = 0xFFFFFFFF


@pytest.fixture(scope="module", autouse=True)
def _device():
    A.init(0)
    torch.cuda.init()


def score(logits, tokens, k=0, entropy=True, **kw):
    """(logprobs, entropy, ids, top) as numpy; logits may be a column block."""
    rows, n = logits.shape
    tok = np.ascontiguousarray(tokens, dtype=np.uint32)
    t = torch.from_numpy(tok.view(np.int32)).cuda()
    lp = torch.full(tok.shape, -9.0, device="cuda")
    ent = torch.full((rows,), -9.0, device="cuda") if entropy else None
    ids = torch.full((rows, max(k, 1)), 7, dtype=torch.int32, device="cuda")
    top = torch.full((rows, max(k, 1)), -9.0, device="cuda")
    A.token_logprobs_dev(logits, rows, n, t, tok.shape[1], lp, entropy=ent, k=k, top_ids=ids, top_logprobs=top, **kw)
    torch.cuda.synchronize()
    return lp.cpu().numpy(), None if ent is None else ent.cpu().numpy(), ids.cpu().numpy().view(np.uint32), top.cpu().numpy()


def close(got, want, tol, what):
    # a value beyond f32's range (the difference of two logits can be) has an
    # infinity as its nearest f32: 2^128 - 2^103, half a step past the largest, on
    inf = np.abs(want) >= 2.0**128 - 2.0**103
    assert np.array_equal(got[inf], np.copysign(np.inf, want[inf]).astype(np.float32)), what
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    ok = ~inf & ~np.isnan(want)
    bad = np.abs(got[ok].astype(np.float64) - want[ok]) > np.broadcast_to(tol, want.shape)[ok]
    assert not bad.any(), (what, got[ok][bad][:4], want[ok][bad][:4])


def check(logits, tokens, k, lp, ent, ids, top):
    x = logits.double().cpu().numpy()
    n = x.shape[1]
    tok = np.asarray(tokens, dtype=np.uint32)
    for r in range(x.shape[0]):
        M = x[r].max()
        d = x[r] - M
        e = np.exp(d)
        S = e.sum()
        T = (d[e > 0] * e[e > 0]).sum()
        share = (n / 256 + 84) * U + 2 * U * abs(T) / S
        all_lp = d - np.log(S)
        tol = share + U * np.where(np.isinf(d), 0, np.abs(d)) + 3 * U * (np.log(S) + 1)
        want = np.array([0.0 if t == NONE else all_lp[t] if t < n else np.nan for t in tok[r]])
        close(lp[r], want, np.array([tol[t] if t < n else 0.0 for t in tok[r]]), f"row {r}: log-probs")
        if ent is not None:
            H = np.log(S) - T / S
            close(ent[r : r + 1], np.array([H]), 2 * share * (1 + abs(T) / S) + 3 * U * (np.log(S) + abs(T) / S), f"row {r}: entropy")
        order = np.argsort(-x[r], kind="stable")[:k]
        order = order[x[r][order] > -np.inf]
        assert ids[r, : len(order)].tolist() == order.tolist(), f"row {r}: alternatives"
        close(top[r, : len(order)], all_lp[order], tol[order], f"row {r}: alternatives' log-probs")
        assert np.all(ids[r, len(order) : k] == NONE) and np.all(np.isneginf(top[r, len(order) : k]))
    if k == 0:
        assert np.all(ids == 7) and np.all(top == -9)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("n", [1, 2, 31, 63, 64, 65, 255, 257, 1000, 2048, 4095, 4097, 8193, 51866, 131072, 262147])
@pytest.mark.parametrize("k", [0, 1, 5, 32])
def test_sizes(dtype, n, k):
    rng = np.random.default_rng(n + k)
    logits = (torch.randn(3, n, device="cuda") * 3).to(DTYPES[dtype])
    tokens = rng.integers(0, n, (3, 4))
    check(logits, tokens, k, *score(logits, tokens, k))


@pytest.mark.parametrize("rows,n,k", [(r, n, k) for r in (1, 2, 5, 33, 300) for n, k in ((257, 5), (5003, 16), (51866, 5))]
                         + [(1500, 257, 5), (1500, 5003, 16), (2100, 3000, 32)])
def test_rows(rows, n, k):
    logits = torch.randn(rows, n, device="cuda") * 2
    tokens = np.random.default_rng(rows).integers(0, n, (rows, 1))
    check(logits, tokens, k, *score(logits, tokens, k))


def test_a_vocabulary_of_millions():
    """More than 64 steps per part, 64 parts."""
    n, k = 3_000_001, 32
    logits = torch.randn(2, n, device="cuda") * 2
    tokens = [[0, n - 1], [n // 2, n]]
    check(logits, tokens, k, *score(logits, tokens, k))


def test_a_captured_call_brings_its_workspace():
    x = torch.randn(1, 51866, device="cuda")
    t, lp = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.empty(1, 1, device="cuda")
    assert A.token_logprobs_workspace_size(1, 51866, 0) > 0
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        lp.zero_()
        with pytest.raises(A.RwError, match="captured call needs a workspace"):
            A.token_logprobs_dev(x, 1, 51866, t, 1, lp, stream=torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("n_tok", [0, 1, 2, 99, 1000])
def test_tokens_per_row(n_tok):
    n = 5001
    logits = torch.randn(4, n, device="cuda")
    tokens = np.random.default_rng(n_tok).integers(0, n, (4, n_tok)).astype(np.uint32)
    if n_tok > 1:
        tokens[:, 1] = tokens[:, 0]  # the same id twice
        tokens[2] = NONE
        tokens[3, 0], tokens[3, -1] = n, n - 1
        tokens[1, -1] = NONE - 1
    check(logits, tokens, 3, *score(logits, tokens, 3))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("ld,at", [(1003, 0), (1024, 1), (1001, 1), (1007, 3)])
def test_strides_and_alignment(dtype, ld, at):
    n = 1000
    wide = torch.full((6, ld), float("nan"), dtype=DTYPES[dtype], device="cuda")
    wide[:, at : at + n] = torch.randn(6, n, device="cuda").to(DTYPES[dtype])
    logits = wide[:, at : at + n]
    tokens = np.arange(6)[:, None] * 199
    check(logits, tokens, 8, *score(logits, tokens, 8, ld=ld))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("n", [70, 3000, 51866])
def test_ties(dtype, n):
    """Equal logits: lowest id first, wherever they are."""
    rng = np.random.default_rng(n)
    rows = [np.zeros(n), rng.integers(0, 3, n) * 0.5, np.repeat(np.arange(n // 10 + 1), 10)[:n] % 7 * 1.0,
            np.where(np.arange(n) % 64 == 5, 4.0, -1.0), np.where(np.arange(n) >= n - 40, 2.0, 1.0),
            np.where(np.arange(n) < 40, 0.0, -0.0)]
    logits = torch.from_numpy(np.stack(rows).astype(np.float32)).to(DTYPES[dtype]).cuda()
    tokens = rng.integers(0, n, (len(rows), 2))
    for k in (1, 16, 32):
        check(logits, tokens, k, *score(logits, tokens, k))


@pytest.mark.parametrize("n", [64, 5000, 51866])
def test_sorted_rows(n):
    """Every candidate in a few neighbouring lanes, or in the last chunk."""
    up = torch.arange(n, device="cuda", dtype=torch.float32) * 2.0**-9
    far = up.clone()
    far[n // 2 : n // 2 + 64] += 500.0
    logits = torch.stack([up, up.flip(0), far])
    tokens = [[0, n - 1]] * 3
    for k in (5, 32):
        check(logits, tokens, k, *score(logits, tokens, k))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("n", [40, 3000, 51866])
def test_suppressed_and_lowest(dtype, n):
    t = DTYPES[dtype]
    inf, low = float("inf"), torch.finfo(t).min
    x = torch.randn(6, n, device="cuda").to(t)
    x[0, 1:] = -inf                      # one candidate
    x[1, ::2] = -inf
    x[2, : n - 3] = -inf                 # fewer than k
    x[3, :] = low                        # all at the type's lowest value
    x[4, :] = low
    x[4, 7] = torch.finfo(t).max         # differences beyond the type's range
    x[5, 10:] = low
    tokens = [[0, 1, n - 1, 7]] * 6
    check(x, tokens, 16, *score(x, tokens, 16))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("mask", ["-inf", "lowest"])
@pytest.mark.parametrize("rows", [1, 600])
def test_masks_that_leave_a_range(dtype, mask, rows):
    """As after a rule on timestamps: a few hundred neighbouring ids are left."""
    n, t = 51866, DTYPES[dtype]
    x = torch.full((rows, n), -float("inf") if mask == "-inf" else torch.finfo(t).min, dtype=t, device="cuda")
    at = torch.arange(rows, device="cuda") * 61 % (n - 700)
    x.scatter_(1, at[:, None] + torch.arange(700, device="cuda"), torch.randn(rows, 700, device="cuda").to(t))
    tokens = np.stack([at.cpu().numpy() + 3, np.zeros(rows, np.int64)], 1)
    for k in (5, 32):
        check(x, tokens, k, *score(x, tokens, k))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("n", [33, 4100, 51866])
def test_rows_without_a_distribution(dtype, n):
    inf = float("inf")
    x = torch.randn(6, n, device="cuda").to(DTYPES[dtype])
    x[0, n // 2] = float("nan")
    x[1, n - 1] = inf
    x[2, :] = -inf
    x[3, :] = float("nan")
    x[4, 0], x[4, n - 1] = inf, float("nan")
    tokens = [[0, n - 1, NONE, n]] * 6
    lp, ent, ids, top = score(x, tokens, 5)
    for r in range(5):
        assert np.all(np.isnan(lp[r, [0, 1, 3]])) and lp[r, 2] == 0 and np.isnan(ent[r])
        assert np.all(ids[r] == NONE) and np.all(np.isnan(top[r]))
    check(x[5:], tokens[5:], 5, lp[5:], ent[5:], ids[5:], top[5:])


def test_without_entropy_and_without_tokens():
    x = torch.randn(2, 3000, device="cuda")
    lp, ent, ids, top = score(x, np.empty((2, 0)), 4, entropy=False)
    check(x, np.empty((2, 0)), 4, lp, None, ids, top)
    A.token_logprobs_dev(x, 2, 3000, None, 0, None)  # nothing asked for: nothing written
    torch.cuda.synchronize()


def test_workspace_and_stream():
    rows, n, k = 4, 51866, 7
    x = torch.randn(rows, n, device="cuda")
    tokens = [[3]] * rows
    need = A.token_logprobs_workspace_size(rows, n, k)
    ws = torch.full((need + 512,), 77, dtype=torch.uint8, device="cuda")
    ref = score(x, tokens, k)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = score(x, tokens, k, workspace=ws[256:], workspace_len=need, stream=s.cuda_stream)
    for a, b in zip(ref, got):
        assert np.array_equal(a, b)
    assert torch.all(ws[:256] == 77) and torch.all(ws[256 + need :] == 77)
    if need:
        with pytest.raises(A.RwError, match="workspace"):
            score(x, tokens, k, workspace=ws, workspace_len=need - 1)


@pytest.mark.parametrize("rows,n", [(2, 51866), (400, 3000)])
def test_captured_and_replayed(rows, n):
    k = 5
    x, t = torch.randn(rows, n, device="cuda"), torch.zeros(rows, 2, dtype=torch.int32, device="cuda")
    lp, ent = torch.empty(rows, 2, device="cuda"), torch.empty(rows, device="cuda")
    ids, top = torch.empty(rows, k, dtype=torch.int32, device="cuda"), torch.empty(rows, k, device="cuda")
    ws = torch.empty(max(1, A.token_logprobs_workspace_size(rows, n, k)), dtype=torch.uint8, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        A.token_logprobs_dev(x, rows, n, t, 2, lp, entropy=ent, k=k, top_ids=ids, top_logprobs=top, workspace=ws,
                             workspace_len=ws.numel(), stream=torch.cuda.current_stream().cuda_stream)
    for i in range(4):
        x.normal_()
        tokens = np.random.default_rng(i).integers(0, n, (rows, 2)).astype(np.int32)
        t.copy_(torch.from_numpy(tokens))
        g.replay()
        torch.cuda.synchronize()
        check(x, tokens, k, lp.cpu().numpy(), ent.cpu().numpy(), ids.cpu().numpy().view(np.uint32), top.cpu().numpy())
        eager = score(x, tokens, k)
        assert np.array_equal(eager[0], lp.cpu().numpy()) and np.array_equal(eager[3], top.cpu().numpy())


def test_agrees_with_logits_topk():
    """The k best of both entries on rows without equal logits."""
    n, k = 51866, 5
    x = torch.randn(4, n, device="cuda") * 3
    ids2, lps2 = torch.empty(4, k, dtype=torch.int32, device="cuda"), torch.empty(4, k, device="cuda")
    A.logits_topk_dev(x, 4, n, k, ids2, lps2)
    _, _, ids, top = score(x, np.zeros((4, 1)), k)
    torch.cuda.synchronize()
    assert np.array_equal(ids, ids2.cpu().numpy().view(np.uint32))
    assert np.max(np.abs(top - lps2.cpu().numpy())) <= 2e-5

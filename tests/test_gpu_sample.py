"""Sampling on the GPU: the same token as the definition in 64 bits gives.

The log of a token's share: rounded once to f32 (half a step, 2^-24 of it), and
the kept weight, a sum of n weights each off by 2^-43 of the largest."""
import numpy as np
import pytest
import torch

from _draft import sample
from _paged import U, i32
from rusty_whisper_amd import _abi as A

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
NONE = 0xFFFFFFFF


@pytest.fixture(scope="module", autouse=True)
def _device():
    A.init(0)
    torch.cuda.init()


def f32(a):
    return torch.from_numpy(np.array(a, dtype=np.float32)).cuda()


def draw(logits, u, t=None, top_k=None, top_p=None, min_p=None, **kw):
    """(tokens, logprobs) of rows; settings: None, a number or one per row."""
    rows, n = logits.shape
    each = lambda x, f: None if x is None else f(np.broadcast_to(np.asarray(x), (rows,)))  # noqa: E731
    tok = torch.full((rows,), 77, dtype=torch.int32, device="cuda")
    lp = torch.full((rows,), 9.0, device="cuda")
    A.sample_tokens_dev(logits, rows, n, f32(np.broadcast_to(u, (rows,))), tok, logprobs=lp, temperature=each(t, f32),
                        top_k=each(top_k, lambda a: i32(a.copy())), top_p=each(top_p, f32), min_p=each(min_p, f32), **kw)
    torch.cuda.synchronize()
    return tok.cpu().numpy().view(np.uint32), lp.cpu().numpy()


def check(logits, u, got, t=1.0, top_k=0, top_p=1.0, min_p=0.0):
    x = logits.double().cpu().numpy()
    rows, n = x.shape
    u, t, top_k, top_p, min_p = (np.broadcast_to(np.asarray(v, np.float32), (rows,)) for v in (u, t, top_k, top_p, min_p))
    for r in range(rows):
        tok, lp = sample(x[r], float(u[r]), float(t[r]), int(top_k[r]), float(top_p[r]), float(min_p[r]))
        assert got[0][r] == tok, (r, got[0][r], tok)
        assert abs(float(got[1][r]) - lp) <= 2 * U * (abs(lp) + 1e-3) + n * 2.0**-43, (r, got[1][r], lp)


SETTINGS = [dict(), dict(t=0.7), dict(t=0.0), dict(top_k=1), dict(top_k=7), dict(top_k=400, t=1.7), dict(top_p=0.5),
            dict(top_p=0.95, t=1.3), dict(min_p=0.05), dict(top_k=50, top_p=0.9, min_p=0.02, t=0.9)]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("n", [1, 2, 5, 64, 1000, 4099, 16411, 51866, 57355, 100003, 262147])
@pytest.mark.parametrize("setting", SETTINGS, ids=str)
def test_sizes_and_settings(dtype, n, setting):
    rng = np.random.default_rng(n)
    logits = (torch.randn(4, n, device="cuda") * 2.5).to(DTYPES[dtype])
    u = rng.random(4, dtype=np.float32)
    check(logits, u, draw(logits, u, **setting), **setting)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_settings_of_each_row(dtype):
    rng = np.random.default_rng(1)
    rows, n = 200, 5003
    logits = (torch.randn(rows, n, device="cuda") * 3).to(DTYPES[dtype])
    logits[:, ::7] = -float("inf")
    u = rng.random(rows, dtype=np.float32)
    kw = dict(t=rng.choice([0.0, 0.2, 1.0, 5.0], rows), top_k=rng.choice([0, 1, 3, 90], rows),
              top_p=rng.choice([1.0, 0.3, 0.9, 0.999], rows), min_p=rng.choice([0.0, 0.01, 0.5], rows))
    check(logits, u, draw(logits, u, **kw), **kw)


@pytest.mark.parametrize("setting", SETTINGS, ids=str)
@pytest.mark.parametrize("levels", [1, 2, 40])
def test_many_equal_logits(setting, levels):
    """Ties go by lowest id, also where a question falls among thousands of them."""
    rng = np.random.default_rng(levels)
    n = 60001
    logits = torch.from_numpy(rng.integers(0, levels, (3, n)).astype(np.float32) * 0.25).cuda()
    # (not next to a border between equal shares, where the definition's own sums round)
    u = np.array([0.123457, 0.5000031, 0.987653], np.float32)
    check(logits, u, draw(logits, u, **setting), **setting)


@pytest.mark.parametrize("spread", [1e-30, 1e-3, 1.0, 1e4, 1e30])
@pytest.mark.parametrize("t", [1e-20, 0.01, 1.0, 100.0, 1e30])
def test_spreads_and_temperatures(spread, t):
    rng = np.random.default_rng(3)
    logits = torch.randn(3, 3001, device="cuda") * spread
    u = rng.random(3, dtype=np.float32)
    for kw in (dict(), dict(top_p=0.8), dict(top_k=100, min_p=0.1)):
        check(logits, u, draw(logits, u, t=t, **kw), t=t, **kw)


def test_logits_at_the_ends_of_the_range():
    big = float(np.finfo(np.float32).max)
    x = torch.full((4, 500), -big, device="cuda")
    x[0, 3], x[0, 9] = big, big
    x[1, 499] = 0.0
    x[2] = torch.from_numpy(np.linspace(-1, 1, 500) * big).float()  # (in f32, linspace passes its end)
    u = np.array([0.6, 0.99, 0.5, 0.5041], np.float32)
    check(x, u, draw(x, u))
    for t in (1e38, 3e38):
        check(x, u, draw(x, u, t=t, top_p=0.7), t=t, top_p=0.7)


def test_u_at_its_ends():
    logits = torch.randn(1, 999, device="cuda")
    x = logits.double().cpu().numpy()[0]
    order = np.argsort(-x, kind="stable")
    assert draw(logits, 0.0)[0][0] == order[0]
    assert draw(logits, 1.0)[0][0] == order[-1] == draw(logits, 7.0)[0][0]
    assert draw(logits, -3.0)[0][0] == order[0]
    assert draw(logits, 1.0, top_k=10)[0][0] == order[9]
    assert draw(logits, 0.99999994, top_p=0.0)[0][0] == order[0] == draw(logits, 0.99999994, top_p=-1.0)[0][0]
    assert draw(logits, 0.99999994, min_p=2.0)[0][0] == order[0]


def test_rows_without_a_token():
    x = torch.randn(8, 100, device="cuda")
    x[0, 5] = float("nan")
    x[1, 5] = float("inf")
    x[2] = -float("inf")
    t = np.array([1, 1, 1, np.nan, np.inf, 1, 1, 1], np.float32)
    p = np.array([1, 1, 1, 1, 1, np.nan, 1, 1], np.float32)
    m = np.array([0, 0, 0, 0, 0, 0, np.nan, 0], np.float32)
    tok, lp = draw(x, 0.5, t=t, top_p=p, min_p=m)
    assert np.all(tok[:7] == NONE) and np.isnan(lp[:7]).all() and tok[7] < 100 and np.isfinite(lp[7])
    tok, lp = draw(x, np.array([0.5] * 7 + [np.nan], np.float32))
    assert tok[7] == NONE and np.isnan(lp[7])
    tok, lp = draw(x, 0.5, t=0.0)
    assert np.all(tok[:3] == NONE) and np.all(tok[3:] < 100)


def test_a_greedy_row_takes_the_lowest_id():
    x = torch.zeros(3, 40000, device="cuda")
    x[0, 39999] = x[0, 20000] = 1.0
    x[1, 0] = -1.0
    x[2] = -float("inf")
    x[2, 77] = -5.0
    for kw in (dict(t=0.0), dict(t=-1.0), dict(top_k=1)):
        tok, lp = draw(x, 0.9, **kw)
        assert tok.tolist() == [20000, 1, 77] and np.all(lp == 0)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("ld,at", [(1003, 0), (1024, 1), (1001, 1), (1007, 3)])
def test_strides_and_alignment(dtype, ld, at):
    n = 1000
    wide = torch.full((6, ld), float("nan"), dtype=DTYPES[dtype], device="cuda")
    wide[:, at : at + n] = (torch.randn(6, n, device="cuda") * 2).to(DTYPES[dtype])
    logits = wide[:, at : at + n]
    u = np.random.default_rng(at).random(6, dtype=np.float32)
    check(logits, u, draw(logits, u, top_p=0.9, ld=ld), top_p=0.9)


def test_the_largest_vocabulary():
    n = 1 << 20
    logits = torch.randn(2, n, device="cuda") * 2
    u = np.array([0.3, 0.9], np.float32)
    for kw in (dict(), dict(top_p=0.9), dict(top_k=5000)):
        check(logits, u, draw(logits, u, **kw), **kw)
    logits = torch.zeros(2, n, device="cuda")  # one value: the id is all there is to tell
    check(logits, u, draw(logits, u, top_k=700001), top_k=700001)


@pytest.mark.parametrize("rows", [1, 3, 700])
def test_the_draws_follow_the_shares(rows):
    """Evenly spaced numbers take each token as often as its share says."""
    x = torch.tensor([[2.0, 1.0, 0.0, 1.0, -9.0]], device="cuda").repeat(rows * 100, 1)
    u = (np.arange(rows * 100) + 0.5) / (rows * 100)
    tok, _ = draw(x, u.astype(np.float32), t=2.0)
    p = np.exp(np.array([1.0, 0.5, 0.0, 0.5, -4.5]))
    count = np.bincount(tok, minlength=5) / (rows * 100)
    assert np.all(np.abs(count - p / p.sum()) <= 1.01 / (rows * 100) + 1e-6)


def test_calls_repeat_themselves():
    logits = (torch.randn(50, 51866, device="cuda") * 2).bfloat16()
    u = np.random.default_rng(0).random(50, dtype=np.float32)
    first = draw(logits, u, top_p=0.95)
    for _ in range(5):
        again = draw(logits, u, top_p=0.95)
        assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1])


def test_a_captured_call_replayed_with_other_contents():
    rows, n = 7, 51866
    logits, u = torch.randn(rows, n, device="cuda"), torch.rand(rows, device="cuda")
    tok, lp = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(rows, device="cuda")
    p = torch.full((rows,), 0.9, device="cuda")
    size = A.sample_tokens_workspace_size(rows, n)
    ws = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        A.sample_tokens_dev(logits, rows, n, u, tok, logprobs=lp, top_p=p, workspace=ws, workspace_len=ws.numel(),
                            stream=torch.cuda.current_stream().cuda_stream)
    for _ in range(4):
        logits.normal_(std=3.0), u.uniform_()
        graph.replay()
        torch.cuda.synchronize()
        check(logits, u.cpu().numpy(), (tok.cpu().numpy().view(np.uint32), lp.cpu().numpy()), top_p=0.9)


def test_more_rows_than_a_launch_has_threads_for():
    rows = 2**23  # of 512 threads each
    x = torch.rand(rows, 1, device="cuda").repeat(1, 2)
    x[:, 0] += 1
    x[rows - 5, 1] = 3
    tok = torch.full((rows,), 77, dtype=torch.int32, device="cuda")
    A.sample_tokens_dev(x, rows, 2, torch.zeros(rows, device="cuda"), tok)
    torch.cuda.synchronize()
    assert tok[rows - 5] == 1
    tok[rows - 5] = 0
    assert not tok.any()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("n", [2, 1000, 51866])
def test_a_min_p_above_1_keeps_the_first_alone(dtype, n):
    """Also where others equal it; of 1 it keeps those that do."""
    logits = (torch.randn(4, n, device="cuda").clamp(max=0.5)).to(DTYPES[dtype])
    logits[:, n // 2 :] = 0.5  # half of them are the largest
    logits[3] = 0.5
    first = (logits == 0.5).cpu().numpy().argmax(1).tolist()
    for p in (1.0000001, 1.5, float("inf")):
        for kw in (dict(), dict(top_p=0.9), dict(top_k=3), dict(t=0.3)):
            tok, lp = draw(logits, 0.9375, min_p=p, **kw)
            assert tok.tolist() == first and np.all(lp == 0), (p, kw)
    u = np.array([0.123457, 0.5000031, 0.987653, 0.76543], np.float32)
    check(logits, u, draw(logits, u, min_p=1.0), min_p=1.0)


def test_a_call_needs_no_workspace():
    """None at any size, so a captured call takes none either."""
    assert all(A.sample_tokens_workspace_size(r, n) == 0 for r in (1, 61, 2**23) for n in (1, 51866, 2**20))
    logits, u = torch.randn(3, 5003, device="cuda"), torch.rand(3, device="cuda")
    tok, lp = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(3, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        A.sample_tokens_dev(logits, 3, 5003, u, tok, logprobs=lp, stream=torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        logits.normal_(std=2.0), u.uniform_()
        graph.replay()
        torch.cuda.synchronize()
        check(logits, u.cpu().numpy(), (tok.cpu().numpy().view(np.uint32), lp.cpu().numpy()))


def test_a_temperature_of_minus_infinity_takes_the_first():
    x = torch.randn(2, 300, device="cuda")
    tok, lp = draw(x, 0.9, t=np.array([-np.inf, np.inf], np.float32))
    assert tok[0] == int(x[0].argmax()) and lp[0] == 0 and tok[1] == NONE and np.isnan(lp[1])

"""Attention over pages where weights, queries or values are of very unlike
size: what f32 arithmetic keeps, every type of pool keeps."""
import numpy as np
import pytest
import torch

from _paged import DTYPES, U, attend, gather, i32, pool, tables
from rusty_whisper_amd import _abi as A

pytestmark = pytest.mark.gpu

PAGE, DIM = 32, 64


@pytest.fixture(scope="module", autouse=True)
def _device():
    A.init(0)
    torch.cuda.init()


def run(P, q, table, lens, group=1):
    out = torch.full(q.shape, float("nan"), device="cuda")
    A.paged_attention_dev(P, 0, q, q.shape[0], P.st.n_head * group, i32(table), i32(lens), int(max(lens)), out)
    torch.cuda.synchronize()
    return out.double().cpu().numpy().reshape(q.shape[0], -1, P.st.head_size)


# ------------------------------------------------------- small weights

@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("gap", [5.0, 14.0, 18.5, 20.0, 24.75, 40.0, 60.0, 75.0])
@pytest.mark.parametrize("n", [32, 448, 3000])
def test_one_key_outweighs_the_others_and_has_no_value(dtype, gap, n):
    """The result is the others' alone, whose weights are e^-gap of the largest.

    q and k have one value each that is not zero, of 8 bits or fewer, so a score
    is one exact product.  The exponential's argument, in powers of two, is
    rounded four times at most (the constant twice, its product, the
    difference): a weight is off by 4 (|s| + |largest s|) <= 8 (gap + 1) half
    steps of itself, by 4 for the exponential; sums of n products and of n
    weights by n each, the rest by 8."""
    pages = -(-n // PAGE)
    k, v = pool(dtype, 1, pages, 1, PAGE, DIM, seed=n)
    rng = np.random.default_rng(n)
    s = rng.integers(-32, 33, pages * PAGE) / 64.0
    s[3] = gap
    k.zero_()
    k[0, :, 0, :, 0] = torch.from_numpy(s).cuda().reshape(pages, PAGE).to(k.dtype)
    v[0, 0, 0, :, 3] = 0
    q = torch.zeros(1, DIM, device="cuda")
    q[0, 0] = 8.0  # scores are k's first value
    table = np.arange(pages, dtype=np.int32)[None]
    P = A.KvPages(k, v)
    got = run(P, q, table, [n])[0, 0]
    _, V = gather(k, v, 0, table[0], n)
    p = np.exp(s[:n] - s[:n].max())
    p /= p.sum()
    tol = 2 * (8 * (gap + 1) + 12 + n) * U * (p @ np.abs(V[0]))
    bad = ~(np.abs(got - p @ V[0]) <= tol)
    assert not bad.any(), (np.max(np.abs(got - p @ V[0]) / (p @ np.abs(V[0]))), np.max(tol / (p @ np.abs(V[0]))))


# ------------------------------------------- values of unlike size in q

@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("group", [1, 4])
@pytest.mark.parametrize("power", [0, 14, 22, 30, 36])
def test_a_large_value_of_q_that_meets_zeros(dtype, group, power):
    """q's first value is 2^power, all of k's first values are 0: the scores are
    the other values' (`attend`'s bound takes sum |q k|)."""
    lens = [1, 33, 700, 3000]
    n_pages = sum(-(-n // PAGE) for n in lens)
    k, v = pool(dtype, 1, n_pages, 2, PAGE, DIM, seed=power)
    k[..., 0] = 0
    q = torch.randn(4, 2 * group, DIM, device="cuda") * 2
    q[..., 0] = 2.0**power
    q = q.reshape(4, -1)
    table = tables(lens, PAGE, n_pages, seed=power)
    P = A.KvPages(k, v)
    got = run(P, q, table, lens, group)
    for r, n in enumerate(lens):
        want, tol = attend(q[r].double().cpu().numpy().reshape(-1, DIM), *gather(k, v, 0, table[r, : -(-n // PAGE)], n))
        bad = ~(np.abs(got[r] - want) <= tol)
        assert not bad.any(), (r, np.max(np.abs(got[r] - want)), np.max(tol))


# --------------------------------------------- values at the type's ends

# A product, a mean, a sum that is subnormal is off by half of 2^-149: n products,
# the divisions and joins of means below 40 more.
def subnormal(n):
    return (n + 40) * 2.0**-150


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("size", [-72, -100, -110, -120])
def test_small_values(dtype, size):
    lens = [1, 2, 33, 448, 3000]
    n_pages = sum(-(-n // PAGE) for n in lens)
    k, v = pool(dtype, 1, n_pages, 2, PAGE, DIM, seed=-size)
    v.copy_((v.double() * 2.0**size).to(v.dtype))
    q = torch.randn(len(lens), 2 * DIM, device="cuda")
    table = tables(lens, PAGE, n_pages, seed=-size)
    P = A.KvPages(k, v)
    got = run(P, q, table, lens)
    for r, n in enumerate(lens):
        K, V = gather(k, v, 0, table[r, : -(-n // PAGE)], n)
        want, tol = attend(q[r].double().cpu().numpy().reshape(-1, DIM), K, V)
        bad = ~(np.abs(got[r] - want) <= tol + subnormal(n))
        assert not bad.any(), (r, np.max(np.abs(got[r] - want)), np.max(tol))
        if n == 1:
            assert np.array_equal(got[r], V[:, 0])  # a mean of one value


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_one_key_is_its_value(dtype):
    """Whatever the value is."""
    t = torch.finfo(DTYPES[dtype])
    k, v = pool(dtype, 1, 1, 1, PAGE, DIM, seed=1)
    ends = torch.tensor([t.max, t.min, t.tiny, -t.tiny, t.tiny / 2, 0.0, 1.0, t.max / 2, t.smallest_normal * 1.5, t.eps])
    v[0, 0, 0, : len(ends), 0] = ends.to(v.dtype).cuda()
    P = A.KvPages(k, v)
    got = run(P, torch.randn(1, DIM, device="cuda"), np.zeros((1, 1), np.int32), [1])[0, 0]
    assert np.array_equal(got, v[0, 0, 0, :, 0].double().cpu().numpy())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [2, 40, 3000])
def test_largest_and_small_values_in_one_head(dtype, n):
    """Sums that pass f32's range beside ones that are small: of one head's
    values, of one query head's and another's, of one part of the keys only."""
    n_pages = -(-n // PAGE)
    k, v = pool(dtype, 1, n_pages, 2, PAGE, DIM, seed=n)
    big = torch.finfo(v.dtype).max
    v[:, :, 0, ::3] = big                                    # every key the largest
    v[:, :, 0, 1::3] = (v[:, :, 0, 1::3].double() * 2.0**-110).to(v.dtype)
    v[:, 0, 1, 5] = -big                                     # in the first page only
    q = torch.randn(1, 4 * DIM, device="cuda")
    table = np.arange(n_pages, dtype=np.int32)[None]
    P = A.KvPages(k, v)
    got = run(P, q, table, [n], group=2)[0]
    want, tol = attend(q[0].double().cpu().numpy().reshape(-1, DIM), *gather(k, v, 0, table[0], n))
    bad = ~(np.abs(got - want) <= tol + subnormal(n))
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], want[bad][:4])


# ------------------------------------------------- the largest queries

@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("q0", [torch.finfo(torch.float32).max, -torch.finfo(torch.float32).max, 3.39e38, 3.3953e38])
def test_queries_at_the_end_of_f32(dtype, q0):
    """One value of q and k is not zero; scores are about -32 .. 32 (f16, whose
    smallest value is 2^-24: of 2^101, the largest take all).  Tolerance as for
    the first test here, with scores for the gap."""
    n = 448
    pages = n // PAGE
    k, v = pool(dtype, 1, pages, 1, PAGE, DIM, seed=3)
    k0 = np.random.default_rng(3).integers(-32, 33, n) * 2.0 ** (-24 if dtype == "f16" else -125)
    k.zero_()
    k[0, :, 0, :, 0] = torch.from_numpy(k0).cuda().reshape(pages, PAGE).to(k.dtype)
    q = torch.zeros(1, DIM, device="cuda")
    q[0, 0] = q0
    table = np.arange(pages, dtype=np.int32)[None]
    P = A.KvPages(k, v)
    got = run(P, q, table, [n])[0, 0]
    _, V = gather(k, v, 0, table[0], n)
    s = float(q[0, 0]) * k0 / 8.0
    p = np.exp(s - s.max())
    p /= p.sum()
    tol = 2 * (8 * 33 + 12 + n) * U * (p @ np.abs(V[0]))
    assert np.all(np.abs(got - p @ V[0]) <= tol), (got[:4], (p @ V[0])[:4])


# ------------------------------- key heads of several query heads, infinities

@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("gap", [14.0, 20.0, 40.0, 75.0])
@pytest.mark.parametrize("n", [32, 448, 3000])
def test_small_weights_of_grouped_heads(dtype, dim, gap, n):
    """As the first test here, three query heads to a key head, each with an
    outweighing key of its own, and heads of every size (q's value is
    sqrt(dim), rounded: the scores' share of the tolerance covers it)."""
    pages, group = -(-n // PAGE), 3
    k, v = pool(dtype, 1, pages, 1, PAGE, dim, seed=n + dim)
    rng = np.random.default_rng(n)
    s = rng.integers(-32, 33, (pages * PAGE, group)) / 64.0
    for g in range(group):
        s[3 + 5 * g, g] = gap
        v[0, 0, 0, :, 3 + 5 * g] = 0
    k.zero_()
    k[0, :, 0, :, :group] = torch.from_numpy(s).cuda().reshape(pages, PAGE, group).to(k.dtype)
    q = torch.zeros(group, dim, device="cuda")
    for g in range(group):
        q[g, g] = dim**0.5
    table = np.arange(pages, dtype=np.int32)[None]
    P = A.KvPages(k, v)
    got = run(P, q.reshape(1, -1), table, [n], group)[0]
    _, V = gather(k, v, 0, table[0], n)
    for g in range(group):
        x = s[:n, g] * (float(q[g, g]) / np.sqrt(dim))
        p = np.exp(x - x.max())
        p /= p.sum()
        tol = 2 * (8 * (gap + 1) + 12 + n) * U * (p @ np.abs(V[0]))
        assert np.all(np.abs(got[g] - p @ V[0]) <= tol), (g, np.max(np.abs(got[g] - p @ V[0])), np.max(tol))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("group", [2, 17])
def test_one_key_is_its_value_for_grouped_heads(dtype, group):
    t = torch.finfo(DTYPES[dtype])
    k, v = pool(dtype, 1, 1, 1, PAGE, DIM, seed=1)
    ends = torch.tensor([t.max, t.min, t.tiny, -t.tiny, t.tiny / 2, 0.0, 1.0, t.max / 2, t.smallest_normal * 1.5, t.eps])
    v[0, 0, 0, : len(ends), 0] = ends.to(v.dtype).cuda()
    P = A.KvPages(k, v)
    got = run(P, torch.randn(1, group * DIM, device="cuda"), np.zeros((1, 1), np.int32), [1], group)[0]
    assert np.array_equal(got, np.broadcast_to(v[0, 0, 0, :, 0].double().cpu().numpy(), got.shape))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("group", [1, 2])
@pytest.mark.parametrize("n", [1, 40, 3000])
def test_infinite_values_are_not_made_finite(dtype, group, n):
    """What kv_write rounded past the type's largest shows in the result, and
    in its own place only."""
    n_pages = -(-n // PAGE)
    k, v = pool(dtype, 1, n_pages, 1, PAGE, DIM, seed=n)
    v[0, 0, 0, 7, 0] = float("inf")
    v[0, 0, 0, 9, 0] = -float("inf")
    q = torch.randn(1, group * DIM, device="cuda")
    table = np.arange(n_pages, dtype=np.int32)[None]
    P = A.KvPages(k, v)
    got = run(P, q, table, [n], group)[0]
    K, V = gather(k, v, 0, table[0], n)
    assert not np.isfinite(got[:, [7, 9]]).any()
    V[:, :, [7, 9]] = 0
    got[:, [7, 9]] = 0
    want, tol = attend(q[0].double().cpu().numpy().reshape(-1, DIM), K, V)
    assert np.all(np.abs(got - want) <= tol)

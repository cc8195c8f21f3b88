"""Keys and values in pages on the GPU: rows written, pages copied, attention
of one token per row, each against a plain implementation in 64 bits
(tests/_paged.py derives attention's tolerances)."""
import numpy as np
import pytest
import torch

from _paged import DTYPES, attend, gather, i32, norm_tol, pool, tables
from rusty_whisper_amd import _abi as A

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _device():
    A.init(0)
    torch.cuda.init()


def run(pages, q, table, lens, max_len, layer=0, seq=None, **kw):
    rows, hq = q.shape[0], q.shape[1] // pages.st.head_size
    out = torch.full((rows, q.shape[1]), float("nan"), device="cuda")
    A.paged_attention_dev(pages, layer, q, rows, hq, i32(table), i32(lens), max_len, out,
                          seq=None if seq is None else i32(seq), **kw)
    torch.cuda.synchronize()
    return out


def compare(out, pages, q, table, lens, layer=0, seq=None, sigma=2.0):
    dim, page = pages.st.head_size, pages.st.page_rows
    got, qq = out.double().cpu().numpy(), q.double().cpu().numpy()
    for r, n in enumerate(lens):
        n = max(0, int(n))
        row = table[r if seq is None else seq[r]]
        K, V = gather(pages.k, pages.v, layer, row[: -(-n // page)], n)
        want, tol = attend(qq[r].reshape(-1, dim), K, V)
        g = got[r].reshape(-1, dim)
        assert np.all(np.isfinite(g)), f"row {r} of length {n}"
        bad = np.abs(g - want) > tol
        assert not bad.any(), (r, n, float(np.max(np.abs(g - want))), float(np.max(tol)))
        if n:
            rel = float(np.linalg.norm(g - want) / np.linalg.norm(want))
            assert rel <= norm_tol(sigma, dim, n), (r, n, rel, norm_tol(sigma, dim, n))


# ------------------------------------------------------------- attention

@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("dim,page", [(32, 16), (64, 16), (64, 32), (96, 64), (128, 32), (128, 256)])
@pytest.mark.parametrize("group", [1, 4])
def test_lengths(dtype, dim, page, group):
    heads = 3
    lens = [1, 2, 0, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 255, 257, 300]
    n_pages = 20 + sum(-(-n // page) for n in lens)
    P = A.KvPages(*pool(dtype, 2, n_pages, heads, page, dim, seed=dim + page))
    table = tables(lens, page, n_pages, seed=1)
    q = torch.randn(len(lens), heads * group * dim, device="cuda") * 2
    out = run(P, q, table, lens, 300, layer=1)
    compare(out, P, q, table, lens, layer=1)
    assert torch.all(out[2] == 0)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("heads,group", [(1, 1), (1, 16), (1, 17), (2, 5), (2, 7), (1, 40), (6, 2), (20, 1)])
def test_groups(dtype, heads, group):
    lens, page, dim = [70, 1, 200], 32, 64
    P = A.KvPages(*pool(dtype, 1, 16, heads, page, dim, seed=heads))
    table = tables(lens, page, 16, seed=2)
    q = torch.randn(3, heads * group * dim, device="cuda") * 2
    compare(run(P, q, table, lens, 200), P, q, table, lens)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,heads,group,dim,n", [(1, 1, 1, 64, 5000), (1, 2, 8, 128, 9999), (2, 1, 3, 96, 4097),
                                                    (40, 4, 1, 64, 700), (3, 8, 4, 128, 2049)])
def test_long_and_split(dtype, rows, heads, group, dim, n):
    page = 64
    lens = [max(0, n - 613 * i) for i in range(rows)]
    n_pages = sum(-(-x // page) for x in lens) + 1
    P = A.KvPages(*pool(dtype, 1, n_pages, heads, page, dim, seed=n))
    table = tables(lens, page, n_pages, seed=3)
    q = torch.randn(rows, heads * group * dim, device="cuda") * 2
    compare(run(P, q, table, lens, n), P, q, table, lens)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("scale", [1e-6, 1e-2, 30.0, 3e4])
def test_query_magnitudes(dtype, scale):
    """Scores from 0 to the one-key softmax; queries beyond f16's range."""
    lens, page, dim, heads = [1, 40, 333], 16, 64, 2
    P = A.KvPages(*pool(dtype, 1, 32, heads, page, dim, seed=5))
    table = tables(lens, page, 32, seed=5)
    q = torch.randn(3, heads * dim, device="cuda") * scale
    q[:, ::3] *= 1e-3  # values of unlike size in one row
    compare(run(P, q, table, lens, 333), P, q, table, lens, sigma=scale)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("size", ["largest", "small"])
def test_values_at_the_ends_of_the_range(dtype, size):
    """Weighted means of values near the type's largest are finite; small ones
    (down to 2^-60; f16's down to 2^-10, where it still has all its bits) keep
    their precision."""
    page, dim, heads, lens = 64, 64, 2, [1, 33, 3000]
    k, v = pool(dtype, 1, 64, heads, page, dim, seed=24)
    big = torch.finfo(v.dtype).max if size == "largest" else 2.0**-60 if dtype != "f16" else 2.0**-10
    v.uniform_(0.5, 1.0)
    v.copy_((v.double() * big).to(v.dtype))
    table = tables(lens, page, 64, seed=24)
    P = A.KvPages(k, v)
    q = torch.randn(3, heads * dim, device="cuda")
    compare(run(P, q, table, lens, 3000), P, q, table, lens, sigma=1.0)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_rising_scores_and_small_weights(dtype):
    """Each block of keys outweighs those before it; then one key far above
    4000 others whose weights add up."""
    page, dim, n = 32, 64, 4096
    k, v = pool(dtype, 1, n // page, 1, page, dim, seed=6)
    P = A.KvPages(k, v)
    table = np.arange(n // page, dtype=np.int32)[None]
    q = torch.zeros(1, dim, device="cuda")
    q[0, 0] = 8.0
    k[0, :, 0, :, 0] = torch.arange(n, device="cuda").reshape(-1, page).to(k.dtype) / 64
    compare(run(P, q, table, [n], n), P, q, table, [n], sigma=64.0)
    k[0, :, 0, :, 0] = 0
    k[0, 7, 0, 3, 0] = 10.0  # e^10 against 4095 of weight 1
    compare(run(P, q, table, [n], n), P, q, table, [n], sigma=10.0)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_what_is_behind_a_length_is_not_looked_at(dtype, value):
    lens, page, dim, heads = [1, 9, 16, 17, 40, 0, 200], 16, 64, 2
    n_pages = 40
    k, v = pool(dtype, 1, n_pages, heads, page, dim, seed=7)
    table = tables(lens, page, n_pages, seed=7)
    P = A.KvPages(k, v)
    held = {int(p) for i, n in enumerate(lens) for p in table[i, : -(-n // page)]}
    for p in range(n_pages):
        if p not in held:
            k[0, p], v[0, p] = value, value
    for i, n in enumerate(lens):
        if n % page:
            p = int(table[i, n // page])
            k[0, p, :, n % page :], v[0, p, :, :, n % page :] = value, value
    q = torch.randn(len(lens), heads * dim, device="cuda")
    compare(run(P, q, table, lens, 200), P, q, table, lens, sigma=1.0)


def test_lengths_are_cut_and_indexes_checked():
    page, dim, heads, n_pages = 16, 64, 2, 12
    P = A.KvPages(*pool("f16", 1, n_pages, heads, page, dim, seed=8))
    table = tables([60, 60, 60], page, n_pages, seed=8)  # 4 pages each
    q = torch.randn(8, heads * dim, device="cuda")
    seq = [0, 1, 2, 3, -1, 2, 1, 2**31 - 1]
    lens = [60, -5, 1000, 5, 5, 33, -(2**31), 7]
    out = run(P, q, table, lens, 50, seq=seq)
    seen = [50, 0, 50, 0, 0, 33, 0, 0]  # max_len; no such sequence
    compare(out, P, q, table, seen, seq=[0, 1, 2, 0, 0, 2, 1, 0], sigma=1.0)
    out = run(P, q, table, lens, 2**31 - 1, seq=seq)
    compare(out, P, q, table, [60, 0, 64, 0, 0, 33, 0, 0], seq=[0, 1, 2, 0, 0, 2, 1, 0], sigma=1.0)  # what the table holds
    # a page outside the pool holds no rows: the softmax runs over the others
    broken = table.copy()
    broken[0, 1], broken[2, 0], broken[2, 1], broken[2, 2], broken[2, 3] = n_pages, -1, n_pages, -(2**31), 2**31 - 1
    out = run(P, q[:3], broken, [60, 60, 60], 60)
    assert torch.all(out[2] == 0)
    K, V = gather(P.k, P.v, 0, table[0], 60)
    keep = np.r_[0:16, 32:60]
    want, tol = attend(q[0].double().cpu().numpy().reshape(heads, dim), K[:, keep], V[:, keep])
    assert np.all(np.abs(out[0].double().cpu().numpy().reshape(heads, dim) - want) <= tol)


def test_strides_and_places_beside_the_rows():
    page, dim, heads, group, lens = 32, 96, 2, 3, [100, 5]
    n = heads * group * dim
    P = A.KvPages(*pool("bf16", 1, 8, heads, page, dim, seed=9))
    table = tables(lens, page, 8, seed=9, width=7)
    wide = torch.randn(2, 3 * n + 4, device="cuda")
    q = wide[:, n : 2 * n]
    out = torch.full((4, n + 12), -7.0, device="cuda")
    A.paged_attention_dev(P, 0, q, 2, heads * group, i32(table), i32(lens), 100, out[1:3, 4 : 4 + n])
    torch.cuda.synchronize()
    compare(out[1:3, 4 : 4 + n], P, q, table, lens, sigma=1.0)
    assert torch.all(out[0] == -7) and torch.all(out[3] == -7)
    assert torch.all(out[:, :4] == -7) and torch.all(out[:, 4 + n :] == -7)


def test_rows_of_one_sequence_are_a_causal_prompt():
    """A prompt's tokens as rows of their own lengths, against
    rw_rocm_attention_dev on the same rows."""
    t, heads, dim, page = 37, 4, 64, 16
    n = heads * dim
    k, v, q = (torch.randn(t, n, device="cuda") for _ in range(3))
    P = A.KvPages(*pool("f32", 1, 5, heads, page, dim, seed=10, fill=float("nan")))
    table = np.array([[4, 0, 3]], np.int32)
    A.kv_write_dev(P, 0, k, v, t, i32(table), i32(np.arange(t)), seq=i32(np.zeros(t)))
    out = run(P, q, table, np.arange(1, t + 1), t, seq=np.zeros(t, np.int32))
    ref = torch.empty_like(out)
    A.attention_dev(q, k, v, t, t, n, heads, True, ref)
    torch.cuda.synchronize()
    compare(out, P, q, table, np.arange(1, t + 1), seq=np.zeros(t, np.int32), sigma=1.0)
    assert float((out - ref).abs().max()) <= 1e-5


def test_offsets_past_32_bits():
    """Pages whose first element lies beyond 2^31 (and byte beyond 2^32)."""
    page, dim, heads, n_pages, lens = 256, 128, 8, 8400, [700]
    k = torch.empty(1, n_pages, heads, page, dim, dtype=torch.float16, device="cuda")
    v = torch.empty(1, n_pages, heads, dim, page, dtype=torch.float16, device="cuda")
    assert k[0, n_pages - 4 :].storage_offset() > 2**31
    P = A.KvPages(k, v)
    table = np.array([[n_pages - 1, 3, n_pages - 3]], np.int32)
    rows = torch.randn(2, 700, heads * dim, device="cuda")
    A.kv_write_dev(P, 0, rows[0], rows[1], 700, i32(table), i32(np.arange(700)), seq=i32(np.zeros(700)))
    A.kv_copy_pages_dev(P, [3], [n_pages - 4])
    q = torch.randn(1, heads * 2 * dim, device="cuda")
    table[0, 1] = n_pages - 4
    torch.cuda.synchronize()
    assert torch.equal(k[0, n_pages - 4], rows[0, 256:512].reshape(256, heads, dim).transpose(0, 1).half())
    compare(run(P, q, table, lens, 700), P, q, table, lens, sigma=1.0)


def test_workspace_stream_and_bounds():
    page, dim, heads, lens = 64, 64, 2, [3000, 20]
    P = A.KvPages(*pool("f16", 1, 64, heads, page, dim, seed=11))
    table = tables(lens, page, 64, seed=11)
    q = torch.randn(2, heads * dim, device="cuda")
    need = A.paged_attention_workspace_size(P, 2, heads, 3000)
    ws = torch.full((need + 512,), 77, dtype=torch.uint8, device="cuda")
    ref = run(P, q, table, lens, 3000)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    out = run(P, q, table, lens, 3000, workspace=ws[256:], workspace_len=need, stream=s.cuda_stream)
    s.synchronize()
    assert torch.equal(out, ref)
    assert torch.all(ws[:256] == 77) and torch.all(ws[256 + need :] == 77)
    if need:
        with pytest.raises(A.RwError, match="workspace"):
            run(P, q, table, lens, 3000, workspace=ws, workspace_len=need - 1)


def test_more_chunks_than_one_launch_keeps():
    """A length whose chunks would be more than the most there are, beside a
    short row of the same launch."""
    page, dim, n = 256, 128, 200_000
    n_pages = -(-n // page) + 1
    P = A.KvPages(*pool("f32", 1, n_pages, 1, page, dim, seed=18))
    table = tables([n, 5], page, n_pages, seed=18)
    q = torch.randn(2, dim, device="cuda")
    compare(run(P, q, table, [n, 5], n), P, q, table, [n, 5], sigma=1.0)


def test_capacity_far_above_the_lengths():
    """max_len as a graph's program gives it: the table's capacity."""
    page, dim, heads, lens = 16, 64, 3, [0, 1, 500, 33]
    P = A.KvPages(*pool("bf16", 1, 64, heads, page, dim, seed=19))
    table = tables(lens, page, 64, seed=19, width=20_000)
    q = torch.randn(4, heads * dim, device="cuda")
    compare(run(P, q, table, lens, 20_000 * page), P, q, table, lens, sigma=1.0)


def test_a_captured_call_brings_its_workspace():
    page, dim, heads = 64, 64, 1
    P = A.KvPages(*pool("f16", 1, 64, heads, page, dim, seed=20))
    q, out = torch.randn(1, dim, device="cuda"), torch.empty(1, dim, device="cuda")
    table, lens = i32(np.arange(64)[None]), i32([4096])
    assert A.paged_attention_workspace_size(P, 1, 1, 4096) > 0
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out.zero_()
        with pytest.raises(A.RwError, match="captured call needs a workspace"):
            A.paged_attention_dev(P, 0, q, 1, 1, table, lens, 4096, out, stream=torch.cuda.current_stream().cuda_stream)


def test_two_graphs_on_one_workspace_and_eager_calls_between():
    page, dim, heads = 64, 64, 2
    P = A.KvPages(*pool("f16", 1, 130, heads, page, dim, seed=21))
    q = [torch.randn(2, heads * dim, device="cuda") for _ in range(2)]
    out = [torch.empty_like(x) for x in q]
    lens = [[4100, 9], [70, 3000]]
    table = [tables(n, page, 130, seed=i, width=65) for i, n in enumerate(lens)]
    dev = [(i32(t), i32(n)) for t, n in zip(table, lens)]
    need = A.paged_attention_workspace_size(P, 2, heads, 65 * page)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    graphs = []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            A.paged_attention_dev(P, 0, q[i], 2, heads, dev[i][0], dev[i][1], 65 * page, out[i], workspace=ws,
                                  workspace_len=need, stream=torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        for i in (0, 1, 1, 0):
            q[i].normal_()
            graphs[i].replay()
            big = torch.randn(8, heads * dim, device="cuda")  # the library's own workspace grows meanwhile
            run(P, big, np.repeat(table[0][:1], 8, 0), [4100] * 8, 4100)
            torch.cuda.synchronize()
            compare(out[i], P, q[i], table[i], lens[i], sigma=1.0)


def test_threads_on_streams_of_their_own():
    """Calls at once, each thread with its stream's own workspace."""
    import threading

    page, dim, heads, n = 64, 64, 2, 5000
    P = A.KvPages(*pool("bf16", 1, 80, heads, page, dim, seed=22))
    table = tables([n], page, 80, seed=22)
    td, ld = i32(table), i32([n])
    qs = [torch.randn(1, heads * dim, device="cuda") for _ in range(4)]
    outs = [torch.empty_like(x) for x in qs]
    torch.cuda.synchronize()
    errors = []

    def work(i):
        try:
            A.init(0)
            s = torch.cuda.Stream()
            for _ in range(50):
                A.paged_attention_dev(P, 0, qs[i], 1, heads, td, ld, n, outs[i], stream=s.cuda_stream)
            s.synchronize()
        except Exception as e:  # reported by the main thread
            errors.append(e)

    ts = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in ts], [t.join() for t in ts]
    assert not errors
    for q, out in zip(qs, outs):
        compare(out, P, q, table, [n], sigma=1.0)


def test_tensors_elsewhere_are_refused():
    P = A.KvPages(*pool("f32", 1, 2, 1, 16, 32, seed=23))
    q, out, t, n = torch.zeros(1, 32, device="cuda"), torch.empty(1, 32, device="cuda"), i32([[0]]), i32([1])
    for i in range(4):
        args = [q, t, n, out]
        args[i] = args[i].cpu()
        with pytest.raises(ValueError, match="another device"):
            A.paged_attention_dev(P, 0, args[0], 1, 1, args[1], args[2], 1, args[3])
    with pytest.raises(ValueError, match="another device"):
        A.kv_write_dev(P, 0, q.cpu(), q, 1, t, n)
    with pytest.raises(ValueError, match="different devices"):
        A.KvPages(P.k, P.v.cpu())


def test_captured_and_replayed_with_other_contents():
    """Lengths, sequences and table change between replays; eager calls of the
    library run between them."""
    page, dim, heads, cap = 32, 64, 4, 2048
    P = A.KvPages(*pool("f16", 1, 200, heads, page, dim, seed=12))
    q = torch.randn(3, heads * dim, device="cuda")
    table, lens, seq = (torch.zeros(s, dtype=torch.int32, device="cuda") for s in ((5, cap // page), (3,), (3,)))
    out = torch.empty_like(q)
    ws = torch.empty(max(1, A.paged_attention_workspace_size(P, 3, heads, cap)), dtype=torch.uint8, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        A.paged_attention_dev(P, 0, q, 3, heads, table, lens, cap, out, seq=seq, workspace=ws, workspace_len=ws.numel(),
                              stream=torch.cuda.current_stream().cuda_stream)
    rng = np.random.default_rng(12)
    for i, n in enumerate([[5, 0, 1], [2048, 1, 700], [33, 2047, 64], [0, 0, 0]]):
        sq = rng.permutation(5)[:3].astype(np.int32)
        t = np.zeros((5, cap // page), np.int32)
        t[sq] = tables(n, page, 200, seed=i, width=cap // page)
        table.copy_(torch.from_numpy(t)), lens.copy_(i32(n)), seq.copy_(i32(sq))
        q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        compare(out, P, q, t, n, seq=sq, sigma=1.0)
        eager = run(P, q, t, n, cap, seq=sq)
        assert torch.equal(eager, out)


# ----------------------------------------------------- writes and copies

@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("heads,dim,page", [(1, 32, 16), (3, 64, 32), (2, 96, 256), (5, 128, 64)])
@pytest.mark.parametrize("new,past", [(1, 0), (1, 31), (45, 9), (64, 64), (7, 250), (86, 3), (101, 130)])
def test_write(dtype, heads, dim, page, new, past):
    seqs, n = 3, heads * dim
    width = -(-(past + new) // page)
    n_pages = seqs * width + 2
    k, v = pool(dtype, 2, n_pages, heads, page, dim, seed=13, fill=-3.0)
    table = np.random.default_rng(past).permutation(n_pages)[: seqs * width].reshape(seqs, width).astype(np.int32)
    seq = np.repeat(np.array([2, 0, 1]), new)
    pos = np.tile(past + np.arange(new), seqs)
    rows = torch.randn(seqs * new, 2 * n + 8, device="cuda")
    rows[0, :4] = torch.tensor([1.0 + 2.0**-11, 65519.0, 2.0**-25, -0.0])  # roundings of the small types
    want_k, want_v = k.clone(), v.clone()
    for r in range(seqs * new):
        p, slot = int(table[seq[r], pos[r] // page]), int(pos[r] % page)
        want_k[1, p, :, slot] = rows[r, :n].reshape(heads, dim).to(k.dtype)
        want_v[1, p, :, :, slot] = rows[r, n + 4 : 2 * n + 4].reshape(heads, dim).to(k.dtype)
    A.kv_write_dev(A.KvPages(k, v), 1, rows[:, :n], rows[:, n + 4 : 2 * n + 4], seqs * new, i32(table), i32(pos),
                   seq=i32(seq))
    torch.cuda.synchronize()
    assert torch.equal(k, want_k) and torch.equal(v, want_v)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_write_values_beyond_the_type(dtype):
    """Rounded once, to nearest even, as a conversion: to infinity beyond the
    largest value, NaN stays NaN."""
    k, v = pool(dtype, 1, 1, 1, 16, 32, seed=0, fill=0.0)
    x = torch.tensor([[3.4e38, -3.4e38, 65504.0, 65520.0, float("inf"), float("nan"), 1e-45, 6e-8] * 4], device="cuda")
    A.kv_write_dev(A.KvPages(k, v), 0, x, x, 1, i32([[0]]), i32([5]))
    torch.cuda.synchronize()
    want = x[0].to(k.dtype)
    for got in (k[0, 0, 0, 5], v[0, 0, 0, :, 5]):
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[~want.isnan()], want[~want.isnan()])


def test_write_skips_what_the_table_does_not_have():
    page, heads, dim, n_pages = 16, 2, 64, 4
    k, v = pool("f32", 1, n_pages, heads, page, dim, seed=14, fill=5.0)
    table = np.array([[0, 1], [2, n_pages], [-1, 3]], np.int32)
    seq = np.array([0, 0, 0, 3, -1, 1, 1, 2, 2, 0])
    pos = np.array([-1, 32, 2**31 - 1, 0, 0, 16, 15, 0, 17, 31])
    rows = torch.randn(10, heads * dim, device="cuda")
    wk, wv = k.clone(), v.clone()
    for r, p, slot in ((6, 2, 15), (8, 3, 1), (9, 1, 15)):
        wk[0, p, :, slot] = wv[0, p, :, :, slot] = rows[r].reshape(heads, dim)
    A.kv_write_dev(A.KvPages(k, v), 0, rows, rows, 10, i32(table), i32(pos), seq=i32(seq))
    torch.cuda.synchronize()
    assert torch.equal(k, wk) and torch.equal(v, wv)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("layers,heads,dim,page,n", [(1, 1, 32, 16, 1), (3, 2, 96, 32, 5), (2, 5, 64, 16, 1200),
                                                     (2, 7, 128, 256, 33)])
def test_copy(dtype, layers, heads, dim, page, n):
    n_pages = 2 * n + 3
    k, v = pool(dtype, layers, n_pages, heads, page, dim, seed=15)
    ids = np.random.default_rng(n).permutation(n_pages)
    src, dst = ids[:n].copy(), ids[n : 2 * n]
    src[n // 2 :] = src[0]  # one page to many
    wk, wv = k.clone(), v.clone()
    s, d = torch.from_numpy(src).cuda(), torch.from_numpy(dst).cuda()
    wk[:, d], wv[:, d] = k[:, s], v[:, s]
    A.kv_copy_pages_dev(A.KvPages(k, v), src, dst)
    torch.cuda.synchronize()
    assert torch.equal(k, wk) and torch.equal(v, wv)


def test_write_and_copy_in_a_graph():
    """A captured step repeats its copies and reads its indexes at replay."""
    page, heads, dim = 16, 2, 64
    k, v = pool("f16", 2, 6, heads, page, dim, seed=16, fill=0.0)
    P = A.KvPages(k, v)
    rows = torch.randn(1, heads * dim, device="cuda")
    table, pos = i32([[3]]), i32([0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        s = torch.cuda.current_stream().cuda_stream
        A.kv_write_dev(P, 1, rows, rows, 1, table, pos, stream=s)
        A.kv_copy_pages_dev(P, [3], [5], stream=s)
    for i in range(3):
        pos.fill_(i)
        rows.normal_()
        g.replay()
        torch.cuda.synchronize()
        want = rows.reshape(heads, dim).half()
        assert torch.equal(k[1, 5, :, i], want) and torch.equal(v[1, 5, :, :, i], want)
        assert torch.equal(k[:, 5], k[:, 3]) and torch.all(k[1, 3, :, i + 1 :] == 0)


def test_host_arrays_are_refused():
    k, v = pool("f32", 1, 2, 1, 16, 32, seed=17)
    P = A.KvPages(k, v)
    host = np.zeros(4096, np.float32)
    P.st.k = (host.ctypes.data + 15) // 16 * 16
    with pytest.raises(A.RwError, match="not device memory"):
        A.kv_copy_pages_dev(P, [0], [1])

"""8-bit pages on the GPU: rows quantised as they are written, rows of every
type of pool read back, page copies, and attention of one token per row."""
import numpy as np
import pytest
import torch

from _draft import POOLS, TOP, any_pool, bytes_of, gather_any, quantized
from _paged import attend, i32, tables
from rusty_whisper_amd import _abi as A

pytestmark = pytest.mark.gpu
KINDS8 = ["i8", "e4m3"]


@pytest.fixture(scope="module", autouse=True)
def _device():
    A.init(0)
    torch.cuda.init()


def empty8(kind, layers, n_pages, heads, page, dim):
    """Every byte 0x55, every scale 7: places that a call leaves alone are told by them."""
    ks = [torch.full(s, 0x55, dtype=torch.uint8, device="cuda").view(POOLS[kind])
          for s in ((layers, n_pages, heads, page, dim), (layers, n_pages, heads, dim, page))]
    return ks + [torch.full((layers, n_pages, heads, page), 7.0, device="cuda") for _ in range(2)]


def check_written(pool, before, layer, table, seq, pos, k, v, kind, page):
    """Every byte of the pool after rows were written: theirs, and all others."""
    heads, dim = pool[0].shape[2], pool[0].shape[4]
    want = [bytes_of(x).clone().cpu().numpy() if x.element_size() == 1 else x.cpu().numpy().copy() for x in before]
    n_seqs, width = table.shape
    for x, values, scales, is_v in ((k, 0, 2, False), (v, 1, 3, True)):
        q, s = quantized(x.reshape(len(pos), heads, dim), kind)
        codes = torch.from_numpy(q).to(torch.float32).to(POOLS[kind]).view(torch.uint8).numpy()
        for r, p in enumerate(pos):
            if not (0 <= seq[r] < n_seqs) or p < 0 or p // page >= width:
                continue
            at = table[seq[r], p // page]
            if not 0 <= at < pool[0].shape[1]:
                continue
            if is_v:
                want[values][layer, at, :, :, p % page] = codes[r]
            else:
                want[values][layer, at, :, p % page] = codes[r]
            want[scales][layer, at, :, p % page] = s[r]
    for got, w in zip(pool, want):
        g = bytes_of(got).cpu().numpy()
        if g.dtype == np.uint8:
            bad = g != w
            assert not bad.any(), (int(bad.sum()), g[bad][:5], w[bad][:5])
        else:
            assert np.array_equal(g.view(np.uint32) & ~np.uint32(0), w.view(np.uint32)) or np.array_equal(g, w, equal_nan=True)


@pytest.mark.parametrize("kind", KINDS8)
@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("page", [16, 32, 128])
@pytest.mark.parametrize("heads,past,new", [(1, 0, 1), (3, 5, 1), (2, 13, 70), (5, 0, 33)])
def test_rows_into_pages_and_back(kind, dim, page, heads, past, new):
    rng = np.random.default_rng(dim + page + new)
    seqs = 3
    table = tables([past + new] * seqs, page, 3 * 12 + 2, 5)
    n_pages = 3 * 12 + 2
    pool = empty8(kind, 2, n_pages, heads, page, dim)
    before = [x.clone() for x in pool]
    n = heads * dim
    seq, pos = np.repeat(np.arange(seqs), new), np.tile(past + np.arange(new), seqs)
    order = rng.permutation(len(pos)) if new > 1 and heads == 2 else np.arange(len(pos))
    seq, pos = seq[order], pos[order]
    qkv = (rng.standard_normal((len(pos), 3 * n)) * rng.uniform(0.01, 30, (len(pos), 1))).astype(np.float32)
    d = torch.from_numpy(qkv).cuda()
    pages = A.KvPages(*pool)
    A.kv_write_dev(pages, 1, d[:, n : 2 * n], d[:, 2 * n :], len(pos), i32(table), i32(pos), seq=i32(seq))
    check_written(pool, before, 1, table, seq, pos, qkv[:, n : 2 * n], qkv[:, 2 * n :], kind, page)
    out = torch.full((len(pos), 2 * n + 8), -3.0, device="cuda")
    A.kv_read_dev(pages, 1, out[:, :n], out[:, n + 4 : 2 * n + 4], len(pos), i32(table), i32(pos), seq=i32(seq))
    got = out.cpu().numpy()
    assert np.all(got[:, n : n + 4] == -3) and np.all(got[:, 2 * n + 4 :] == -3)
    for x, g in ((qkv[:, n : 2 * n], got[:, :n]), (qkv[:, 2 * n :], got[:, n + 4 : 2 * n + 4])):
        q, s = quantized(x.reshape(len(pos), heads, dim), kind)
        want = (q.astype(np.float32) * s[..., None]).reshape(len(pos), n)  # one rounding, as the kernel's
        assert np.array_equal(g, want)


SPECIAL = {
    "zeros": lambda x: x * 0,
    "the smallest": lambda x: x * 0 + np.float32(1e-45),
    "subnormal": lambda x: (x * 1e-40).astype(np.float32),
    "below the scale's least": lambda x: (x * 1e-38).astype(np.float32),
    "the largest": lambda x: np.where(x > 0, np.float32(3.4028235e38), np.float32(-1e38)).astype(np.float32),
    "ties": lambda x: np.resize(np.array([127, 0.5, 1.5, 2.5, -0.5, -3.5, 126.5, 63.5], np.float32), x.shape),
    "ties of e4m3": lambda x: np.resize(np.array([448, 2.0**-10, 3 * 2.0**-10, -(2.0**-10), 17, 19, -0.0302734375, 232], np.float32),
                                        x.shape),
    "one large value": lambda x: np.where(np.arange(x.shape[-1]) == 3, np.float32(1e6), x).astype(np.float32),
    "an infinity": lambda x: np.where(np.arange(x.shape[-1]) == 5, np.float32(np.inf), x).astype(np.float32),
    "a NaN": lambda x: np.where(np.arange(x.shape[-1]) == 30, np.float32(np.nan), x).astype(np.float32),
}


@pytest.mark.parametrize("kind", KINDS8)
@pytest.mark.parametrize("name", list(SPECIAL))
def test_rows_of_special_values(kind, name):
    heads, dim, page = 2, 64, 16
    rng = np.random.default_rng(3)
    base = rng.standard_normal((9, heads * dim)).astype(np.float32)
    k, v = base.copy(), rng.standard_normal((9, heads * dim)).astype(np.float32)
    # the first head only: the other's scale is its own
    k[:, :dim] = SPECIAL[name](k[:, :dim])
    v[:, dim:] = SPECIAL[name](v[:, dim:])
    table = tables([12], page, 3, 1)
    pool = empty8(kind, 1, 3, heads, page, dim)
    before = [x.clone() for x in pool]
    pos, seq = 3 + np.arange(9), np.zeros(9, np.int64)
    dk, dv = torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda()
    A.kv_write_dev(A.KvPages(*pool), 0, dk, dv, 9, i32(table), i32(pos), seq=i32(seq))
    check_written(pool, before, 0, table, seq, pos, k, v, kind, page)
    ok, ov = torch.empty_like(dk), torch.empty_like(dv)
    A.kv_read_dev(A.KvPages(*pool), 0, ok, ov, 9, i32(table), i32(pos), seq=i32(seq))
    odd = name in ("an infinity", "a NaN")
    assert torch.isnan(ok[:, :dim]).all() == odd and torch.isnan(ov[:, dim:]).all() == odd
    assert torch.isfinite(ok[:, dim:]).all() and torch.isfinite(ov[:, :dim]).all()


@pytest.mark.parametrize("kind", list(POOLS))
def test_rows_without_a_place(kind):
    """They are not written; they read as zeros."""
    heads, dim, page, n_pages = 2, 32, 16, 4
    table = np.array([[0, 1], [2, n_pages], [-1, 3]], np.int32)
    seq = np.array([0, 1, 1, 2, 2, 3, -1, 0, 0], np.int64)
    pos = np.array([5, 15, 16, 3, 31, 0, 0, 32, -1], np.int64)
    ok = [True, True, False, False, True, False, False, False, False]
    rng = np.random.default_rng(1)
    k, v = (rng.standard_normal((9, heads * dim)).astype(np.float32) for _ in range(2))
    dk, dv = torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda()
    if kind in TOP:
        pool = empty8(kind, 1, n_pages, heads, page, dim)
        before = [x.clone() for x in pool]
        A.kv_write_dev(A.KvPages(*pool), 0, dk, dv, 9, i32(table), i32(pos), seq=i32(seq))
        check_written(pool, before, 0, table, seq, pos, k, v, kind, page)
    else:
        pool = any_pool(kind, 1, n_pages, heads, page, dim, 4)
        A.kv_write_dev(A.KvPages(*pool), 0, dk, dv, 9, i32(table), i32(pos), seq=i32(seq))
    ok_k, ok_v = torch.full_like(dk, 9.0), torch.full_like(dv, 9.0)
    A.kv_read_dev(A.KvPages(*pool), 0, ok_k, ok_v, 9, i32(table), i32(pos), seq=i32(seq))
    for r in range(9):
        for got, x in ((ok_k, k), (ok_v, v)):
            g = got[r].cpu().numpy()
            if not ok[r]:
                assert np.all(g == 0), r
            elif kind in TOP:
                q, s = quantized(x[r : r + 1].reshape(1, heads, dim), kind)
                assert np.array_equal(g, (q.astype(np.float32) * s[..., None]).reshape(-1)), r
            else:
                assert np.array_equal(g, torch.from_numpy(x[r]).to(POOLS[kind]).float().numpy()), r


@pytest.mark.parametrize("kind", list(POOLS))
@pytest.mark.parametrize("heads,dim,page", [(1, 32, 16), (3, 96, 64), (5, 128, 256)])
def test_rows_read_back(kind, heads, dim, page):
    pool = any_pool(kind, 2, 7, heads, page, dim, 8)
    lens = [page + 5, 3 * page]
    table = tables(lens, page, 7, 2)
    rng = np.random.default_rng(0)
    seq = rng.integers(0, 2, 77)
    pos = np.array([rng.integers(0, lens[s]) for s in seq])
    n = heads * dim
    k, v = torch.empty(77, n, device="cuda"), torch.empty(77, n, device="cuda")
    A.kv_read_dev(A.KvPages(*pool), 1, k, v, 77, i32(table), i32(pos), seq=i32(seq))
    for s in range(2):
        K, V = gather_any(pool, 1, table[s, : -(-lens[s] // page)], lens[s])
        at = seq == s
        for got, x in ((k, K), (v, V)):
            # a value times its scale, rounded once
            assert np.array_equal(got.cpu().numpy()[at], x[:, pos[at]].transpose(1, 0, 2).reshape(-1, n).astype(np.float32))


@pytest.mark.parametrize("kind", list(POOLS))
@pytest.mark.parametrize("heads,dim,page", [(40, 32, 16), (40, 96, 64), (80, 64, 32)])
def test_many_rows_read_back(kind, heads, dim, page):
    # (what is read by 64 rows at a time): runs of rows, single ones, and some without a place
    lens = [20 * page, 13 * page + 3]
    pool = any_pool(kind, 1, 36, heads, page, dim, 4)
    table = tables(lens, page, 36, 5)
    rng = np.random.default_rng(1)
    rows = 131072 // heads + 37
    seq, pos = rng.integers(0, 2, rows), np.zeros(rows, np.int64)
    r = 0
    while r < rows:
        n = min(rows - r, int(rng.choice([1, 2, 7, 64, 100])))
        s = int(rng.integers(0, 2))
        first = int(rng.integers(0, lens[s]))
        seq[r : r + n], pos[r : r + n] = s, (first + np.arange(n)) % lens[s]
        r += n
    gone = rng.random(rows) < 0.03
    pos[gone] = -1
    n = heads * dim
    k, v = torch.empty(rows, n, device="cuda"), torch.empty(rows, n, device="cuda")
    A.kv_read_dev(A.KvPages(*pool), 0, k, v, rows, i32(table), i32(pos), seq=i32(seq))
    for s in range(2):
        K, V = gather_any(pool, 0, table[s, : -(-lens[s] // page)], lens[s])
        at = (seq == s) & ~gone
        for got, x in ((k, K), (v, V)):
            assert np.array_equal(got.cpu().numpy()[at], x[:, pos[at]].transpose(1, 0, 2).reshape(-1, n).astype(np.float32))
    assert not k.cpu().numpy()[gone].any() and not v.cpu().numpy()[gone].any()


@pytest.mark.parametrize("kind", KINDS8)
def test_page_copies_take_the_scales(kind):
    pool = any_pool(kind, 3, 9, 2, 16, 32, 3)
    before = [bytes_of(x).clone() for x in pool]
    A.kv_copy_pages_dev(A.KvPages(*pool), [0, 0, 7], [3, 8, 1])
    for got, old in zip(pool, before):
        old[:, [3, 8, 1]] = old[:, [0, 0, 7]]
        assert torch.equal(bytes_of(got), old)


def attention(pool, layer, q, n_head, table, lens, max_len, seq=None, **kw):
    out = torch.full_like(q, 5.0)
    A.paged_attention_dev(A.KvPages(*pool), layer, q, q.shape[0], n_head, i32(table), i32(lens), max_len, out,
                          seq=None if seq is None else i32(seq), **kw)
    torch.cuda.synchronize()
    return out.double().cpu().numpy()


def check_attention(pool, kind, layer, q, n_head, table, lens, seq, got):
    page, n_pages = pool[0].shape[3], pool[0].shape[1]
    for r, n in enumerate(lens):
        row = table[seq[r]]
        n = max(0, min(int(n), len(row) * page))
        K, V = gather_any(pool, layer, row[: -(-n // page)], n)
        want, tol = attend(q[r].double().cpu().numpy().reshape(n_head, -1), K, V)
        err = np.abs(got[r].reshape(n_head, -1) - want)
        assert np.all(err <= tol), (r, n, float(err.max()), float(tol[err > tol].min()))


@pytest.mark.parametrize("kind", KINDS8)
@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 256])
@pytest.mark.parametrize("heads,group", [(1, 1), (3, 4), (2, 17)])
def test_attention(kind, dim, page, heads, group):
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 0, 300, 129, -4]
    n_pages = sum(-(-max(n, 0) // page) for n in lens) + 1
    table = tables(lens, page, n_pages, 4)
    pool = any_pool(kind, 2, n_pages, heads, page, dim, 6)
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    q = torch.randn(len(lens), heads * group * dim, device="cuda", generator=g) * 2
    seq = np.random.default_rng(2).permutation(len(lens))
    lens = np.array(lens)[seq]
    got = attention(pool, 1, q, heads * group, table, lens, 300, seq)
    check_attention(pool, kind, 1, q, heads * group, table, lens, seq, got)


@pytest.mark.parametrize("kind", KINDS8)
@pytest.mark.parametrize("rows,length,heads,dim", [(1, 20011, 1, 128), (2, 9001, 2, 64), (1, 140000, 1, 32), (40, 3333, 1, 96)])
def test_attention_over_chunks(kind, rows, length, heads, dim):
    page, group = 64, 3
    rng = np.random.default_rng(length)
    lens = np.array([length] + [int(rng.integers(0, length)) for _ in range(rows - 1)])
    n_pages = int(sum(-(-n // page) for n in lens)) + 1
    table = tables(lens, page, n_pages, 4)
    pool = any_pool(kind, 1, n_pages, heads, page, dim, 6)
    q = torch.randn(rows, heads * group * dim, device="cuda") * 2
    got = attention(pool, 0, q, heads * group, table, lens, length)
    check_attention(pool, kind, 0, q, heads * group, table, lens, np.arange(rows), got)


@pytest.mark.parametrize("kind", KINDS8)
def test_what_lies_behind_a_length_has_no_effect(kind):
    heads, dim, page = 2, 64, 32
    lens = np.array([5, 33, 70])
    table = tables(lens, page, 8, 1)
    pool = any_pool(kind, 1, 8, heads, page, dim, 2)
    q = torch.randn(3, heads * dim, device="cuda")
    want = attention(pool, 0, q, heads, table, lens, 70)
    for i, n in enumerate(lens):
        last, slot = table[i, (n - 1) // page], (n - 1) % page
        for x in pool[2:]:
            x[0, last, :, slot + 1 :] = float("nan") if kind == "i8" else float("inf")
        bytes_of(pool[0])[0, last, :, slot + 1 :] = 0x7F
        bytes_of(pool[1])[0, last, :, :, slot + 1 :] = 0x7F  # e4m3: NaN
    assert np.array_equal(attention(pool, 0, q, heads, table, lens, 70), want)


@pytest.mark.parametrize("kind", KINDS8)
@pytest.mark.parametrize("size", [1e-30, 1e30, 7e35])
def test_scales_of_any_size(kind, size):
    """Values near f32's ends, keys of their own size: the means stay finite."""
    heads, dim, page, n = 1, 64, 32, 200
    table = tables([n], page, 7, 1)
    pool = any_pool(kind, 1, 7, heads, page, dim, 2)
    pool[3] *= size * (127.0 / TOP[kind])
    q = torch.randn(1, dim, device="cuda")
    got = attention(pool, 0, q, 1, table, [n], n)
    check_attention(pool, kind, 0, q, 1, table, [n], [0], got)


@pytest.mark.parametrize("kind", KINDS8)
def test_a_captured_call_replayed_with_other_contents(kind):
    heads, dim, page, rows, most = 2, 64, 64, 5, 6000
    lens = np.array([6000, 1, 0, 777, 4097])
    table = tables(lens, page, 190, 3, width=94)
    pool = any_pool(kind, 1, 190, heads, page, dim, 9)
    pages = A.KvPages(*pool)
    size = A.paged_attention_workspace_size(pages, rows, heads * 2, most)
    assert size > 0
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    q, out = torch.randn(rows, heads * 2 * dim, device="cuda"), torch.empty(rows, heads * 2 * dim, device="cuda")
    t, n = i32(table), i32(lens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        A.paged_attention_dev(pages, 0, q, rows, heads * 2, t, n, most, out, workspace=ws, workspace_len=size,
                              stream=torch.cuda.current_stream().cuda_stream)
    for turn in range(4):
        lens = np.roll(lens, turn)
        table = tables(lens, page, 190, 10 + turn, width=94)
        t.copy_(i32(table)), n.copy_(i32(lens)), q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        check_attention(pool, kind, 0, q, heads * 2, table, lens, np.arange(rows), out.double().cpu().numpy())
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        out.zero_()
        with pytest.raises(A.RwError, match="captured call needs a workspace"):
            A.paged_attention_dev(pages, 0, q, rows, heads * 2, t, n, most, out, stream=torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("kind", KINDS8)
@pytest.mark.parametrize("q_power,k_power", [(-149, 0), (-140, 0), (-134, 0), (-120, 0), (-101, 101), (-120, 120), (-40, 40), (100, -100)])
@pytest.mark.parametrize("group", [1, 20])
def test_queries_and_key_scales_of_any_size(kind, q_power, k_power, group):
    heads, dim, page, lens = 2, 64, 32, [200, 1, 77]
    table = tables(lens, page, 12, 1)
    pool = any_pool(kind, 1, 12, heads, page, dim, 2)
    pool[2] = torch.from_numpy(np.ldexp(pool[2].double().cpu().numpy(), k_power).astype(np.float32)).cuda()
    q = np.random.default_rng(7).standard_normal((3, heads * group * dim)) * 2
    q = torch.from_numpy(np.ldexp(q, q_power).astype(np.float32)).cuda()
    assert torch.any(q != 0)
    got = attention(pool, 0, q, heads * group, table, lens, 200)
    assert np.isfinite(got).all()
    check_attention(pool, kind, 0, q, heads * group, table, lens, np.arange(3), got)


@pytest.mark.parametrize("kind", KINDS8)
@pytest.mark.parametrize("power", [-140, -126, -118, -112, -100, -60, 60, 80, 100, 112])
@pytest.mark.parametrize("group,length", [(1, 200), (20, 200), (2, 9000)])
def test_value_scales_of_any_size(kind, power, group, length):
    """Of one chunk and of several; subnormal results are multiples of 2^-149 (a mean of every wavefront and chunk, its
    share of the whole, the whole: at most 6 half steps, and 2 for every chunk)."""
    dim, page = 128, 32
    table = tables([length], page, 290, 1)
    pool = any_pool(kind, 1, 290, 1, page, dim, 2)
    pool[3] = torch.from_numpy(np.ldexp(pool[3].double().cpu().numpy(), power).astype(np.float32)).cuda()
    q = torch.randn(1, group * dim, device="cuda", generator=torch.Generator("cuda").manual_seed(3)) * 2
    got = attention(pool, 0, q, group, table, [length], length)
    K, V = gather_any(pool, 0, table[0], length)
    want, tol = attend(q[0].double().cpu().numpy().reshape(group, -1), K, V)
    err = np.abs(got[0].reshape(group, -1) - want)
    assert np.all(err <= tol + (6 + 2 * 64) * 2.0**-150), (float(err.max()), float(np.abs(want).max()))

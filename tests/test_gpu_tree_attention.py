"""Attention of several new tokens per sequence on the GPU against 64 bits: trees
of drafted tokens, chunks of prompts."""
import numpy as np
import pytest
import torch

from _draft import POOLS, TOP, ancestors, any_pool, bytes_of, gather_any, trees, words
from _paged import attend, i32, norm_tol, tables
from rusty_whisper_amd import _abi as A

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _device():
    A.init(0)
    torch.cuda.init()


class Call:
    """A call's inputs: sizes[i] nodes behind past[i] rows, masks (bool
    [nodes, nodes] per tree) or None for chains."""

    def __init__(self, kind, heads, group, dim, page, past, sizes, masks, seed=0, n_words=None, gap=0):
        rng = np.random.default_rng(seed)
        self.kind, self.heads, self.group, self.dim, self.page = kind, heads, group, dim, page
        self.past, self.sizes, self.masks = np.array(past), np.array(sizes), masks
        lens = np.maximum(self.past, 0) + self.sizes
        self.n_pages = int(sum(-(-n // page) for n in lens)) + 1
        order = rng.permutation(len(lens))
        self.table = np.empty((0, 0), np.int32)
        t = tables(lens, page, self.n_pages, seed)
        self.seq = order
        self.table = np.empty_like(t)
        self.table[order] = t
        self.pool = any_pool(kind, 2, self.n_pages, heads, page, dim, seed)
        self.starts = gap + np.concatenate([[0], np.cumsum(self.sizes)])
        self.rows = int(self.starts[-1]) + gap
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.q = torch.randn(self.rows, heads * group * dim, device="cuda", generator=g) * 2
        self.max_rows, self.max_len = max(1, int(self.sizes.max())), max(1, int(lens.max()))
        if masks is None:
            self.mask = None
        else:
            w = words(masks, n_words)
            self.mask = np.zeros((self.rows, w.shape[1]), np.int32)
            self.mask[gap : gap + len(w)] = w

    def run(self, out=None, **kw):
        out = torch.full_like(self.q, 5.0) if out is None else out
        args = dict(seq=i32(self.seq), mask=None if self.mask is None else i32(self.mask))
        args.update(kw)
        A.tree_attention_dev(A.KvPages(*self.pool), 1, self.q, self.rows, self.heads * self.group, i32(self.table),
                             i32(self.starts), self.max_rows, i32(self.past), self.max_len, out, **args)
        torch.cuda.synchronize()
        return out.double().cpu().numpy()

    def check(self, got):
        G = self.heads * self.group
        done = np.zeros(self.rows, bool)
        for i, n in enumerate(self.sizes):
            past = int(self.past[i])
            total = past + int(n)
            ids = self.table[self.seq[i]][: -(-total // self.page)]
            K, V = gather_any(self.pool, 1, ids, total)
            for j in range(n):
                r = self.starts[i] + j
                seen = np.arange(total) < past
                if self.masks is None:
                    seen |= np.arange(total) <= past + j
                else:
                    seen[past:] |= self.masks[i][j]
                q = self.q[r].double().cpu().numpy().reshape(G, -1)
                want, tol = attend(q, K[:, seen], V[:, seen])
                err = np.abs(got[r].reshape(G, -1) - want)
                assert np.all(err <= tol), (i, j, past, n, float(err.max()))
                done[r] = True
        assert np.all(got[~done] == 5.0)  # rows of no tree


@pytest.mark.parametrize("kind", list(POOLS))
@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("heads,group,page", [(1, 1, 16), (2, 5, 64), (3, 3, 32)])
def test_trees(kind, dim, heads, group, page):
    rng = np.random.default_rng(dim)
    sizes = [1, 2, 13, 33, 7]
    masks = [ancestors(p) for p in trees(rng, sizes)]
    c = Call(kind, heads, group, dim, page, [0, 17, 64, 121, 5], sizes, masks, seed=dim + page)
    c.check(c.run())


@pytest.mark.parametrize("kind", list(POOLS))
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 256)])
@pytest.mark.parametrize("past,sizes", [([0], [1]), ([0], [130]), ([33, 0, 64], [40, 3, 65]), ([7, 1], [0, 19])])
def test_chunks(kind, dim, page, past, sizes):
    c = Call(kind, 2, 2, dim, page, past, sizes, None, seed=dim, gap=3)
    c.check(c.run())


@pytest.mark.parametrize("kind", list(POOLS))
def test_any_mask(kind):
    """Nodes that see nothing, all, later ones, not themselves; more words than
    nodes, fewer words than nodes."""
    rng = np.random.default_rng(5)
    sizes = [40, 70, 5]
    masks = [rng.random((n, n)) < 0.5 for n in sizes]
    masks[0][3] = False
    masks[1][0] = True
    masks[2][:] = False
    c = Call(kind, 2, 3, 64, 16, [0, 9, 31], sizes, masks, seed=2, n_words=5)
    got = c.run()
    c.check(got)
    assert np.all(got[c.starts[0] + 3] == 0)  # past 0, no node
    c = Call(kind, 2, 3, 64, 16, [0, 9, 31], sizes, masks, seed=2, n_words=1)
    for m in masks:
        m[:, 32:] = False
    c.check(c.run())


@pytest.mark.parametrize("kind", list(POOLS))
@pytest.mark.parametrize("n_trees,past,nodes,heads,dim,group", [(1, 20001, 12, 1, 128, 4), (2, 9000, 20, 2, 64, 1),
                                                               (9, 2500, 30, 1, 96, 3)])
def test_over_chunks_of_keys(kind, n_trees, past, nodes, heads, dim, group):
    rng = np.random.default_rng(nodes)
    pasts = [past] + [int(rng.integers(0, past)) for _ in range(n_trees - 1)]
    sizes = [nodes] + [int(rng.integers(1, nodes + 1)) for _ in range(n_trees - 1)]
    for masks in ([ancestors(p) for p in trees(rng, sizes)], None):
        c = Call(kind, heads, group, dim, 64, pasts, sizes, masks, seed=past)
        c.check(c.run())


@pytest.mark.parametrize("kind", list(POOLS))
@pytest.mark.parametrize("n_trees,past,nodes,heads,dim,group,page", [(1, 30000, 21, 1, 64, 4, 16), (3, 5000, 50, 2, 128, 3, 256),
                                                                    (2, 3000, 70, 1, 96, 2, 32), (2, 2500, 9, 2, 32, 8, 128)])
def test_many_queries_over_chunks_of_keys(kind, n_trees, past, nodes, heads, dim, group, page):
    """(keys and values shared by 64 or 128 queries: pages longer and shorter than their tiles)"""
    rng = np.random.default_rng(nodes)
    pasts = [past] + [int(rng.integers(0, past)) for _ in range(n_trees - 1)]
    sizes = [nodes] + [int(rng.integers(1, nodes + 1)) for _ in range(n_trees - 1)]
    for masks in ([rng.random((n, n)) < 0.3 for n in sizes], None):
        c = Call(kind, heads, group, dim, page, pasts, sizes, masks, seed=past)
        c.check(c.run())


@pytest.mark.parametrize("kind", list(POOLS))
@pytest.mark.parametrize("page", [16, 128])
def test_many_queries_with_pages_that_are_not_there(kind, page):
    """Their rows, in the middle and at the end, are not seen, whatever v's tile held."""
    n, past, nodes = 2, [300, 700], [20, 33]
    c = Call(kind, 1, 4, 64, page, past, nodes, None, seed=11)
    whole = c.table.copy()
    gone = [np.zeros(p + m, bool) for p, m in zip(past, nodes)]
    for i in range(n):
        for at in (1, (past[i] + nodes[i] - 1) // page):
            gone[i][at * page : (at + 1) * page] = True
            c.table[c.seq[i]][at] = c.n_pages if at == 1 else -1
    got = c.run()
    for i in range(n):
        K, V = gather_any(c.pool, 1, whole[c.seq[i]][: -(-(past[i] + nodes[i]) // page)], past[i] + nodes[i])
        for j in range(nodes[i]):
            r = c.starts[i] + j
            seen = (np.arange(past[i] + nodes[i]) <= past[i] + j) & ~gone[i]
            y, tol = attend(c.q[r].double().cpu().numpy().reshape(4, -1), K[:, seen], V[:, seen])
            assert np.all(np.abs(got[r].reshape(4, -1) - y) <= tol), (i, j)


def spoil(c, tree, node, what):
    """k, v (and scales) of a node's row become `what`."""
    row = int(c.past[tree]) + node
    at, slot = c.table[c.seq[tree]][row // c.page], row % c.page
    if c.kind in TOP:
        for x in c.pool[2:]:
            x[1, at, :, slot] = what
        bytes_of(c.pool[0])[1, at, :, slot] = 0x7F
        bytes_of(c.pool[1])[1, at, :, :, slot] = 0x7F
    else:
        c.pool[0][1, at, :, slot] = what
        c.pool[1][1, at, :, :, slot] = what


@pytest.mark.parametrize("kind", list(POOLS))
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_rows_that_a_node_does_not_see_may_hold_anything(kind, what):
    """Also where other nodes see them: those, and they alone, come out odd."""
    rng = np.random.default_rng(1)
    sizes = [20, 37]
    masks = [ancestors(p) for p in trees(rng, sizes)]
    c = Call(kind, 2, 2, 64, 16, [21, 40], sizes, masks, seed=3)
    want = c.run()
    spoil(c, 0, 4, what)
    spoil(c, 1, 35, what)
    got = c.run()
    for i, bad in ((0, 4), (1, 35)):
        for j in range(sizes[i]):
            r = c.starts[i] + j
            if masks[i][j][bad]:
                assert not np.isfinite(got[r]).any(), (i, j)
            else:
                assert np.array_equal(got[r], want[r]), (i, j)


@pytest.mark.parametrize("kind", list(POOLS))
def test_a_query_of_nan_is_its_own(kind):
    c = Call(kind, 1, 2, 64, 32, [50], [18], [np.tril(np.ones((18, 18), bool))], seed=4)
    want = c.run()
    c.q[7, :64] = float("nan")
    got = c.run()
    assert np.isnan(got[7, :64]).all()
    got[7, :64] = want[7, :64]
    assert np.array_equal(got, want)


@pytest.mark.parametrize("kind", ["f16", "i8"])
def test_bad_places(kind):
    """Sequences and pages that are not there, starts out of order: nothing is
    read or written outside."""
    sizes = [5, 6, 7, 8]
    masks = [np.ones((n, n), bool) for n in sizes]
    c = Call(kind, 2, 1, 64, 16, [20, 3, 40, 10], sizes, masks, seed=6)
    c.seq = np.array([0, 9, -1, 1])
    got = c.run()
    assert np.all(got[c.starts[1] : c.starts[3]] == 0)
    c.seq = np.arange(4)
    c.table[:] = c.n_pages  # no page of the pool
    assert np.all(c.run() == 0)
    c.table[:] = 0
    c.past[1] = -5
    c.past[2] = 2**31 - 1
    got = c.run()
    assert np.all(got[c.starts[1] : c.starts[2]] == 0) and np.isfinite(got).all()
    c.past[:] = 3
    c.starts = np.array([-3, 4, 2, 100, 200])  # tree 0 and 1 have no rows, tree 2 rows 2 .., tree 3 none
    got = c.run()
    assert np.all(got[:2] == 5) and not np.any(got[2 : 2 + c.max_rows] == 5) and np.all(got[2 + c.max_rows :] == 5)


def test_lengths_are_cut():
    """max_len and the table's width cut what is seen."""
    c = Call("f32", 1, 1, 64, 16, [60], [4], [np.ones((4, 4), bool)], seed=7)
    c.max_len = 40
    got = c.run()
    c2 = Call("f32", 1, 1, 64, 16, [60], [4], [np.zeros((4, 4), bool)], seed=7)
    c2.past, c2.masks = np.array([40]), [np.zeros((4, 4), bool)]
    c2.check(got)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_a_captured_call_replayed_with_other_contents(kind):
    """With a caller's workspace that two graphs share, on a stream of its own,
    the program's eager calls between the replays."""
    rng = np.random.default_rng(8)
    sizes = [17, 9]
    calls, graphs = [], []
    for k in range(2):
        masks = [ancestors(p) for p in trees(rng, sizes)]
        calls.append(Call(kind, 2, 2, 64, 32, [5000, 3000 + k], sizes, masks, seed=k))
    n_head = 4
    size = max(A.tree_attention_workspace_size(A.KvPages(*c.pool), c.rows, n_head, 2, c.max_rows, c.max_len) for c in calls)
    assert size > 0
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    stream = torch.cuda.Stream()
    outs, held = [], []
    for c in calls:
        out = torch.full_like(c.q, 5.0)
        t = dict(table=i32(c.table), starts=i32(c.starts), past=i32(c.past), seq=i32(c.seq), mask=i32(c.mask), pages=A.KvPages(*c.pool))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            A.tree_attention_dev(t["pages"], 1, c.q, c.rows, n_head, t["table"], t["starts"], c.max_rows, t["past"], c.max_len,
                                 out, mask=t["mask"], seq=t["seq"], workspace=ws, workspace_len=size, stream=stream.cuda_stream)
        outs.append(out), held.append(t), graphs.append(graph)
    for turn in range(4):
        for c, t, out, graph in zip(calls, held, outs, graphs):
            c.masks = [ancestors(p) for p in trees(rng, sizes)]
            c.mask = words(c.masks, c.mask.shape[1])
            t["mask"].copy_(i32(c.mask))
            c.q.normal_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            c.check(out.double().cpu().numpy())
            assert np.array_equal(out.double().cpu().numpy(), c.run())  # the same, eagerly


def test_two_streams_at_once():
    """The library's own workspaces are per stream."""
    rng = np.random.default_rng(9)
    calls = [Call("f16", 2, 4, 128, 64, [9000 + i], [11], [ancestors(p) for p in trees(rng, [11])], seed=i) for i in range(2)]
    want = [c.run() for c in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    outs = [torch.zeros_like(c.q) for c in calls]
    held = [dict(seq=i32(c.seq), mask=i32(c.mask)) for c in calls]
    rest = [(i32(c.table), i32(c.starts), i32(c.past)) for c in calls]
    torch.cuda.synchronize()
    for _ in range(5):
        for c, s, out, kw, (t, st, p) in zip(calls, streams, outs, held, rest):
            A.tree_attention_dev(A.KvPages(*c.pool), 1, c.q, c.rows, 8, t, st, c.max_rows, p, c.max_len, out,
                                 stream=s.cuda_stream, **kw)
    torch.cuda.synchronize()
    for w, out in zip(want, outs):
        assert np.array_equal(out.double().cpu().numpy(), w)


@pytest.mark.parametrize("kind", ["f32", "bf16", "i8", "e4m3"])
def test_values_near_the_end_of_the_range(kind):
    """Sums of weights and values pass f32's range, means do not."""
    c = Call(kind, 1, 2, 64, 32, [90], [9], None, seed=3)
    if kind in TOP:
        c.pool[3] *= 1e36 * 127 / TOP[kind]
    else:
        c.pool[1].copy_((c.pool[1].float() * 8e37).to(POOLS[kind]))
    got = c.run()
    assert np.isfinite(got).all()
    c.check(got)


def test_rows_at_a_distance():
    """q and out as column blocks of wider rows."""
    c = Call("bf16", 2, 2, 64, 32, [70, 5], [9, 4], None, seed=3)
    want = c.run()
    wide = torch.full((c.rows, 3 * 256 + 4), 5.0, device="cuda")
    wide[:, 256:512] = c.q
    out = torch.full((c.rows, 256 + 12), 5.0, device="cuda")
    c.q = wide[:, 256:512]
    got = c.run(out=out[:, 4:260])
    assert np.array_equal(got, want)
    assert torch.all(out[:, :4] == 5) and torch.all(out[:, 260:] == 5)


@pytest.mark.parametrize("kind", list(POOLS))
@pytest.mark.parametrize("nodes", [3, 50])
def test_pages_behind_4_gib(kind, nodes):
    """The same pages at the far end of a large pool: the same bits."""
    c = Call(kind, 1, 2, 128, 128, [700, 90], [nodes, nodes], None, seed=12)
    want = c.run()
    small, size = c.pool, bytes_of(c.pool[0]).element_size()
    far = 2**32 // (128 * 128 * size) + 50  # pages of a layer
    c.pool = [torch.empty((x.shape[0], far) + tuple(x.shape[2:]), dtype=x.dtype, device="cuda") for x in small]
    for big, x in zip(c.pool, small):
        bytes_of(big)[:, far - c.n_pages :] = bytes_of(x)
    c.table = c.table + np.int32(far - c.n_pages)
    assert np.array_equal(c.run(), want)
    # ... and rows read back from there
    rows = 790
    k, v = (torch.empty(rows, 128, device="cuda") for _ in range(2))
    A.kv_read_dev(A.KvPages(*c.pool), 1, k, v, rows, i32(c.table), i32(np.arange(rows) % 90), seq=i32(np.arange(rows) % 2))
    K, V = gather_any(small, 1, c.table[1, : 1] - np.int32(far - c.n_pages), 90)
    at = np.arange(rows) % 2 == 1
    for got, x in ((k, K), (v, V)):
        assert np.array_equal(got.cpu().numpy()[at], x[:, np.arange(rows)[at] % 90].transpose(1, 0, 2).reshape(-1, 128).astype(np.float32))


def scaled_by(x, power):
    """x times 2^power, rounded once to f32 (subnormal values too)."""
    return torch.from_numpy(np.ldexp(x.double().cpu().numpy(), power).astype(np.float32)).cuda()


@pytest.mark.parametrize("kind", list(POOLS))
@pytest.mark.parametrize("power", [-149, -140, -134, -127, -120, -104, -60, 60, 100])
@pytest.mark.parametrize("nodes", [3, 40])
def test_queries_of_any_size(kind, power, nodes):
    """Finite ones down to f32's smallest; the ends of rows lie inside tiles."""
    for masks in (None, [np.eye(nodes, dtype=bool)]):
        c = Call(kind, 1, 2, 64, 16, [41], [nodes], masks, seed=power % 97)
        if power > 0:  # (keys of zero, so that scores stay in range)
            c.pool[0].zero_() if kind not in TOP else bytes_of(c.pool[0]).zero_()
        c.q = scaled_by(c.q, power)
        assert torch.any(c.q != 0)
        got = c.run()
        assert np.isfinite(got).all()
        c.check(got)


@pytest.mark.parametrize("kind", list(TOP))
@pytest.mark.parametrize("power", [-116, -90, -40, 40, 90, 101, 112, 120])
@pytest.mark.parametrize("nodes", [3, 40])
def test_key_scales_of_any_size(kind, power, nodes):
    """Keys of 2^power of the usual size and queries of 2^-power of theirs: the scores are the usual ones."""
    for masks in (None, [np.eye(nodes, dtype=bool)]):
        c = Call(kind, 1, 2, 64, 16, [41], [nodes], masks, seed=5)
        c.pool[2] = scaled_by(c.pool[2], power)
        c.q = scaled_by(c.q, -power)
        got = c.run()
        assert np.isfinite(got).all()
        c.check(got)


@pytest.mark.parametrize("kind", list(POOLS))
@pytest.mark.parametrize("page", [16, 32, 128])
@pytest.mark.parametrize("nodes", [3, 40])
@pytest.mark.parametrize("dim", [64, 128])
def test_an_infinity_beside_a_page_that_is_not_there(kind, page, nodes, dim):
    """It stays visible to those who see it, however many they are."""
    past, row, value = 3 * page + 70, 5, 7
    c = Call(kind, 1, 2, dim, page, [past], [nodes], None, seed=4)
    whole = c.table[0].copy()
    gone = np.zeros(past + nodes, bool)
    gone[page : 2 * page] = True
    c.table[0, 1] = c.n_pages
    at = whole[0]
    if kind == "i8":  # (no code for one: a scale)
        c.pool[3][1, at, :, row] = float("nan")
        odd = slice(None)
    else:
        if kind == "e4m3":
            bytes_of(c.pool[1])[1, at, :, value, row] = 0x7F
        else:
            c.pool[1][1, at, :, value, row] = float("inf")
        odd = value
    got = c.run().reshape(nodes, 2, dim)
    assert not np.isfinite(got[:, :, odd]).any()
    if odd == value:
        K, V = gather_any(c.pool, 1, whole[: -(-(past + nodes) // page)], past + nodes)
        V[:, row, value] = 0
        for j in range(nodes):
            seen = (np.arange(past + nodes) <= past + j) & ~gone
            want, tol = attend(c.q[j].double().cpu().numpy().reshape(2, -1), K[:, seen], V[:, seen])
            rest = np.arange(dim) != value
            assert np.all(np.abs(got[j] - want)[:, rest] <= tol[:, rest]), j


@pytest.mark.parametrize("kind", ["f32", "f16", "i8"])
@pytest.mark.parametrize("nodes", [7, 40])
def test_starts_at_the_ends_of_their_range(kind, nodes):
    """Trees whose rows end before they begin, however far, have none."""
    c = Call(kind, 2, 1, 64, 16, [20, 3, 40], [nodes] * 3, [np.ones((nodes, nodes), bool)] * 3, seed=6)
    for a, b in ((1, -(2**31)), (1, -(2**31) + 1), (2, -(2**31)), (2**31 - 1, -(2**31)), (2**31 - 1, 0)):
        c.starts = np.array([a, b, 3, 3 + nodes])
        got = c.run()
        first = 3 if b < 0 else b  # (rows b .. 2 are the second tree's)
        assert np.all(got[:first] == 5) and np.all(got[3 + nodes :] == 5), (a, b)
        assert np.isfinite(got).all() and not np.any(got[first : 3 + nodes] == 5), (a, b)


# Up to 16 queries a key head: every type of pool straight from memory.
SMALL = [(1, [13, 1, 0, 16, 5], [0, 17, 40, 121, 300]), (4, [4, 1, 3, 2], [70, 0, 255, 16]), (8, [2, 1], [33, 90])]


def small_masks(rng, sizes):
    """Ancestors; any bits, with a node that sees nothing and one that sees all; chains."""
    some = [rng.random((n, n)) < 0.4 for n in sizes]
    some[0][-1] = False
    some[-1][0] = True
    return [ancestors(p) if n else np.zeros((0, 0), bool) for n, p in zip(sizes, trees(rng, sizes))], some, None


@pytest.mark.parametrize("kind", list(POOLS))
@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("group,sizes,past", SMALL)
def test_few_queries_of_trees(kind, dim, page, group, sizes, past):
    for masks in small_masks(np.random.default_rng(dim + page), sizes):
        c = Call(kind, 2, group, dim, page, past, sizes, masks, seed=dim + page, gap=2)
        c.check(c.run())


@pytest.mark.parametrize("kind", list(POOLS))
@pytest.mark.parametrize("dim,page", [(32, 256), (64, 16), (96, 16), (128, 128)])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_few_queries_of_which_not_all_see_an_odd_row(kind, dim, page, what):
    rng = np.random.default_rng(3)
    sizes, past = [13, 16], [21, 60]
    masks = [ancestors(p) for p in trees(rng, sizes)]
    c = Call(kind, 2, 1, dim, page, past, sizes, masks, seed=3)
    want = c.run()
    bad = [int(np.argmin(np.abs(m.sum(0) - m.shape[0] / 3))) for m in masks]  # a third of them see it
    for i, b in enumerate(bad):
        assert 0 < masks[i][:, b].sum() < sizes[i]
        spoil(c, i, b, what)
    got = c.run()
    for i, b in enumerate(bad):
        for j in range(sizes[i]):
            r = c.starts[i] + j
            if masks[i][j][b]:
                assert not np.isfinite(got[r]).any(), (i, j)
            else:
                assert np.array_equal(got[r], want[r]), (i, j)


@pytest.mark.parametrize("kind", list(POOLS))
@pytest.mark.parametrize("page,dim", [(16, 32), (16, 128), (32, 96), (128, 64)])
@pytest.mark.parametrize("masked", [False, True])
def test_few_queries_with_pages_that_are_not_there(kind, page, dim, masked):
    rng = np.random.default_rng(page)
    past, nodes = [300, 2 * page + 5], [4, 3]
    masks = [rng.random((n, n)) < 0.6 for n in nodes] if masked else None
    c = Call(kind, 1, 4, dim, page, past, nodes, masks, seed=11)
    whole = c.table.copy()
    gone = [np.zeros(p + m, bool) for p, m in zip(past, nodes)]
    for i in range(2):
        for at in (1, (past[i] + nodes[i] - 1) // page):
            gone[i][at * page : (at + 1) * page] = True
            c.table[c.seq[i]][at] = c.n_pages if at == 1 else -1
    got = c.run()
    for i in range(2):
        total = past[i] + nodes[i]
        K, V = gather_any(c.pool, 1, whole[c.seq[i]][: -(-total // page)], total)
        for j in range(nodes[i]):
            r = c.starts[i] + j
            seen = np.arange(total) <= past[i] + j
            if masked:
                seen[past[i] :] = masks[i][j]
            seen &= ~gone[i]
            y, tol = attend(c.q[r].double().cpu().numpy().reshape(4, -1), K[:, seen], V[:, seen])
            assert np.all(np.abs(got[r].reshape(4, -1) - y) <= tol), (i, j)


@pytest.mark.parametrize("kind", list(POOLS))
@pytest.mark.parametrize("dim,page", [(32, 16), (64, 256), (96, 64), (128, 16)])
@pytest.mark.parametrize("group,sizes,past", [(1, [13], [9001]), (4, [4, 2, 4], [9000, 4007, 20]), (16, [1, 1], [5000, 700])])
def test_few_queries_of_trees_over_chunks_of_keys(kind, dim, page, group, sizes, past):
    for masks in small_masks(np.random.default_rng(dim), sizes):
        c = Call(kind, 1, group, dim, page, past, sizes, masks, seed=dim)
        assert A.tree_attention_workspace_size(A.KvPages(*c.pool), c.rows, group, len(sizes), c.max_rows, c.max_len) > 0
        c.check(c.run())


@pytest.mark.parametrize("kind", list(POOLS))
@pytest.mark.parametrize("power", [-140, -126, -118, -112, -100, -60, 60, 80, 100, 112])
@pytest.mark.parametrize("nodes", [3, 40])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 128)])
def test_values_of_any_size(kind, power, nodes, dim, page):
    """Down to where results are subnormal: there they are rounded to multiples of 2^-149, a wavefront's mean
    once, its share of the whole once (up to four of them), the whole once: 6 half steps.  Sums of weights and values
    that have no scale are subnormal themselves: one half step more for each of n products and, for tiles of 16 keys at
    least, for a rescaling of the sum (weights' sum is 1 at least, so dividing makes none of these larger)."""
    if kind == "f16":
        power = max(-14, min(power, 12))
    c = Call(kind, 1, 2, dim, page, [141], [nodes], None, seed=8)
    i = 3 if kind in TOP else 1
    c.pool[i] = scaled_by(c.pool[i], power).to(c.pool[i].dtype)
    got = c.run()
    K, V = gather_any(c.pool, 1, c.table[0], 141 + nodes)
    for j in range(nodes):
        n = 141 + j + 1
        want, tol = attend(c.q[j].double().cpu().numpy().reshape(2, -1), K[:, :n], V[:, :n])
        err = np.abs(got[j].reshape(2, -1) - want)
        steps = 6 if kind in TOP else 6 + n + n / 16
        assert np.all(err <= tol + steps * 2.0**-150), (j, float(err.max()), float(np.abs(want).max()))


@pytest.mark.parametrize("kind", list(TOP))
@pytest.mark.parametrize("large,small", [(100, 0), (100, -80), (75, -90), (40, -90), (112, -60)])
@pytest.mark.parametrize("nodes", [3, 40])
def test_value_scales_of_unlike_size(kind, large, small, nodes):
    """Where the rows of large scales hold zeros, the others' values count: every weight's share of them is
    off by 2^-133 of 2^0, as those with a scale of 2^100 leave it (bf16's last place), which is in the bound's own n + 8 half steps."""
    c = Call(kind, 1, 2, 64, 16, [141], [nodes], None, seed=8)
    n = 141 + nodes
    rows = np.arange(n)
    at, slot = c.table[0][rows // 16], rows % 16
    power = np.where(rows % 5 == 0, large, small)
    c.pool[3][1, at, 0, slot] = scaled_by(torch.ones(n, device="cuda"), power) * c.pool[3][1, at, 0, slot]
    big = rows % 5 == 0
    for r in rows[big]:
        bytes_of(c.pool[1])[1, at[r], 0, :32, slot[r]] = 0
    got = c.run()
    assert np.isfinite(got).all()
    c.check(got)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("power", [-116, -60, 60, 79, 82, 100, 112, 120, 124])
@pytest.mark.parametrize("nodes", [0, 3, 40])
def test_keys_of_any_size(kind, power, nodes):
    """Keys of 2^power of the usual size and queries of 2^-power of theirs: the scores, and errors, are the usual ones.
    (nodes 0: single rows)"""
    c = Call(kind, 1, 2, 64, 32, [141], [max(nodes, 3)], None, seed=5)
    c.pool[0] = scaled_by(c.pool[0], power).to(POOLS[kind])
    c.q = scaled_by(c.q, -power)
    if nodes:
        got = c.run()
    else:
        out = torch.empty_like(c.q)
        A.paged_attention_dev(A.KvPages(*c.pool), 1, c.q, 3, 2, i32(c.table), i32([142, 143, 144]), 144, out, seq=i32([0, 0, 0]))
        torch.cuda.synchronize()
        got = out.double().cpu().numpy()
    c.check(got)
    # far below the bound, which takes all roundings to fall one way
    K, V = gather_any(c.pool, 1, c.table[0], 144)
    want = attend(c.q[0].double().cpu().numpy().reshape(2, -1), K[:, :142], V[:, :142])[0]
    sigma = float(np.std(c.q[0].double().cpu().numpy()) * np.std(K))
    assert np.linalg.norm(got[0].reshape(2, -1) - want) <= norm_tol(sigma, 64, 142) * np.linalg.norm(want)

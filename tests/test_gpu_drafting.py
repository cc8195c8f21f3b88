"""What becomes of drafted tokens on the GPU: the accepted path and its rows; and
a program that drafts, samples, accepts and keeps its cache in any type of pages."""
import numpy as np
import pytest
import torch

from _draft import POOLS, TOP, accept, ancestors, any_pool, bytes_of, quantized, sample, trees, words
from _paged import attend, i32, tables
from rusty_whisper_amd import _abi as A

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _device():
    A.init(0)
    torch.cuda.init()


def accepted(tokens, parent, sampled, starts, most, **kw):
    n = len(starts) - 1
    kept = torch.full((n, most), 99, dtype=torch.int32, device="cuda")
    count, nxt = (torch.full((n,), 99, dtype=torch.int32, device="cuda") for _ in range(2))
    A.tree_accept_dev(i32(tokens), i32(parent), i32(sampled), len(tokens), i32(starts), most, kept, count, nxt, **kw)
    torch.cuda.synchronize()
    return kept.cpu().numpy(), count.cpu().numpy(), nxt.cpu().numpy().view(np.uint32)


@pytest.mark.parametrize("sizes", [[1], [0, 5, 0], [64, 65, 1, 13], [700, 3], [1024, 1025, 3000]], ids=str)
@pytest.mark.parametrize("vocab", [2, 50])
def test_accepted_paths(sizes, vocab):
    """Few tokens: several children of a node may hold its sample; the first counts."""
    rng = np.random.default_rng(len(sizes) + vocab)
    ps = trees(rng, sizes)
    starts = np.concatenate([[0], np.cumsum(sizes)])
    total = int(starts[-1])
    tokens, sampled = rng.integers(0, vocab, total), rng.integers(0, vocab, total)
    parent = np.concatenate([np.array(p, np.int64) for p in ps]) if total else np.zeros(0, np.int64)
    most = max(sizes) + 2
    kept, count, nxt = accepted(tokens, parent, sampled, starts, most)
    for i, n in enumerate(sizes):
        a = starts[i]
        path, follows = accept(tokens[a : a + n], parent[a : a + n], sampled[a : a + n])
        assert count[i] == len(path) and nxt[i] == follows
        assert kept[i].tolist() == path + [-1] * (most - len(path))


def test_long_paths_and_odd_parents():
    n = 1500  # a chain that is accepted to its end
    tokens = np.arange(n) + 5
    kept, count, nxt = accepted(tokens, np.arange(n) - 1, tokens + 1, [0, n], n)
    assert count[0] == n and nxt[0] == n + 5 and np.array_equal(kept[0], np.arange(n))
    kept, count, nxt = accepted(tokens, np.arange(n) - 1, tokens + 1, [0, n], 100)  # nodes from max_rows on are left out
    assert count[0] == 100 and nxt[0] == 105
    # parents that come later, that are the node itself or no node: those children are never reached
    tokens, sampled = np.array([1, 2, 2, 2, 2]), np.full(5, 2)
    kept, count, _ = accepted(tokens, np.array([-1, 1, 4, 77, 0]), sampled, [0, 5], 5)
    assert kept[0].tolist() == [0, 4, -1, -1, -1] and count[0] == 2
    kept, count, nxt = accepted(tokens, np.zeros(5), sampled, [-1, 3, 2, 9], 5)  # starts that do not fit
    assert count.tolist() == [0, 0, 1] or count.tolist()[:2] == [0, 0]


@pytest.mark.parametrize("kind", list(POOLS))
@pytest.mark.parametrize("heads,dim,page,layers", [(1, 32, 16, 1), (3, 64, 32, 2), (5, 96, 16, 3), (2, 128, 256, 2)])
def test_kept_rows(kind, heads, dim, page, layers):
    rng = np.random.default_rng(dim)
    past, sizes = [0, 13, 31, 7], [40, 1, 35, 20]
    keeps = [[0, 1, 5, 6, 17, 18, 19, 20, 21, 30, 39], [0], [0, 34], [0, 1, 2]]
    lens = np.add(past, sizes)
    n_pages = int(sum(-(-n // page) for n in lens)) + 1
    seq = np.array([2, 0, 3, 1])
    t = tables(lens, page, n_pages, 3)
    table = np.empty_like(t)
    table[seq] = t
    pool = any_pool(kind, layers, n_pages, heads, page, dim, 5)
    want = [bytes_of(x).clone() for x in pool]
    for i, path in enumerate(keeps):
        rows = [past[i] + j for j in path]
        for x, is_v in zip(want, (False, True, False, False)):
            old = x.clone()
            for j, r in enumerate(rows):
                to = past[i] + j
                a, b = t[i, r // page], t[i, to // page]
                if is_v:
                    x[:, b, :, :, to % page] = old[:, a, :, :, r % page]
                else:
                    x[:, b, :, to % page] = old[:, a, :, r % page]
    kept = np.full((4, 12), -1)
    for i, path in enumerate(keeps):
        kept[i, : len(path)] = path
    A.kv_keep_rows_dev(A.KvPages(*pool), i32(table), i32(past), i32(kept), i32([len(p) for p in keeps]), seq=i32(seq))
    for got, w in zip(pool, want):
        assert torch.equal(bytes_of(got).view(torch.uint8), w.view(torch.uint8))


@pytest.mark.parametrize("kind", ["f32", "i8"])
def test_rows_that_cannot_be_kept(kind):
    """Entries without a place are skipped; counts are cut; other sequences stay."""
    table = np.array([[0, 1], [2, 9], [-1, 3]], np.int32)
    pool = any_pool(kind, 1, 4, 2, 16, 32, 5)
    old = [bytes_of(x).clone() for x in pool]
    kept = [[0, 40], [0, 17], [0, 20]]  # behind the table; in a page that is not there; to a page that is not there
    A.kv_keep_rows_dev(A.KvPages(*pool), i32(table), i32([0, 1, 0]), i32(kept), i32([2, 2, 2]))
    A.kv_keep_rows_dev(A.KvPages(*pool), i32(table), i32([-7, 2**31 - 1, 0]), i32([[0, 3], [0, 2**31 - 1], [0, 1]]), i32([2, 2, -3]))
    A.kv_keep_rows_dev(A.KvPages(*pool), i32(table), i32([0]), i32([[0, 3]]), i32([2]), seq=i32([3]))
    for x, o in zip(pool, old):
        assert torch.equal(bytes_of(x), o)
    A.kv_keep_rows_dev(A.KvPages(*pool), i32(table), i32([0]), i32([[0, 3]]), i32([1000]))
    assert torch.equal(bytes_of(pool[0])[0, 0, :, 1], bytes_of(pool[0])[0, 0, :, 3])


@pytest.mark.parametrize("kind", ["f16", "e4m3"])
def test_a_captured_end_of_a_step_replayed_with_other_contents(kind):
    """Accepted paths and their rows in one graph, beside eager work on a stream of its own."""
    rng = np.random.default_rng(4)
    heads, dim, page, layers, sizes, past = 2, 64, 16, 3, [30, 17, 40], [5, 0, 22]
    lens = np.add(past, sizes)
    table = tables(lens, page, 9, 6)
    starts = np.concatenate([[0], np.cumsum(sizes)])
    total, most = int(starts[-1]), max(sizes)
    pool = any_pool(kind, layers, 9, heads, page, dim, 5)
    eager = [x.clone() for x in pool]
    dev = dict(tokens=i32(np.zeros(total)), parent=i32(np.zeros(total)), sampled=i32(np.zeros(total)), starts=i32(starts), table=i32(table),
               past=i32(past))
    made = [torch.zeros((3, most), dtype=torch.int32, device="cuda")] + [torch.zeros(3, dtype=torch.int32, device="cuda") for _ in range(2)]
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()

    def step(pages, s):
        A.tree_accept_dev(dev["tokens"], dev["parent"], dev["sampled"], total, dev["starts"], most, *made, stream=s)
        A.kv_keep_rows_dev(pages, dev["table"], dev["past"], made[0], made[1], stream=s)

    with torch.cuda.graph(graph, stream=stream):
        step(A.KvPages(*pool), stream.cuda_stream)
    for turn in range(4):
        parent = np.concatenate([np.array(p, np.int64) for p in trees(rng, sizes)])
        for name, x in (("tokens", rng.integers(0, 2, total)), ("sampled", rng.integers(0, 2, total)), ("parent", parent)):
            dev[name].copy_(i32(x))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        by_graph = [x.cpu().numpy() for x in made]
        step(A.KvPages(*eager), 0)
        torch.cuda.synchronize()
        for a, b in zip(by_graph, made):
            assert np.array_equal(a, b.cpu().numpy())
        assert by_graph[1].max() > 1  # something moved
        for a, b in zip(pool, eager):
            assert torch.equal(bytes_of(a), bytes_of(b))


LAYERS, HEADS, GROUP, DIM, PAGE, N_PAGES, VOCAB = 2, 2, 2, 64, 16, 40, 499
N = HEADS * DIM


class Program:
    """Sequences whose rows the program also keeps densely, as its pool reads them."""

    def __init__(self, kind, seed):
        self.kind, self.rng = kind, np.random.default_rng(seed)
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed)
        self.pool = any_pool(kind, LAYERS, N_PAGES, HEADS, PAGE, DIM, seed)
        for x in self.pool:
            (x.view(torch.uint8) if x.element_size() == 1 else x).fill_(0x7F if x.element_size() == 1 else float("nan"))
        self.pages = A.KvPages(*self.pool)
        self.book = A.KvBook(N_PAGES, PAGE, 8)
        self.dense = {}

    def reads(self, x):
        """x [rows, N] as the pool gives it back."""
        if self.kind not in TOP:
            return x.to(POOLS[self.kind]).double().cpu().numpy().reshape(-1, HEADS, DIM)
        q, s = quantized(x.cpu().numpy().reshape(-1, HEADS, DIM), self.kind)
        return q * s.astype(np.float64)[..., None]

    def forward(self, seqs, sizes, masks):
        """Writes the rows of every node and checks its attention: rows and table."""
        A.kv_copy_pages_dev(self.pages, *self.book.extend(seqs, sizes))
        past = np.array([self.book.len(s) - n for s, n in zip(seqs, sizes)])
        width = max(-(-self.book.len(s) // PAGE) for s in seqs)
        table = i32(self.book.table(seqs, width))
        starts = np.concatenate([[0], np.cumsum(sizes)])
        rows, most = int(starts[-1]), max(sizes)
        seq = i32(np.repeat(np.arange(len(seqs)), sizes))
        pos = i32(np.concatenate([p + np.arange(n) for p, n in zip(past, sizes)]))
        mask = None if masks is None else i32(words(masks))
        for layer in range(LAYERS):
            qkv = torch.randn(rows, N * GROUP + 2 * N, device="cuda", generator=self.gen)
            q, k, v = qkv[:, : N * GROUP], qkv[:, N * GROUP : N * GROUP + N], qkv[:, N * GROUP + N :]
            out = torch.empty(rows, N * GROUP, device="cuda")
            A.kv_write_dev(self.pages, layer, k, v, rows, table, pos, seq=seq)
            A.tree_attention_dev(self.pages, layer, q, rows, HEADS * GROUP, table, i32(starts), most, i32(past),
                                 int((past + sizes).max()), out, mask=mask)
            K, V = self.reads(k), self.reads(v)
            back = [torch.empty(rows, N, device="cuda") for _ in range(2)]
            A.kv_read_dev(self.pages, layer, *back, rows, table, pos, seq=seq)
            for b, x in zip(back, (K, V)):
                assert np.array_equal(b.cpu().numpy(), x.reshape(rows, N).astype(np.float32))
            for i, s in enumerate(seqs):
                a, n = starts[i], sizes[i]
                old = self.dense.setdefault((s, layer), (np.zeros((0, HEADS, DIM)),) * 2)
                self.dense[s, layer] = new = tuple(np.concatenate([o, x[a : a + n]]) for o, x in zip(old, (K, V)))
                for j in range(n):
                    seen = np.arange(len(new[0])) <= past[i] + j
                    if masks is not None:
                        seen[past[i] :] = masks[i][j]
                    want, tol = attend(q[a + j].double().cpu().numpy().reshape(-1, DIM), *(x[seen].transpose(1, 0, 2) for x in new))
                    got = out[a + j].double().cpu().numpy().reshape(-1, DIM)
                    assert np.all(np.abs(got - want) <= tol), (layer, i, j)
        return starts, past, table

    def step(self, seqs):
        """One tree per sequence: drafted, sampled at every node, accepted, kept."""
        sizes = self.rng.integers(1, 12, len(seqs)).tolist()
        ps = trees(self.rng, sizes)
        masks = [ancestors(p) for p in ps]
        starts, past, table = self.forward(seqs, sizes, masks)
        rows = int(starts[-1])
        logits = torch.randn(rows, VOCAB, device="cuda", generator=self.gen) * 2
        u = torch.rand(rows, device="cuda", generator=self.gen)
        sampled = torch.empty(rows, dtype=torch.int32, device="cuda")
        A.sample_tokens_dev(logits, rows, VOCAB, u, sampled, temperature=torch.full((rows,), 0.8, device="cuda"),
                            top_p=torch.full((rows,), 0.9, device="cuda"))
        got = sampled.cpu().numpy()
        want = [sample(x, float(a), float(np.float32(0.8)), 0, float(np.float32(0.9)))[0]
                for x, a in zip(logits.double().cpu().numpy(), u.cpu().numpy())]
        assert got.tolist() == want
        # drafts that often guess right
        parent = np.concatenate([np.array(p) for p in ps])
        tokens = self.rng.integers(0, VOCAB, rows)
        for i in range(len(seqs)):
            for j in range(1, sizes[i]):
                if self.rng.random() < 0.6:
                    tokens[starts[i] + j] = got[starts[i] + ps[i][j]]
        most = max(sizes)
        kept = torch.empty(len(seqs), most, dtype=torch.int32, device="cuda")
        count, nxt = (torch.empty(len(seqs), dtype=torch.int32, device="cuda") for _ in range(2))
        A.tree_accept_dev(i32(tokens), i32(parent), sampled, rows, i32(starts), most, kept, count, nxt)
        A.kv_keep_rows_dev(self.pages, table, i32(past), kept, count)
        for i, s in enumerate(seqs):
            a, n = starts[i], sizes[i]
            path, follows = accept(tokens[a : a + n], parent[a : a + n], got[a : a + n])
            assert kept[i].tolist()[: len(path)] == path and int(count[i]) == len(path) and int(nxt[i]) == follows
            self.book.truncate(s, int(past[i]) + len(path))
            at = list(range(past[i])) + [past[i] + j for j in path]
            for layer in range(LAYERS):
                self.dense[s, layer] = tuple(x[at] for x in self.dense[s, layer])


@pytest.mark.parametrize("kind", list(POOLS))
def test_a_program(kind):
    p = Program(kind, seed=11)
    seqs = p.book.add(3).tolist()
    p.forward(seqs, [37, 5, 16], None)  # prompts
    p.forward([seqs[0], seqs[2]], [20, 3], None)  # the rest of two of them
    for _ in range(6):
        p.step(seqs)
    child = int(p.book.fork([seqs[1]])[0])  # pages shared until one grows
    for layer in range(LAYERS):
        p.dense[child, layer] = p.dense[seqs[1], layer]
    for _ in range(3):
        p.step([seqs[1], child, seqs[0]])
    p.book.release([seqs[2], seqs[0]])
    A.kv_copy_pages_dev(p.pages, *p.book.compact())
    p.step([child, seqs[1]])


def test_trees_that_end_before_they_begin_or_behind_the_rows():
    rng = np.random.default_rng(2)
    n = 1500  # (past what is walked in LDS)
    tokens, sampled = rng.integers(0, 2, n), rng.integers(0, 2, n)
    parent = np.concatenate([np.array(p, np.int64) for p in trees(rng, [n])])
    for starts, most in (([-1, 3, 2, 9], 5), ([1, -(2**31), 2, 9], 8), ([1, -(2**31) + 1, 0, 2000], 2000), ([2**31 - 1, -(2**31), 4, 900], 900),
                         ([n - 3, -(2**31), n - 5, n + 7], 2000), ([n, 0, n, n + 1], 3)):
        kept, count, nxt = accepted(tokens, parent, sampled, starts, most)
        for i, (a, b) in enumerate(zip(starts, starts[1:])):
            b = min(b, n, a + most)
            path, follows = ([], 0xFFFFFFFF) if a < 0 or b <= a else accept(tokens[a:b], parent[a:b], sampled[a:b])
            assert count[i] == len(path) and nxt[i] == follows, (starts, i)
            assert kept[i].tolist() == path + [-1] * (most - len(path)), (starts, i)
    # two trees without rows, one that the call's rows cut
    tokens, sampled = np.array([1, 2, 2, 2, 2]), np.full(5, 2)
    kept, count, nxt = accepted(tokens, np.zeros(5), sampled, [-1, 3, 2, 9], 5)
    path, follows = accept(tokens[2:], np.zeros(3), sampled[2:])
    assert count.tolist() == [0, 0, len(path)] and nxt.tolist() == [0xFFFFFFFF, 0xFFFFFFFF, follows]
    assert kept.tolist() == [[-1] * 5, [-1] * 5, path + [-1] * (5 - len(path))]

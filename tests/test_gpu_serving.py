"""The paged cache, its attention, its book and the token scores as a serving
program uses them together: prompts of unlike lengths, steps of one token per
sequence, forks that then grow apart, ended sequences, a compaction, rows
dropped again.  Every step's attention is compared with dense copies of the
rows that the program itself keeps, every step's scores with the definition."""
import numpy as np
import pytest
import torch

from _paged import DTYPES, attend, i32, pool
from rusty_whisper_amd import _abi as A

pytestmark = pytest.mark.gpu

LAYERS, HEADS, GROUP, DIM, PAGE, N_PAGES, VOCAB = 2, 2, 2, 64, 16, 30, 997
N = HEADS * DIM


class Program:
    def __init__(self, dtype, seed):
        A.init(0)
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed)
        self.pages = A.KvPages(*pool(dtype, LAYERS, N_PAGES, HEADS, PAGE, DIM, seed, fill=float("nan")))
        self.book = A.KvBook(N_PAGES, PAGE, 12)  # four beams and their four children, and two others
        self.dense = {}  # sequence -> per layer (K rows, V rows), as the pool rounds them

    def randn(self, *shape):
        return torch.randn(*shape, device="cuda", generator=self.gen)

    def add(self, n):
        for s in self.book.add(n).tolist():
            self.dense[s] = [(torch.empty(0, N, device="cuda"),) * 2 for _ in range(LAYERS)]

    def fork(self, seqs):
        out = self.book.fork(seqs).tolist()
        for s, d in zip(seqs, out):
            self.dense[d] = list(self.dense[s])
        return out

    def release(self, seqs):
        self.book.release(seqs)
        for s in seqs:
            del self.dense[s]

    def step(self, seqs, new):
        """new[i] tokens for sequence seqs[i], each attending to what precedes
        it; returns the scores of the last token of each."""
        A.kv_copy_pages_dev(self.pages, *self.book.extend(seqs, new))
        width = max(-(-self.book.len(s) // PAGE) for s in seqs)
        table = i32(self.book.table(seqs, width))
        row_seq = np.repeat(np.arange(len(seqs)), new)
        pos = np.concatenate([self.book.len(s) - n + np.arange(n) for s, n in zip(seqs, new)])
        seq, at, lens = i32(row_seq), i32(pos), i32(pos + 1)
        rows = len(pos)
        for layer in range(LAYERS):
            qkv = self.randn(rows, N * GROUP + 2 * N)
            q, k, v = qkv[:, : N * GROUP], qkv[:, N * GROUP : N * GROUP + N], qkv[:, N * GROUP + N :]
            out = torch.empty(rows, N * GROUP, device="cuda")
            A.kv_write_dev(self.pages, layer, k, v, rows, table, at, seq=seq)
            A.paged_attention_dev(self.pages, layer, q, rows, HEADS * GROUP, table, lens, int(pos.max()) + 1, out, seq=seq)
            dt = self.pages.k.dtype
            for i, s in enumerate(seqs):
                mine = torch.from_numpy(row_seq == i).cuda()
                K, V = self.dense[s][layer]
                self.dense[s][layer] = torch.cat([K, k[mine].to(dt).float()]), torch.cat([V, v[mine].to(dt).float()])
            for r in range(rows):
                K, V = (x[: pos[r] + 1].double().cpu().numpy().reshape(-1, HEADS, DIM).transpose(1, 0, 2)
                        for x in self.dense[seqs[row_seq[r]]][layer])
                want, tol = attend(q[r].double().cpu().numpy().reshape(-1, DIM), K, V)
                got = out[r].double().cpu().numpy().reshape(-1, DIM)
                assert np.all(np.abs(got - want) <= tol), (layer, r, np.max(np.abs(got - want)))
        return self.scores(len(seqs))

    def scores(self, rows, k=3):
        logits = self.randn(rows, VOCAB) * 3
        tokens = torch.arange(rows, dtype=torch.int32, device="cuda")[:, None].contiguous()
        lp, ent = torch.empty(rows, 1, device="cuda"), torch.empty(rows, device="cuda")
        ids, top = torch.empty(rows, k, dtype=torch.int32, device="cuda"), torch.empty(rows, k, device="cuda")
        A.token_logprobs_dev(logits, rows, VOCAB, tokens, 1, lp, entropy=ent, k=k, top_ids=ids, top_logprobs=top)
        want = torch.log_softmax(logits.double(), 1)
        order = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k]
        assert torch.equal(ids.long(), order)
        # 1e-5: a few hundred half steps, at log-probs of up to 20 and sums of 997 terms
        assert torch.allclose(top.double(), want.gather(1, order), rtol=0, atol=1e-5)
        assert torch.allclose(lp.double(), want.gather(1, tokens.long()), rtol=0, atol=1e-5)
        assert torch.allclose(ent.double(), -(want.exp() * want).sum(1), rtol=0, atol=1e-5)
        return ids.cpu().numpy(), top.cpu().numpy()


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_a_program(dtype):
    p = Program(dtype, seed=3)
    p.add(3)
    p.step([0, 1, 2], [5, 33, 16])  # prompts
    for _ in range(3):
        p.step([2, 0, 1], [1, 1, 1])
    beams = [1] + p.fork([1, 1, 1])  # beams of one sequence
    scores = np.zeros(4)
    for _ in range(14):  # past a page's end
        ids, top = p.step(beams, [1] * 4)
        total = scores[:, None] + top
        best = np.argsort(-total, axis=None)[:4]
        parents = [beams[b // top.shape[1]] for b in best]
        scores = total.reshape(-1)[best]
        children = p.fork(parents)
        p.release(beams)
        beams = children
    p.step([0, 2], [20, 1])
    with pytest.raises(A.RwError) as e:
        p.book.extend([0], N_PAGES * PAGE)
    assert e.value.code == A.RW_ENOMEM
    p.release([2] + beams[:2])
    src, dst = p.book.compact()
    assert len(src)
    A.kv_copy_pages_dev(p.pages, src, dst)
    p.step([0] + beams[2:], [1, 2, 1])
    keep = p.book.len(0) - 7  # drafted tokens that were not accepted
    p.book.truncate(0, keep)
    p.dense[0] = [(K[:keep], V[:keep]) for K, V in p.dense[0]]
    p.step([beams[3], 0], [1, 4])
    p.release(list(p.dense))
    assert p.book.info() == (N_PAGES, 0, 0)

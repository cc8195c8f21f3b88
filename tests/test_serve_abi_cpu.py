"""The refusals of the paged cache's and the token scores' entries, without a
device: every check of arguments comes before the device is looked at."""
import ctypes as C

import pytest

from rusty_whisper_amd import _abi as A

K, V, TABLE, SEQ, AT, Q, OUT = (0x10000 * (i + 1) for i in range(7))  # never read: the calls are refused


def pages(**kw):
    f = dict(dtype=A.F16, n_head=4, head_size=64, page_rows=32, n_layer=3, n_pages=10, k=K, v=V)
    f.update(kw)
    return A.RwKvPages(**f)


BAD_PAGES = [(dict(dtype=2), "dtype"), (dict(dtype=-1), "dtype"), (dict(head_size=80), "head_size"),
             (dict(head_size=0), "head_size"), (dict(head_size=256), "head_size"), (dict(page_rows=8), "page_rows"),
             (dict(page_rows=48), "page_rows"), (dict(page_rows=512), "page_rows"), (dict(page_rows=-16), "page_rows"),
             (dict(n_head=0), "n_head"), (dict(n_head=-4), "n_head"), (dict(n_layer=0), "n_layer"),
             (dict(n_layer=40000), "n_layer"), (dict(n_pages=0), "n_pages"), (dict(n_pages=2**31), "n_pages"),
             (dict(k=None), "16-byte"), (dict(v=None), "16-byte"), (dict(k=K + 8), "16-byte")]


def write(p=None, **kw):
    f = dict(layer=0, k=Q, ldk=256, v=OUT, ldv=256, rows=2, table=TABLE, ld=4, n_seqs=2, seq=SEQ, pos=AT)
    f.update(kw)
    return A.lib().rw_rocm_kv_write_dev(p if p is not None else pages(), *f.values(), None)


def attention(p=None, **kw):
    f = dict(layer=0, q=Q, ldq=512, rows=2, n_head=8, table=TABLE, ld=4, n_seqs=2, seq=SEQ, lens=AT, max_len=100, out=OUT,
             ldo=512, ws=None, ws_len=0)
    f.update(kw)
    return A.lib().rw_rocm_paged_attention_dev(p if p is not None else pages(), *f.values(), None)


def refused(rc, needle):
    assert rc == A.RW_EINVAL and needle in A.last_error(), (rc, A.last_error())


@pytest.mark.parametrize("bad,needle", BAD_PAGES, ids=lambda x: str(x))
def test_pages(bad, needle):
    p = pages(**bad)
    refused(write(p), needle)
    refused(attention(p), needle)
    a = (C.c_int32 * 1)(1)
    refused(A.lib().rw_rocm_kv_copy_pages_dev(p, a, a, 1, None), needle)
    assert A.lib().rw_rocm_paged_attention_workspace_size(p, 1, 8, 100) == 0


ROWS = [(dict(layer=3), "layer 3 of 3"), (dict(table=None), "table is NULL"), (dict(ld=0), "a table of"),
        (dict(n_seqs=0), "a table of"), (dict(n_seqs=2**31), "a table of"), (dict(seq=None, rows=3), "and no seq"),
        (dict(seq=SEQ + 2), "4-byte"), (dict(table=TABLE + 1), "4-byte")]


@pytest.mark.parametrize("bad,needle", ROWS + [
    (dict(k=None), "k is NULL"), (dict(v=None), "v is NULL"), (dict(ldk=252), "row stride"), (dict(ldv=258), "16-byte"),
    (dict(k=Q + 4), "16-byte"), (dict(v=OUT + 8), "16-byte"), (dict(pos=None), "pos is NULL"), (dict(pos=AT + 2), "4-byte"),
    (dict(rows=2**31), "rows"), (dict(ldk=2**60), "row stride")], ids=lambda x: str(x))
def test_write(bad, needle):
    refused(write(**bad), needle)


@pytest.mark.parametrize("bad,needle", ROWS + [
    (dict(q=None), "q is NULL"), (dict(out=None), "out is NULL"), (dict(ldq=508), "row stride"), (dict(ldo=514), "16-byte"),
    (dict(q=Q + 4), "16-byte"), (dict(out=OUT + 8), "16-byte"), (dict(lens=None), "len is NULL"),
    (dict(n_head=0), "n_head"), (dict(n_head=6), "n_head"), (dict(n_head=-8), "n_head"), (dict(rows=2**30), "rows"),
    (dict(max_len=2**31), "max_len")], ids=lambda x: str(x))
def test_attention(bad, needle):
    refused(attention(**bad), needle)


def test_no_rows_is_a_call_that_does_nothing():
    assert write(rows=0) == A.RW_OK
    assert attention(rows=0) == A.RW_OK
    assert A.lib().rw_rocm_kv_copy_pages_dev(pages(), None, None, 0, None) == A.RW_OK
    assert A.lib().rw_rocm_token_logprobs_dev(A.F32, None, 10, 0, 10, None, 0, None, None, 0, None, None, None, 0,
                                              None) == A.RW_OK
    refused(write(C.POINTER(A.RwKvPages)()), "pages is NULL")


def test_copies():
    def copy(src, dst):
        a, b = (C.c_int32 * len(src))(*src), (C.c_int32 * len(dst))(*dst)
        return A.lib().rw_rocm_kv_copy_pages_dev(pages(), a, b, len(src), None)

    refused(copy([0, 10], [1, 2]), "page 10 -> 2")
    refused(copy([0, 1], [-1, 2]), "page 0 -> -1")
    refused(copy([0, 1], [5, 5]), "written twice")
    refused(copy([0, 1], [2, 0]), "read and written")
    refused(copy([4], [4]), "read and written")
    refused(A.lib().rw_rocm_kv_copy_pages_dev(pages(), None, None, 2, None), "NULL")
    refused(A.lib().rw_rocm_kv_copy_pages_dev(pages(), K, V, 11, None), "11 copies")
    with pytest.raises(ValueError):
        A.kv_copy_pages_dev(type("P", (), dict(st=pages()))(), [1, 2], [3])


def scores(**kw):
    f = dict(dtype=A.F32, logits=Q, ld=100, rows=3, n_vocab=100, tokens=SEQ, n_tok=2, logprobs=OUT, entropy=AT, k=4,
             ids=TABLE, top=V, ws=None, ws_len=0)
    f.update(kw)
    return A.lib().rw_rocm_token_logprobs_dev(*f.values(), None)


@pytest.mark.parametrize("bad,needle", [
    (dict(dtype=3), "dtype"), (dict(k=33), "k = 33"), (dict(n_vocab=0), "n_vocab"), (dict(n_vocab=2**31, ld=2**31), "n_vocab"),
    (dict(rows=2**31), "rows"), (dict(n_tok=2**31), "n_tok"), (dict(logits=None), "logits"), (dict(logits=Q + 2), "logits"),
    (dict(dtype=A.F16, logits=Q + 1), "logits"), (dict(ld=99), "row stride"), (dict(tokens=None), "tokens"),
    (dict(logprobs=None), "logprobs"), (dict(ids=None), "top_ids"), (dict(top=None), "top_logprobs"),
    (dict(entropy=AT + 1), "4-byte"), (dict(tokens=SEQ + 2), "4-byte")], ids=lambda x: str(x))
def test_scores(bad, needle):
    refused(scores(**bad), needle)


def test_sizes_of_refused_calls_are_zero():
    L = A.lib()
    assert L.rw_rocm_paged_attention_workspace_size(pages(), 4, 6, 100) == 0
    assert L.rw_rocm_paged_attention_workspace_size(pages(), 0, 8, 100) == 0
    assert L.rw_rocm_token_logprobs_workspace_size(0, 100, 1) == 0
    assert L.rw_rocm_token_logprobs_workspace_size(1, 0, 1) == 0
    assert L.rw_rocm_token_logprobs_workspace_size(1, 100, 33) == 0


def test_tensors_of_another_type_are_refused():
    import torch

    f = torch.zeros(1, 2, 1, 16, 32)
    with pytest.raises(ValueError):
        A.KvPages(f, f)  # v is not transposed
    with pytest.raises(ValueError):
        A.KvPages(f, f.transpose(3, 4).half().contiguous())
    with pytest.raises(ValueError):
        A.KvPages(f, f.transpose(3, 4))  # not contiguous
    p = A.KvPages(f, f.transpose(3, 4).contiguous())
    i = torch.zeros(1, 4, dtype=torch.int32)
    with pytest.raises(ValueError, match="table"):
        A.kv_write_dev(p, 0, f[0, 0, 0], f[0, 0, 0], 1, i.long(), i[0])
    with pytest.raises(ValueError, match="pos"):
        A.kv_write_dev(p, 0, f[0, 0, 0], f[0, 0, 0], 1, i, i[0].long())
    with pytest.raises(ValueError, match="lens"):
        A.paged_attention_dev(p, 0, f[0, 0, 0], 1, 1, i, i[0, ::2], 5, f[0, 0, 0])
    with pytest.raises(ValueError, match="q"):
        A.paged_attention_dev(p, 0, f[0, 0, 0].half(), 1, 1, i, i[0], 5, f[0, 0, 0])
    with pytest.raises(ValueError, match="tokens"):
        A.token_logprobs_dev(f[0, 0, 0], 16, 32, i.long(), 1, f)


def test_workspace_of_a_longer_call_is_no_smaller():
    """A caller sizes its workspace by the longest length it will see."""
    import random

    rng = random.Random(4)
    L = A.lib()
    for _ in range(300):
        p = pages(dtype=rng.choice((A.F32, A.F16, A.BF16)), n_head=rng.choice((1, 3, 8, 20)),
                  head_size=rng.choice((32, 64, 96, 128)))
        rows, heads = rng.choice((1, 2, 7, 61, 300, 5000)), p.n_head * rng.choice((1, 4, 17))
        lens = sorted(int(2 ** rng.uniform(0, 31)) for _ in range(12))
        sizes = [L.rw_rocm_paged_attention_workspace_size(p, rows, heads, n) for n in lens]
        assert sizes == sorted(sizes), (rows, heads, lens, sizes)
    for rows, n in ((1, 51866), (5, 51866), (2100, 51866), (3, 2**31 - 1)):
        sizes = [L.rw_rocm_token_logprobs_workspace_size(rows, n, k) for k in range(33)]
        assert sizes == sorted(sizes)

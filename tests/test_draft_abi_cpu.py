"""The refusals of the entries for 8-bit pages, drafted tokens and sampling,
without a device: every check of arguments comes before the device is looked at."""
import ctypes as C

import pytest
import torch

from rusty_whisper_amd import _abi as A
from test_serve_abi_cpu import AT, BAD_PAGES, K, OUT, Q, ROWS, SEQ, TABLE, V, attention, pages, refused, write

KS, VS, X, Y = 0x100000, 0x110000, 0x120000, 0x130000


def pages8(**kw):
    return pages(**{**dict(dtype=A.I8, k_scale=KS, v_scale=VS), **kw})


def read(p=None, **kw):
    f = dict(layer=0, k=Q, ldk=256, v=OUT, ldv=256, rows=2, table=TABLE, ld=4, n_seqs=2, seq=SEQ, pos=AT)
    f.update(kw)
    return A.lib().rw_rocm_kv_read_dev(p if p is not None else pages(), *f.values(), None)


def tree(p=None, **kw):
    f = dict(layer=0, q=Q, ldq=512, rows=9, n_head=8, table=TABLE, ld=4, n_seqs=2, seq=SEQ, n_trees=2, starts=X, max_rows=5,
             past=AT, mask=Y, n_words=1, max_len=100, out=OUT, ldo=512, ws=None, ws_len=0)
    f.update(kw)
    return A.lib().rw_rocm_tree_attention_dev(p if p is not None else pages(), *f.values(), None)


def accept(**kw):
    f = dict(tokens=Q, parent=X, sampled=Y, rows=9, starts=SEQ, n_trees=2, max_rows=5, kept=OUT, n_kept=AT, next=K)
    f.update(kw)
    return A.lib().rw_rocm_tree_accept_dev(*f.values(), None)


def keep(p=None, **kw):
    f = dict(table=TABLE, ld=4, n_seqs=2, seq=SEQ, n_trees=2, past=AT, kept=X, ld_kept=5, n_kept=Y)
    f.update(kw)
    return A.lib().rw_rocm_kv_keep_rows_dev(p if p is not None else pages(), *f.values(), None)


def sample(**kw):
    f = dict(dtype=A.F32, logits=Q, ld=100, rows=3, n_vocab=100, u=X, temperature=Y, top_k=SEQ, top_p=AT, min_p=TABLE,
             tokens=OUT, logprobs=V, ws=None, ws_len=0)
    f.update(kw)
    return A.lib().rw_rocm_sample_tokens_dev(*f.values(), None)


@pytest.mark.parametrize("bad,needle", BAD_PAGES, ids=lambda x: str(x))
def test_pages(bad, needle):
    for call in (read, tree, keep):
        refused(call(pages(**bad)), needle)
    assert A.lib().rw_rocm_tree_attention_workspace_size(pages(**bad), 9, 8, 2, 5, 100) == 0


@pytest.mark.parametrize("dtype", [A.I8, A.E4M3])
@pytest.mark.parametrize("bad", [dict(k_scale=None), dict(v_scale=None), dict(k_scale=KS + 4), dict(v_scale=VS + 8)], ids=str)
def test_scales(dtype, bad):
    p = pages8(dtype=dtype, **bad)
    for call in (read, tree, keep, write, attention):
        refused(call(p), "k_scale and v_scale")
    a = (C.c_int32 * 1)(1)
    refused(A.lib().rw_rocm_kv_copy_pages_dev(p, a, a, 1, None), "k_scale and v_scale")


def test_scales_of_other_types_are_not_looked_at():
    for p in (pages(k_scale=3, v_scale=None), pages()):
        refused(read(p, k=None), "k is NULL")


@pytest.mark.parametrize("bad,needle", ROWS + [
    (dict(k=None), "k is NULL"), (dict(v=None), "v is NULL"), (dict(ldk=252), "row stride"), (dict(ldv=258), "16-byte"),
    (dict(k=Q + 4), "16-byte"), (dict(pos=None), "pos is NULL"), (dict(rows=2**31), "rows")], ids=lambda x: str(x))
def test_read(bad, needle):
    refused(read(**bad), needle)
    refused(read(pages8(), **bad), needle)
    refused(write(pages8(), **bad), needle)


@pytest.mark.parametrize("bad,needle", [b for b in ROWS if "rows" not in b[0]] + [
    (dict(seq=None, n_trees=3), "and no seq"), (dict(q=None), "q is NULL"), (dict(out=None), "out is NULL"),
    (dict(ldq=508), "row stride"), (dict(ldo=514), "16-byte"), (dict(q=Q + 4), "16-byte"), (dict(past=None), "past is NULL"),
    (dict(past=AT + 2), "4-byte"), (dict(starts=None), "starts"), (dict(starts=X + 1), "starts"), (dict(n_words=0), "a mask of"),
    (dict(mask=Y + 2), "a mask of"), (dict(n_head=6), "n_head"), (dict(n_head=0), "n_head"), (dict(rows=2**30), "rows"),
    (dict(max_len=2**31), "max_len"), (dict(n_trees=2**40), "trees"), (dict(max_rows=2**40), "trees"),
    (dict(n_trees=2**12, max_rows=2**10), "trees")], ids=lambda x: str(x))
def test_tree(bad, needle):
    refused(tree(**bad), needle)
    refused(tree(pages8(), **bad), needle)


@pytest.mark.parametrize("bad,needle", [
    (dict(tokens=None), "NULL"), (dict(parent=None), "NULL"), (dict(sampled=None), "NULL"), (dict(starts=None), "NULL"),
    (dict(kept=None), "NULL"), (dict(n_kept=None), "NULL"), (dict(next=None), "NULL"), (dict(tokens=Q + 1), "4-byte"),
    (dict(kept=OUT + 2), "4-byte"), (dict(rows=2**31), "rows"), (dict(n_trees=2**30), "trees"),
    (dict(max_rows=2**31), "trees")], ids=lambda x: str(x))
def test_accept(bad, needle):
    refused(accept(**bad), needle)


@pytest.mark.parametrize("bad,needle", [b for b in ROWS if "layer" not in b[0] and "rows" not in b[0]] + [
    (dict(seq=None, n_trees=3), "and no seq"), (dict(past=None), "past is NULL"), (dict(kept=None), "kept"),
    (dict(n_kept=None), "kept"), (dict(kept=X + 2), "kept"), (dict(ld_kept=2**31), "rows kept"),
    (dict(n_trees=2**30), "trees")], ids=lambda x: str(x))
def test_keep(bad, needle):
    refused(keep(**bad), needle)
    refused(keep(pages8(), **bad), needle)


@pytest.mark.parametrize("bad,needle", [
    (dict(dtype=A.I8), "dtype"), (dict(dtype=A.E4M3), "dtype"), (dict(dtype=3), "dtype"), (dict(n_vocab=0), "n_vocab"),
    (dict(n_vocab=2**20 + 1, ld=2**21), "n_vocab"), (dict(rows=2**31), "rows"), (dict(logits=None), "logits"),
    (dict(logits=Q + 2), "logits"), (dict(ld=99), "row stride"), (dict(u=None), "u or tokens"),
    (dict(tokens=None), "u or tokens"), (dict(u=X + 2), "4-byte"), (dict(top_k=SEQ + 1), "4-byte"),
    (dict(logprobs=V + 2), "4-byte")], ids=lambda x: str(x))
def test_sample(bad, needle):
    refused(sample(**bad), needle)


def test_logits_of_8_bits_are_refused():
    for dtype in (A.I8, A.E4M3):
        refused(A.lib().rw_rocm_token_logprobs_dev(dtype, Q, 100, 3, 100, SEQ, 2, OUT, AT, 0, None, None, None, 0, None), "dtype")


def test_calls_that_do_nothing():
    assert read(rows=0) == A.RW_OK
    assert tree(rows=0) == A.RW_OK and tree(n_trees=0) == A.RW_OK and tree(max_rows=0) == A.RW_OK
    assert accept(n_trees=0) == A.RW_OK
    assert keep(n_trees=0) == A.RW_OK and keep(ld_kept=0) == A.RW_OK
    assert sample(rows=0) == A.RW_OK


def test_workspaces():
    """No smaller for a longer call, 0 for one that is refused."""
    import random

    L, rng = A.lib(), random.Random(6)
    for _ in range(300):
        p = pages8(dtype=rng.choice((A.F32, A.F16, A.BF16, A.I8, A.E4M3)), n_head=rng.choice((1, 3, 8, 20)),
                   head_size=rng.choice((32, 64, 96, 128)))
        trees, most, heads = rng.choice((1, 2, 7, 61)), rng.choice((1, 5, 64, 700)), p.n_head * rng.choice((1, 4, 17))
        lens = sorted(int(2 ** rng.uniform(0, 31)) for _ in range(12))
        sizes = [L.rw_rocm_tree_attention_workspace_size(p, trees * most, heads, trees, most, n) for n in lens]
        assert sizes == sorted(sizes)
        sizes = [L.rw_rocm_paged_attention_workspace_size(p, trees, heads, n) for n in lens]
        assert sizes == sorted(sizes)
    assert L.rw_rocm_tree_attention_workspace_size(pages(), 9, 6, 2, 5, 100) == 0
    assert L.rw_rocm_tree_attention_workspace_size(pages(), 0, 8, 2, 5, 100) == 0
    assert L.rw_rocm_sample_tokens_workspace_size(0, 100) == 0


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def pool8(dtype=torch.int8, scale=(1, 5, 4, 16)):
    return [torch.zeros(1, 5, 4, 16, 32, dtype=dtype), torch.zeros(1, 5, 4, 32, 16, dtype=dtype), torch.zeros(scale),
            torch.zeros(scale)]


def test_pools_of_tensors():
    for dtype, code in ((torch.int8, A.I8), (torch.float8_e4m3fn, A.E4M3)):
        k, v, ks, vs = pool8(dtype)
        assert A.KvPages(k, v, ks, vs).st.dtype == code
        for bad in ((None, vs), (ks, None), (ks[:, :4], vs), (ks, vs[0]), (ks.double(), vs), (ks, vs.transpose(2, 3))):
            with pytest.raises(ValueError, match="_scale"):
                A.KvPages(k, v, *bad)
    f = torch.zeros(1, 5, 4, 16, 32)
    with pytest.raises(ValueError, match="are for int8"):
        A.KvPages(f, torch.zeros(1, 5, 4, 32, 16), ks, vs)
    with pytest.raises(ValueError, match="one type"):
        A.KvPages(f.to(torch.uint8), torch.zeros(1, 5, 4, 32, 16, dtype=torch.uint8), ks, vs)


def call_tree(**kw):
    f = dict(q=torch.zeros(9, 256), table=i32(2, 3), starts=i32(3), past=i32(2), out=torch.zeros(9, 256), mask=i32(9, 1), seq=i32(2))
    f.update(kw)
    A.tree_attention_dev(A.KvPages(*pool8()), 0, f["q"], 9, 8, f["table"], f["starts"], 5, f["past"], 40, f["out"],
                         mask=f["mask"], seq=f["seq"])


def call_sample(**kw):
    f = dict(logits=torch.zeros(3, 50), u=torch.zeros(3), tokens=i32(3), temperature=torch.zeros(3), top_k=i32(3),
             top_p=torch.zeros(3), min_p=torch.zeros(3), logprobs=torch.zeros(3))
    f.update(kw)
    A.sample_tokens_dev(f["logits"], 3, 50, f["u"], f["tokens"], logprobs=f["logprobs"], temperature=f["temperature"],
                        top_k=f["top_k"], top_p=f["top_p"], min_p=f["min_p"])


def call_accept(**kw):
    f = dict(tokens=i32(9), parent=i32(9), sampled=i32(9), starts=i32(3), kept=i32(2, 5), n_kept=i32(2), following=i32(2))
    f.update(kw)
    A.tree_accept_dev(f["tokens"], f["parent"], f["sampled"], 9, f["starts"], 5, f["kept"], f["n_kept"], f["following"])


def call_keep(**kw):
    f = dict(table=i32(2, 3), past=i32(2), kept=i32(2, 5), n_kept=i32(2), seq=i32(2))
    f.update(kw)
    A.kv_keep_rows_dev(A.KvPages(*pool8()), f["table"], f["past"], f["kept"], f["n_kept"], seq=f["seq"])


def call_read(**kw):
    f = dict(k=torch.zeros(6, 128), v=torch.zeros(6, 128), table=i32(2, 3), pos=i32(6), seq=i32(6))
    f.update(kw)
    A.kv_read_dev(A.KvPages(*pool8()), 0, f["k"], f["v"], 6, f["table"], f["pos"], seq=f["seq"])


SHORT = [(call_tree, dict(q=torch.zeros(8, 256)), "q ends"), (call_tree, dict(out=torch.zeros(9, 255)), "out"),
         (call_tree, dict(starts=i32(2)), "starts has 2"), (call_tree, dict(seq=i32(1)), "seq has 1"),
         (call_tree, dict(mask=i32(8, 1)), "mask has 8"), (call_tree, dict(mask=i32(9)), "mask must be"),
         (call_tree, dict(mask=i32(9, 1).long()), "mask must be"), (call_tree, dict(past=i32(2).float()), "past"),
         (call_sample, dict(u=torch.zeros(2)), "u has 2"), (call_sample, dict(tokens=i32(2)), "tokens has 2"),
         (call_sample, dict(logprobs=torch.zeros(1)), "logprobs has 1"), (call_sample, dict(top_k=i32(2)), "top_k has 2"),
         (call_sample, dict(top_p=torch.zeros(2)), "top_p has 2"), (call_sample, dict(min_p=torch.zeros(2)), "min_p has 2"),
         (call_sample, dict(temperature=torch.zeros(2)), "temperature has 2"),
         (call_sample, dict(logits=torch.zeros(3, 49)), "logits"), (call_sample, dict(top_k=torch.zeros(3)), "top_k"),
         (call_accept, dict(tokens=i32(8)), "tokens has 8"), (call_accept, dict(parent=i32(8)), "parent has 8"),
         (call_accept, dict(sampled=i32(8)), "sampled has 8"), (call_accept, dict(starts=i32(2)), "starts has 2"),
         (call_accept, dict(kept=i32(2, 4)), "kept has 8"), (call_accept, dict(following=i32(1)), "next_tokens has 1"),
         (call_keep, dict(past=i32(1)), "past has 1"), (call_keep, dict(n_kept=i32(1)), "n_kept has 1"),
         (call_keep, dict(seq=i32(1)), "seq has 1"), (call_keep, dict(kept=i32(2, 5).long()), "kept"),
         (call_read, dict(k=torch.zeros(5, 128)), "k ends"), (call_read, dict(v=torch.zeros(6, 64)), "v"),
         (call_read, dict(pos=i32(5)), "pos has 5")]


@pytest.mark.parametrize("call,bad,needle", SHORT, ids=[f"{c.__name__}-{i}" for i, (c, _, _) in enumerate(SHORT)])
def test_tensors_that_end_too_early_are_refused(call, bad, needle):
    with pytest.raises(ValueError, match=needle):
        call(**bad)


@pytest.mark.parametrize("call", [call_tree, call_sample, call_accept, call_keep, call_read], ids=lambda c: c.__name__)
def test_tensors_that_just_suffice_reach_the_library(call):
    with pytest.raises(A.RwError):  # no device here, or tensors that are not on it
        call()


def test_accepted_paths_of_another_width_are_refused():
    """Rows of 7 nodes would be written 5 apart: the next call reads them 7 apart."""
    for kept in (i32(2, 7), i32(4, 4)):
        with pytest.raises(ValueError, match="kept must be"):
            call_accept(kept=kept)
    with pytest.raises(A.RwError):  # no device here, or tensors that are not on it
        call_accept(kept=i32(10))

"""How the serving entries' Python wrappers take tensors: which element of
which row a call reads.  On the CPU: pointers and strides are looked at, no
call is queued."""
import numpy as np
import pytest
import torch

from rusty_whisper_amd import _abi as A

H, D, ROWS = 4, 32, 6
N = H * D


def places(a, ld=None):
    """Element [row, value] as `_rows` tells the library to read it: offsets
    from the storage's start."""
    p, step = A._rows(a, ROWS, N, ld, "q", None)
    first = (p - a.untyped_storage().data_ptr()) // 4
    return [[first + r * step + i for i in range(N)] for r in range(ROWS)]


def numbered(*shape):
    """float32, element i of the storage holds i (exact below 2^24)."""
    n = 1
    for s in shape:
        n *= s
    return torch.arange(n, dtype=torch.float32).reshape(shape)


VIEWS = {
    "dense": lambda: numbered(ROWS, N),
    "columns": lambda: numbered(ROWS, 3 * N)[:, N : 2 * N],
    "every second row": lambda: numbered(2 * ROWS, N)[::2],
    "heads": lambda: numbered(ROWS, H, D),
    "heads of a fused projection": lambda: numbered(ROWS, 3 * N).view(ROWS, 3, H, D)[:, 1],
    "heads of a column block": lambda: numbered(ROWS, N + 64)[:, 64:].view(ROWS, H, D),
    "windows and steps": lambda: numbered(2, ROWS // 2, 3, H, D)[:, :, 2],
    "a dimension of one": lambda: numbered(ROWS, 3, H, D)[:, 1:2],
    "an inner dimension of one, strided": lambda: numbered(ROWS, 5, N)[:, 2:3],
}


@pytest.mark.parametrize("name", list(VIEWS))
def test_rows_are_the_tensors_own(name):
    a = VIEWS[name]()
    storage = torch.empty(0).set_(a.untyped_storage())
    assert torch.equal(storage[torch.tensor(places(a))], a.reshape(ROWS, N))


def test_one_row_and_flat_arrays():
    for a in (numbered(1, N), numbered(N), numbered(H, D), numbered(1, 1, N), numbered(7, 1, N)[3:4]):
        assert A._rows(a, 1, N, None, "q", None) == (a.data_ptr(), N)
    assert A._rows(numbered(ROWS * N), ROWS, N, None, "q", None)[1] == N  # rows one behind the other
    assert A._rows(numbered(ROWS, N + 9), ROWS, N, None, "q", None)[1] == N + 9  # the first columns of wider rows
    assert A._rows(numbered(ROWS, 2 * N), 4, N, 3 * N, "q", None)[1] == 3 * N  # the caller's own stride


@pytest.mark.parametrize("a,needle", [
    (numbered(H, ROWS, D).transpose(0, 1), "not contiguous"),  # heads before rows
    (numbered(ROWS, D, H).transpose(1, 2), "not contiguous"),
    (numbered(ROWS, N, 2)[:, :, 0], "not contiguous"),
    (numbered(ROWS, 2 * H, D)[:, ::2], "not contiguous"),
    (numbered(2, 8, N)[:, : ROWS // 2], "one distance"),
    (numbered(ROWS, 2 * H, D + 1)[:, :, :D], "not contiguous"),
    (numbered(ROWS, 2, 3 * D)[:, :, : 2 * D + 16], "not"),
], ids=["heads first", "values first", "every second value", "every second head", "parts of windows",
        "parts of heads", "more than a row"])
@pytest.mark.parametrize("ld", [None, N])
def test_other_layouts_are_refused(a, needle, ld):
    with pytest.raises(ValueError, match=needle):
        A._rows(a, ROWS, N, ld, "q", None)


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def pages():
    return A.KvPages(torch.zeros(1, 5, H, 16, D), torch.zeros(1, 5, H, D, 16))


def write(**kw):
    f = dict(k=torch.zeros(ROWS, N), v=torch.zeros(ROWS, N), table=i32(2, 3), pos=i32(ROWS), seq=i32(ROWS))
    f.update(kw)
    A.kv_write_dev(pages(), 0, f["k"], f["v"], ROWS, f["table"], f["pos"], seq=f["seq"], ldk=f.get("ldk"))


def attention(**kw):
    f = dict(q=torch.zeros(ROWS, 2 * N), table=i32(2, 3), lens=i32(ROWS), seq=i32(ROWS), out=torch.zeros(ROWS, 2 * N),
             workspace=None, workspace_len=0)
    f.update(kw)
    A.paged_attention_dev(pages(), 0, f["q"], ROWS, 2 * H, f["table"], f["lens"], 40, f["out"], seq=f["seq"],
                          workspace=f["workspace"], workspace_len=f["workspace_len"])


def scores(**kw):
    f = dict(logits=torch.zeros(ROWS, 50), tokens=i32(ROWS, 2), logprobs=torch.zeros(ROWS, 2), entropy=torch.zeros(ROWS),
             ids=i32(ROWS, 3), top=torch.zeros(ROWS, 3), workspace=None, workspace_len=0)
    f.update(kw)
    A.token_logprobs_dev(f["logits"], ROWS, 50, f["tokens"], 2, f["logprobs"], entropy=f["entropy"], k=3,
                         top_ids=f["ids"], top_logprobs=f["top"], workspace=f["workspace"],
                         workspace_len=f["workspace_len"])


SHORT = [(write, dict(k=torch.zeros(ROWS - 1, N)), "k ends"), (write, dict(v=torch.zeros(ROWS * N - 1)), "v ends"),
         (write, dict(v=torch.zeros(ROWS, 3, H, D)[: ROWS - 1, 1]), "v ends"),
         (write, dict(ldk=N + 4), "k ends"),
         (write, dict(k=torch.zeros(0, N)), "k ends"),
         (write, dict(pos=i32(ROWS - 1)), "pos has 5"), (write, dict(seq=i32(1)), "seq has 1"),
         (attention, dict(q=torch.zeros(ROWS, N)), "q"), (attention, dict(q=torch.zeros(ROWS - 1, 2 * N)), "q ends"),
         (attention, dict(out=torch.zeros(ROWS - 1, 2 * N)), "out ends"), (attention, dict(lens=i32(2)), "lens has 2"),
         (attention, dict(seq=i32(ROWS - 1)), "seq has 5"),
         (attention, dict(workspace=torch.zeros(1023, dtype=torch.uint8), workspace_len=1024), "workspace"),
         (attention, dict(workspace=torch.zeros(4, 600, dtype=torch.uint8)[:, :300], workspace_len=1024), "workspace"),
         (scores, dict(logits=torch.zeros(ROWS - 1, 50)), "logits ends"), (scores, dict(logits=torch.zeros(ROWS, 49)), "logits"),
         (scores, dict(tokens=i32(ROWS, 1)), "tokens has 6"), (scores, dict(logprobs=torch.zeros(ROWS)), "logprobs has 6"),
         (scores, dict(entropy=torch.zeros(ROWS - 1)), "entropy has 5"), (scores, dict(ids=i32(ROWS, 2)), "top_ids has 12"),
         (scores, dict(top=torch.zeros(3)), "top_logprobs has 3"),
         (scores, dict(workspace=torch.zeros(2), workspace_len=16), "workspace")]


@pytest.mark.parametrize("call,bad,needle", SHORT, ids=[f"{c.__name__}-{i}" for i, (c, _, _) in enumerate(SHORT)])
def test_tensors_that_end_too_early_are_refused(call, bad, needle):
    with pytest.raises(ValueError, match=needle):
        call(**bad)


@pytest.mark.parametrize("call", [write, attention, scores], ids=lambda c: c.__name__)
def test_tensors_that_just_suffice_reach_the_library(call):
    with pytest.raises(A.RwError):  # no device here, or tensors that are not on it
        call()


HOST = [(write, n) for n in ("k", "v", "pos", "seq")] + [(attention, n) for n in ("q", "lens", "seq", "out", "workspace")] + [
    (scores, n) for n in ("logits", "tokens", "logprobs", "entropy", "ids", "top", "workspace")]


@pytest.mark.parametrize("call,name", HOST, ids=[f"{c.__name__}-{n}" for c, n in HOST])
def test_host_arrays_are_refused(call, name):
    with pytest.raises(ValueError, match="host array"):
        call(**{name: np.zeros(4096, np.float32)})


def test_a_type_that_is_not_the_logits_own_is_refused():
    """RW_F32 for f16 logits would read twice their bytes."""
    for own in (torch.float32, torch.float16, torch.bfloat16):
        for dtype in (A.F32, A.F16, A.BF16):
            x, lp = torch.zeros(1, 8, dtype=own), torch.zeros(1, 1)
            right = A._TORCH_DTYPES[own] == dtype
            with pytest.raises(A.RwError if right else ValueError, match="RW_E" if right else "logits"):
                A.token_logprobs_dev(x, 1, 8, i32(1, 1), 1, lp, dtype=dtype)


def test_only_the_calls_rows_need_one_distance():
    a = numbered(2, 8, N)[:, :3]  # three rows, and three more 8 rows from the first
    assert A._rows(a, 3, N, None, "q", None) == (a.data_ptr(), N)
    assert A._rows(a, 1, N, None, "q", None)[0] == a.data_ptr()
    with pytest.raises(ValueError, match="one distance"):
        A._rows(a, 4, N, None, "q", None)

"""How the serving entries' Python wrappers take tensors: which element of
which row a call reads.  On the CPU: pointers and strides are looked at, no
call is queued."""
import pytest
import torch

from rusty_whisper_amd import _abi as A

H, D, ROWS = 4, 32, 6
N = H * D


def places(a, ld=None):
    """Element [row, value] as `_rows` tells the library to read it: offsets
    from the storage's start."""
    p, step = A._rows(a, N, ld, "q", None)
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
        assert A._rows(a, N, None, "q", None) == (a.data_ptr(), N)
    assert A._rows(numbered(ROWS * N), N, None, "q", None)[1] == N  # rows one behind the other
    assert A._rows(numbered(ROWS, N + 9), N, None, "q", None)[1] == N + 9  # the first columns of wider rows
    assert A._rows(numbered(ROWS, 2 * N), N, 3 * N, "q", None)[1] == 3 * N  # the caller's own stride


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
        A._rows(a, N, ld, "q", None)

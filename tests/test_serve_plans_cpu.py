"""How the serving entries cut their work, as the workspaces' sizes tell, and
the life of the page book's handle.  No device."""
import gc
import random

from rusty_whisper_amd import _abi as A


def chunks(rows, n_head, max_len, dtype=A.F32, kv=1, dim=128):
    """Of a row's keys, at most: a partial result is dim + 2 floats."""
    p = A.RwKvPages(dtype, kv, dim, 256, 1, 1, 0x10000, 0x20000)
    size = A.lib().rw_rocm_paged_attention_workspace_size(p, rows, n_head, max_len)
    assert size % (rows * n_head * (dim + 2) * 4) == 0
    return size // (rows * n_head * (dim + 2) * 4)


def test_the_most_chunks_are_512():
    assert chunks(1, 1, 65530) == 512 == chunks(1, 1, 2**30)
    rng = random.Random(8)
    for _ in range(2000):
        rows, kv, group = rng.choice((1, 1, 2, 3, 48, 1000)), rng.choice((1, 2, 8, 20)), rng.choice((1, 4, 17, 40))
        n = chunks(rows, kv * group, int(2 ** rng.uniform(0, 31)), rng.choice((A.F32, A.F16, A.BF16)), kv,
                   rng.choice((32, 64, 96, 128)))
        assert n <= (512 if rows == 1 else 256)


def test_a_book_is_freed_once(monkeypatch):
    freed, real = [], A.lib()

    class Lib:
        def __getattr__(self, name):
            if name != "rw_rocm_kv_book_free":
                return getattr(real, name)
            return lambda h: (freed.append(h), real.rw_rocm_kv_book_free(h))[1]

    monkeypatch.setattr(A, "lib", lambda: Lib())
    b = A.KvBook(4, 16, 1)
    h = b.handle
    del b
    gc.collect()
    assert freed == [h]
    b = A.KvBook(4, 16, 1)
    h = b.handle
    b.free()
    b.free()
    del b
    gc.collect()
    assert freed[1:] == [h]

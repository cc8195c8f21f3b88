"""The book of a paged key/value cache (rusty_whisper_amd/csrc/rw_kvbook.hpp)
without a device: against a model that holds every row's value, over random
histories; refusals change nothing; under AddressSanitizer as a native
program (tests/native/kv_book.cpp)."""
import os
import random
import shutil
import subprocess

import numpy as np
import pytest

from rusty_whisper_amd import _abi as A

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "rusty_whisper_amd", "csrc")


class Rows:
    """Sequences as lists of values, and a pool of pages that only the book's
    tables and copies can keep equal to them."""

    def __init__(self, n_pages, page_rows, max_seqs):
        self.book = A.KvBook(n_pages, page_rows, max_seqs)
        self.P = page_rows
        self.pool = np.full((n_pages, page_rows), -1, np.int64)
        self.seqs = {}
        self.next = 0

    def copy(self, src, dst):
        assert len(set(dst.tolist())) == len(dst) and not set(dst.tolist()) & set(src.tolist())
        self.pool[dst] = self.pool[src]

    def extend(self, seqs, more):
        self.copy(*self.book.extend(seqs, more))
        width = max([1] + [-(-(len(self.seqs[s]) + m) // self.P) for s, m in zip(seqs, more)])
        table = self.book.table(seqs, width)
        for row, s, m in zip(table, seqs, more):
            for _ in range(m):
                pos = len(self.seqs[s])
                self.pool[row[pos // self.P], pos % self.P] = self.next
                self.seqs[s].append(self.next)
                self.next += 1

    def check(self):
        n_pages = self.pool.shape[0]
        used = set()
        for s, want in self.seqs.items():
            assert self.book.len(s) == len(want)
            n = -(-len(want) // self.P)
            table = self.book.table([s], n + 1)[0]
            assert table[n] == 0
            got = self.pool[table[:n]].reshape(-1)[: len(want)]
            assert got.tolist() == want
            used |= set(table[:n].tolist())
        assert self.book.info() == (n_pages - len(used), len(used), len(self.seqs))
        return used


@pytest.mark.parametrize("seed", range(8))
@pytest.mark.parametrize("page_rows", [16, 64])
def test_random_histories(seed, page_rows):
    rng = random.Random(100 * seed + page_rows)
    n_pages, max_seqs = 41, 9
    m = Rows(n_pages, page_rows, max_seqs)
    refused = compacted = shared = 0
    for _ in range(400):
        live = sorted(m.seqs)
        what = rng.choice(["add", "fork", "extend", "extend", "extend", "truncate", "release", "compact"])
        try:
            if what == "add":
                for s in m.book.add(rng.randrange(3)).tolist():
                    m.seqs[s] = []
            elif what == "fork" and live:
                src = [rng.choice(live) for _ in range(rng.randrange(1, 4))]
                for s, d in zip(src, m.book.fork(src).tolist()):
                    m.seqs[d] = list(m.seqs[s])
            elif what == "extend" and live:
                seqs = rng.sample(live, rng.randrange(1, len(live) + 1))
                m.extend(seqs, [rng.choice([0, 1, 1, 2, page_rows - 1, page_rows, 3 * page_rows + 1]) for _ in seqs])
            elif what == "truncate" and live:
                s = rng.choice(live)
                n = rng.randrange(len(m.seqs[s]) + 1)
                m.book.truncate(s, n)
                del m.seqs[s][n:]
            elif what == "release" and live and rng.random() < 0.6:
                seqs = rng.sample(live, rng.randrange(1, len(live) + 1))
                m.book.release(seqs)
                for s in seqs:
                    del m.seqs[s]
            elif what == "compact":
                src, dst = m.book.compact()
                assert np.all(dst < m.book.info()[1]) and np.all(src >= m.book.info()[1])
                m.copy(src, dst)
                compacted += len(src)
        except A.RwError as e:
            assert e.code == A.RW_ENOMEM
            refused += 1
        used = m.check()
        shared += sum(-(-len(v) // page_rows) for v in m.seqs.values()) > len(used)
        if what == "compact":
            assert used == set(range(len(used)))
    assert refused and compacted and shared  # the histories reach all of it


def test_shared_tail_is_copied_once_per_growing_sequence_but_the_last():
    b = A.KvBook(16, 16, 8)
    (s,) = b.add()
    b.extend([s], 20)  # pages 0, 1
    f = b.fork([s, s, s])
    assert b.info() == (14, 2, 4)
    src, dst = b.extend(np.concatenate([[s], f[:2]]), 1)  # three of four grow: all copy, the fourth still holds the page
    assert src.tolist() == [1, 1, 1] and dst.tolist() == [2, 3, 4]
    src, dst = b.extend(f[2:], 1)  # the last holder keeps it
    assert len(src) == 0
    g = b.fork([s])
    src, dst = b.extend([s, g[0]], [1, 1])  # both grow: one copy is enough
    assert src.tolist() == [2] and dst.tolist() == [5]
    assert b.table([s, g[0]], 2).tolist() == [[0, 5], [0, 2]]


def test_full_last_page_and_empty_sequences_need_no_copy():
    b = A.KvBook(8, 16, 8)
    (s,) = b.add()
    (e,) = b.fork([s])
    src, _ = b.extend([s, e], [16, 0])
    assert len(src) == 0
    (t,) = b.fork([s])
    src, _ = b.extend([s, t], 1)
    assert len(src) == 0 and b.table([s, t], 2).tolist() == [[0, 1], [0, 2]]


def test_lowest_ids_first():
    b = A.KvBook(200, 16, 8)
    s = b.add(4)
    assert s.tolist() == [0, 1, 2, 3]
    b.extend(s, 16 * 40)
    b.release([1, 3])
    assert b.add(2).tolist() == [1, 3]
    b.extend([3], 16 * 41)
    assert b.table([3], 41)[0].tolist() == list(range(40, 80)) + [120]


def _raises(code, needle, f, *a):
    with pytest.raises(A.RwError) as e:
        f(*a)
    assert e.value.code == code and needle in e.value.message, e.value


def test_refusals_change_nothing():
    b = A.KvBook(4, 16, 3)
    s = b.add(2)
    b.extend(s, [20, 3])
    before = (b.info(), b.table(s, 4).tolist(), [b.len(i) for i in s])
    _raises(A.RW_ENOMEM, "not enough free pages", b.extend, s, [13, 14])
    _raises(A.RW_EINVAL, "listed twice", b.extend, [0, 1, 0], 1)
    _raises(A.RW_EINVAL, "no such sequence", b.extend, [0, 2], 1)
    _raises(A.RW_EINVAL, "no such sequence", b.extend, [-1], 1)
    _raises(A.RW_EINVAL, "length out of range", b.extend, [0], 2**31)
    _raises(A.RW_ENOMEM, "all sequences", b.add, 2)
    _raises(A.RW_ENOMEM, "all sequences", b.fork, [0, 0])
    _raises(A.RW_EINVAL, "no such sequence", b.fork, [7])
    _raises(A.RW_EINVAL, "length out of range", b.truncate, 0, 21)
    _raises(A.RW_EINVAL, "no such sequence", b.truncate, 2, 0)
    _raises(A.RW_EINVAL, "listed twice", b.release, [0, 0])
    _raises(A.RW_EINVAL, "no such sequence", b.release, [0, 5])
    _raises(A.RW_EINVAL, "no such sequence", b.len, 5)
    _raises(A.RW_EINVAL, "pages, a table row", b.table, s, 1)
    with pytest.raises(ValueError):
        b.extend([0], -1)
    assert before == (b.info(), b.table(s, 4).tolist(), [b.len(i) for i in s])


def test_compact_says_how_many_it_needs():
    import ctypes as C

    b = A.KvBook(8, 16, 4)
    s = b.add(2)
    b.extend(s, [48, 40])
    b.release(s[:1])  # pages 3, 4, 5 in use
    n = C.c_size_t()
    a = np.zeros(2, np.int32)
    rc = A.lib().rw_rocm_kv_book_compact(b.handle, a.ctypes.data, a.ctypes.data, 2, C.byref(n))
    assert rc == A.RW_EINVAL and n.value == 3 and b.table(s[1:], 3).tolist() == [[3, 4, 5]]
    src, dst = b.compact()
    assert src.tolist() == [3, 4, 5] and dst.tolist() == [0, 1, 2] and b.table(s[1:], 3).tolist() == [[0, 1, 2]]
    assert [x.size for x in b.compact()] == [0, 0]


def test_create_and_null_arguments():
    import ctypes as C

    for args, needle in [((0, 16, 1), "n_pages"), ((2**31, 16, 1), "n_pages"), ((4, 24, 1), "page_rows"),
                         ((4, 8, 1), "page_rows"), ((4, 512, 1), "page_rows"), ((4, 16, 0), "max_seqs")]:
        _raises(A.RW_EINVAL, needle, A.KvBook, *args)
    L, n = A.lib(), C.c_size_t()
    assert L.rw_rocm_kv_book_create(4, 16, 1, None) == A.RW_EINVAL
    assert L.rw_rocm_kv_book_add(None, 1, None) == A.RW_EINVAL
    assert L.rw_rocm_kv_book_extend(None, None, 0, None, None, None, C.byref(n)) == A.RW_EINVAL
    assert L.rw_rocm_kv_book_info(None, None, None, None) == A.RW_EINVAL
    assert L.rw_rocm_kv_book_len(None, 0, C.byref(n)) == A.RW_EINVAL
    L.rw_rocm_kv_book_free(None)
    b = A.KvBook(4, 16, 1)
    for rc in (L.rw_rocm_kv_book_add(b.handle, 1, None), L.rw_rocm_kv_book_fork(b.handle, None, 1, None),
               L.rw_rocm_kv_book_release(b.handle, None, 1), L.rw_rocm_kv_book_table(b.handle, None, 1, None, 1),
               L.rw_rocm_kv_book_compact(b.handle, None, None, 1, C.byref(n))):
        assert rc == A.RW_EINVAL
    assert L.rw_rocm_kv_book_add(b.handle, 0, None) == A.RW_OK
    assert b.info() == (4, 0, 0)


def test_frees_on_collection():
    assert "free" in vars(A.KvBook) and "__del__" in vars(A.KvBook)


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_native_under_address_sanitizer(tmp_path):
    exe = str(tmp_path / "kv_book")
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-Wall", "-Wextra", "-fsanitize=address,undefined", f"-I{CSRC}",
                    os.path.join(HERE, "native", "kv_book.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "bad=0" in r.stdout, r.stdout + r.stderr

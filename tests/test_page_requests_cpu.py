"""Launches of the page operations for more requests than a grid takes, on the host emulation of the kernels, which here
refuses launches above a limit as a GPU refuses those of 2^32 threads."""
import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

import indexed_util as iu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EMUL = os.path.join(ROOT, "tests", "emul")
CLANG = "/opt/rocm/lib/llvm/bin/clang++"
pytestmark = pytest.mark.skipif(not os.path.exists(CLANG) or shutil.which("make") is None,
                                reason="needs the ROCm clang++ and make to build the host emulation")


@pytest.fixture(scope="module")
def emul():
    r = subprocess.run(["make", "-C", EMUL, "SAN=none", "-j4"], capture_output=True, text=True, timeout=1800)
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-3000:]
    return ctypes.CDLL(os.path.join(EMUL, "_build", "none", "libdfccl_emul.so"))


class Cache:
    """A cache in host memory with its definition beside it."""

    def __init__(self, emul, pages, page_tokens, sequences, per_seq):
        from dfccl_amd import _lib
        contents = np.random.RandomState(3).randint(0, 256, (pages, 24)).astype(np.uint8)
        self.emul, self.books = emul, iu.Books([contents], page_tokens, sequences, per_seq)
        need = ctypes.c_size_t()
        assert emul.dfcclPageCacheWorkspace(pages, sequences, ctypes.byref(need)) == 0
        self.pool, self.refs, self.lengths = contents.copy(), np.zeros(pages, np.int32), np.zeros(sequences, np.int32)
        self.tables, self.report = np.full((sequences, per_seq), -1, np.int32), np.zeros(3, np.int32)
        self.workspace = np.zeros(need.value, np.uint8)
        pools = (ctypes.c_void_p * 1)(self.pool.ctypes.data)
        self.struct = _lib.PageCacheStruct(
            ctypes.sizeof(_lib.PageCacheStruct), pools, 24, 1, pages, page_tokens, sequences, per_seq,
            *(a.ctypes.data for a in (self.refs, self.tables, self.lengths, self.report, self.workspace)), need.value)

    def call(self, name, *lists):
        lists = [np.asarray(x, np.int32) for x in lists]
        rc = getattr(self.emul, "dfcclPages" + name)(ctypes.byref(self.struct), *(ctypes.c_void_p(x.ctypes.data) for x in lists),
                                                    len(lists[0]), None)
        self.emul.emulNullStreamSynchronize()
        assert rc == 0, f"{name}: {rc}"
        getattr(self.books, name.lower())(*(x.tolist() for x in lists))
        for got, want in ((self.refs, self.books.refs), (self.tables, self.books.tables), (self.lengths, self.books.lengths),
                          (self.pool, self.books.contents[0])):
            assert np.array_equal(got, want), name
        assert self.report[0] == self.books.refused


@pytest.fixture
def limited(emul):
    emul.emulLaunchLimit.argtypes = [ctypes.c_uint64]
    emul.emulLaunchLimit(16000)  # threads a launch may have
    yield emul
    emul.emulLaunchLimit((1 << 32) - 1)


def test_extend_and_fork_of_more_requests_than_a_grid_has_workgroups(limited):
    cache = Cache(limited, pages=5000, page_tokens=4, sequences=400, per_seq=6)
    rs = np.random.RandomState(4)
    cache.call("Extend", rs.permutation(200), rs.randint(0, 25, 200))
    cache.call("Fork", rs.randint(-1, 201, 199), 200 + rs.permutation(199))  # (refusals and shared parents among them)
    cache.call("Extend", rs.permutation(400), rs.randint(0, 26, 400))
    cache.call("Free", rs.permutation(400)[:250])


def test_no_walk_over_a_list_counts_in_a_type_that_its_last_step_leaves():
    # lists, sequences and table rows have up to 2^31 - 1 entries, and a walk's last step goes beyond the last one by up
    # to a grid: with a signed counter of 32 bits it would come out negative, and be followed
    import re
    with open(os.path.join(ROOT, "dfccl_amd", "csrc", "pages.hip")) as f:
        walks = re.findall(r"for \((\w+) (\w+) = [^;]*; ([^;]*); \2 \+= [^)]*", f.read())
    kinds = {kind for kind, _, end in walks if "npools" not in end}
    assert len(walks) >= 15 and kinds <= {"int64_t", "uint64_t", "uint32_t", "ListIndex"}

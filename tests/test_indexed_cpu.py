"""The row and page operators without a GPU: what the C entry points refuse, and the GPU tests of these operators run
on the host emulation of their kernels (tests/emul: one OS thread per GPU thread, buffers in host memory)."""
import ctypes
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EMUL = os.path.join(ROOT, "tests", "emul")
LIB = os.path.join(ROOT, "dfccl_amd", "libdfccl.so")
built = pytest.mark.skipif(not os.path.exists(LIB), reason="libdfccl.so not built")
OK, INVALID = 0, 4
F32, F16, F64, BF16, I32, I64, I8, U32 = 7, 6, 8, 9, 2, 4, 0, 3
PTR = 1 << 20  # an address that is never followed: every call here ends before a launch


def lib():
    from dfccl_amd import _lib
    return _lib.load()


@built
def test_lookup_refuses():
    good = dict(table=PTR, table_type=BF16, rows=10, table_stride=8, first=0, ids=PTR, id_type=I64, tokens=3, width=8,
                scale=1.0, out=PTR, out_type=BF16, out_stride=8, stream=None)

    def call(**change):
        return lib().dfcclEmbeddingLookup(*{**good, **change}.values())
    for change in (dict(table_type=F64), dict(table_type=I8), dict(out_type=I32), dict(out_type=99), dict(id_type=U32),
                   dict(id_type=F32), dict(table_stride=7), dict(out_stride=7), dict(first=-1), dict(table=None),
                   dict(ids=None), dict(out=None), dict(rows=1 << 31), dict(width=1 << 31, table_stride=1 << 31, out_stride=1 << 31),
                   dict(tokens=1 << 31)):
        assert call(**change) == INVALID, change
    assert call(tokens=0) == OK and call(width=0) == OK  # nothing to do, nothing launched


@built
def test_gradient_refuses():
    two = (ctypes.c_void_p * 2)(PTR, PTR)
    sizes = (ctypes.c_size_t * 2)(5, 7)
    need = ctypes.c_size_t()
    assert lib().dfcclEmbeddingGradWorkspace(2, sizes, 10, 8, ctypes.byref(need)) == OK and need.value > 0
    good = dict(grads=two, ids=two, tokens=sizes, nsrcs=2, grad_type=BF16, grad_stride=8, id_type=I64, first=0, rows=10,
                width=8, padding=-1, scale=1.0, accumulate=0, out=PTR, table_type=F32, table_stride=8, ws=PTR,
                ws_bytes=need.value, stream=None)

    def call(**change):
        return lib().dfcclEmbeddingGrad(*{**good, **change}.values())
    missing, huge = (ctypes.c_void_p * 2)(PTR, None), (ctypes.c_size_t * 2)(5, 1 << 28)
    for change in (dict(grad_type=F64), dict(table_type=I32), dict(id_type=U32), dict(nsrcs=0), dict(nsrcs=9),
                   dict(grad_stride=7), dict(table_stride=7), dict(first=-1), dict(grads=None), dict(ids=None),
                   dict(grads=missing), dict(ids=missing), dict(tokens=None), dict(tokens=huge), dict(out=None),
                   dict(ws=None), dict(ws_bytes=need.value - 1), dict(ws=PTR + 8), dict(rows=1 << 31)):
        assert call(**change) == INVALID, change
    none = (ctypes.c_size_t * 2)(0, 0)
    assert call(rows=0) == OK and call(width=0) == OK and call(tokens=none, accumulate=1) == OK
    w = lib().dfcclEmbeddingGradWorkspace
    assert w(0, sizes, 10, 8, ctypes.byref(need)) == INVALID and w(9, sizes, 10, 8, ctypes.byref(need)) == INVALID
    assert w(2, None, 10, 8, ctypes.byref(need)) == INVALID and w(2, sizes, 10, 8, None) == INVALID
    assert w(2, huge, 10, 8, ctypes.byref(need)) == INVALID


@built
def test_pages_refuse():
    from dfccl_amd import _lib
    L = lib()
    need = ctypes.c_size_t()
    assert L.dfcclPageCacheWorkspace(6, 3, ctypes.byref(need)) == OK and need.value > 0
    for args in ((0, 3, ctypes.byref(need)), (6, 0, ctypes.byref(need)), (-1, 3, ctypes.byref(need)), (6, 3, None)):
        assert L.dfcclPageCacheWorkspace(*args) == INVALID
    L.dfcclPageCacheWorkspace(6, 3, ctypes.byref(need))
    pools = (ctypes.c_void_p * 2)(PTR, PTR)

    def cache(**change):
        fields = dict(structBytes=ctypes.sizeof(_lib.PageCacheStruct), pools=pools, pageBytes=64, npools=2, pages=6,
                      pageTokens=4, sequences=3, pagesPerSequence=2, refcounts=PTR, tables=PTR, lengths=PTR, report=None,
                      workspace=PTR, workspaceBytes=need.value)
        return _lib.PageCacheStruct(*{**fields, **change}.values())

    def every(c):
        r = ctypes.byref(c) if c is not None else None
        return [L.dfcclPagesExtend(r, PTR, PTR, 1, None), L.dfcclPagesFork(r, PTR, PTR, 1, None),
                L.dfcclPagesFree(r, PTR, 1, None), L.dfcclPagesCompact(r, None)]
    missing = (ctypes.c_void_p * 2)(PTR, None)
    for change in (dict(structBytes=8), dict(pools=None), dict(pools=missing), dict(pageBytes=0), dict(npools=0), dict(pages=0),
                   dict(pageTokens=0), dict(sequences=0), dict(pagesPerSequence=0), dict(refcounts=None), dict(tables=None),
                   dict(lengths=None), dict(workspace=None), dict(workspaceBytes=need.value - 1), dict(workspace=PTR + 2),
                   dict(sequences=1 << 16, pagesPerSequence=1 << 15, workspaceBytes=1 << 30),
                   dict(pagesPerSequence=1 << 20, pageTokens=1 << 11)):
        assert every(cache(**change)) == [INVALID] * 4, change
    assert every(None) == [INVALID] * 4
    good = ctypes.byref(cache())
    assert L.dfcclPagesExtend(good, PTR, PTR, 4, None) == INVALID and L.dfcclPagesExtend(good, PTR, PTR, -1, None) == INVALID
    assert L.dfcclPagesExtend(good, None, PTR, 1, None) == INVALID and L.dfcclPagesExtend(good, PTR, None, 1, None) == INVALID
    assert L.dfcclPagesFork(good, PTR, PTR, 4, None) == INVALID and L.dfcclPagesFork(good, PTR, None, 1, None) == INVALID
    assert L.dfcclPagesFree(good, None, 1, None) == INVALID and L.dfcclPagesFree(good, PTR, -1, None) == INVALID
    assert L.dfcclPagesFree(good, None, 0, None) == OK
    bare = ctypes.byref(cache(refcounts=None, tables=None, lengths=None, workspace=None, workspaceBytes=0))
    assert L.dfcclPagesCopy(bare, bare, None, None, 0, None) == OK  # a copy looks at no bookkeeping
    assert L.dfcclPagesCopy(bare, bare, None, PTR, 1, None) == INVALID
    assert L.dfcclPagesCopy(bare, None, PTR, PTR, 1, None) == INVALID
    assert L.dfcclPagesCopy(bare, bare, PTR, PTR, -1, None) == INVALID
    assert L.dfcclPagesCopy(bare, ctypes.byref(cache(pageBytes=65)), PTR, PTR, 1, None) == INVALID
    assert L.dfcclPagesCopy(bare, ctypes.byref(cache(npools=1)), PTR, PTR, 1, None) == INVALID


@pytest.mark.skipif(not os.path.exists("/opt/rocm/bin/hipcc"), reason="needs hipcc")
@pytest.mark.parametrize("source", ["embedding", "pages"])
def test_kernels_use_no_scratch_and_spill_no_vector_registers(source):
    from test_kernel_resources_cpu import resources
    kernels = resources(source)
    assert len(kernels) >= 10
    for name, k in kernels.items():
        assert int(k["ScratchSize [bytes/lane]"]) == 0 and k["Dynamic Stack"] == "False", name
        assert int(k["VGPRs Spill"]) == 0, name


CLANG = "/opt/rocm/lib/llvm/bin/clang++"


@pytest.mark.skipif(not os.path.exists(CLANG) or shutil.which("make") is None,
                    reason="needs the ROCm clang++ and make to build the host emulation")
@pytest.mark.parametrize("name", ["embedding", "pages"])
def test_gpu_tests_on_the_emulation(name):
    """Everything in the two files but what needs a real GPU's size (and the one that takes 10,000s of threads)."""
    r = subprocess.run(["make", "-C", EMUL, "SAN=none", "-j4"], capture_output=True, text=True, timeout=1800)
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-3000:]
    e = dict(os.environ)
    e.update({"DFCCL_TESTS_ON_EMULATION": os.path.join(EMUL, "_build", "none", "libdfccl_emul.so"), "EMUL_WATCHDOG_S": "120"})
    r = subprocess.run([sys.executable, "-m", "pytest", os.path.join(ROOT, "tests", f"test_{name}_gpu.py"), "-q", "-m", "gpu",
                        "-x", "-p", "no:cacheprovider", "--timeout", "600", "-k", "not several_rows_a_wave"], env=e,
                       capture_output=True, text=True, timeout=1500, cwd=ROOT)
    tail = r.stdout[-3000:] + r.stderr[-2000:]
    assert r.returncode == 0, tail
    assert " passed" in r.stdout and " failed" not in r.stdout, tail

"""The paged cache and the adapters on the host: rows of tables that hold
anything stay in the pool, and malformed calls are refused before a launch."""
import os
import subprocess

import numpy as np
import pytest

import paged_ref as ref
from mdma_amd import backend

HERE = os.path.dirname(os.path.abspath(__file__))
CLANG = "/opt/rocm/llvm/bin/clang++"  # (the internal header names _Float16)


def build_and_run(tmp_path, src, compiler, *flags):
    exe = str(tmp_path / "t")
    subprocess.run([*compiler, "-std=c++17", "-O1", os.path.join(HERE, src), "-o", exe, *flags], check=True,
                   capture_output=True, timeout=300)
    p = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert p.returncode == 0, p.stdout[-3000:] + p.stderr[-1000:]
    assert "ok" in p.stdout


def test_rows_of_any_table_lie_in_the_pool(tmp_path):
    build_and_run(tmp_path, "paged_walk.cpp", ["g++", "-Wall"])


@pytest.mark.skipif(not os.path.exists(CLANG), reason="needs ROCm")
def test_malformed_calls_are_refused_without_a_gpu(tmp_path):
    build_and_run(tmp_path, "serve_refusals.cpp", [CLANG, "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include"],
                  backend.LIB_PATH, "-Wl,-rpath," + os.path.dirname(backend.LIB_PATH), "-L/opt/rocm/lib", "-lamdhip64",
                  "-Wl,-rpath,/opt/rocm/lib")


@pytest.mark.parametrize("seed", range(20))
def test_books_stay_consistent(seed):
    """The plain books that the kernels are held to: pages counted as often as rows hold them, never two owners of a
    page that one of them writes."""
    r = np.random.default_rng(seed)
    S, pl, M = int(r.integers(1, 9)), 16, int(r.integers(1, 9))
    b = ref.Books(int(r.integers(1, 40)), pl, S, M)
    for _ in range(12):
        before = b.lens.copy()
        status, copies = b.grow(r.integers(0, 40, S))
        for s in range(S):
            if b.lens[s] > before[s]:
                first = int(before[s]) // pl
                assert all(b.refs[p] == 1 for p in b.table[s, first:b.used(b.lens[s])])
        for src, dst, rows in copies:
            assert src != dst and 0 < rows < pl
        b.fork(r.integers(0, S + 1, S), r.integers(0, M * pl + 1, S))
        L, moves = b.compact()
        assert set(np.nonzero(b.refs)[0]) == set(range(L))
        rows = [p for s in range(S) for p in b.table[s, :b.used(b.lens[s])]]
        assert np.array_equal(np.bincount(rows, minlength=b.P) if rows else np.zeros(b.P), b.refs)

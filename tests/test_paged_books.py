"""The paged cache's books without a GPU (tests/host/paged_books.cpp): calls that
find no memory, pinned or ordinary, and calls that a capture does not allow change
nothing."""
import os
import subprocess

import pytest

from conftest import ROOT
from llama3pure_b200.build import ARCH_FLAGS, CSRC, INCLUDE, nvcc


@pytest.fixture(scope="module")
def books(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("books") / "paged_books")
    subprocess.run([nvcc(), *ARCH_FLAGS, "-O1", "-std=c++17", "-cudart", "none", "-I", INCLUDE, "-I", CSRC, "-o", exe,
                    os.path.join(ROOT, "tests", "host", "paged_books.cpp"), os.path.join(CSRC, "l3p_paged.cu")], check=True)

    def run(*args):
        r = subprocess.run([exe, *args], capture_output=True, text=True, timeout=120)
        assert r.returncode == 0, r.stdout + r.stderr

    return run


@pytest.mark.parametrize("call", ["begin", "copy", "fork", "compact"])
def test_a_call_without_memory_changes_nothing(books, call):
    books(call)


@pytest.mark.parametrize("call", ["begin", "copy", "fork", "compact"])
def test_no_exception_leaves_a_call_when_memory_is_exhausted(books, call):
    """Every allocation after the failing one fails too."""
    books(call, "rest")


def test_create_without_memory_says_why(books):
    books("create")
    books("create", "rest")


def test_capture_of_the_stream_or_of_one_that_the_null_stream_waits_for(books):
    books("capture")

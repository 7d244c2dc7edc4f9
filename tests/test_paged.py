"""The paged cache's C ABI without a GPU: bad configurations are refused
before the device is touched, and null arguments are errors."""
import ctypes as C
import os
import re

import pytest

from llama3pure_b200 import attn
from llama3pure_b200.build import CSRC


def _cfg(**kw):
    base = dict(n_layers=2, n_heads=8, n_kv_heads=2, head_dim=128, page_size=16, n_pages=8, max_seqs=4, max_tokens=64,
                max_seq_len=0, dtype=0, scale=0.0, is_gemma3=0, swa_window=0, swa_pattern=0, device=0)
    base.update(kw)
    return attn.PagedConfig(**base)


@pytest.mark.parametrize("kw,code", [
    (dict(n_heads=6, n_kv_heads=4), -1),
    (dict(n_heads=0), -1),
    (dict(n_layers=0), -1),
    (dict(head_dim=96), -6),
    (dict(page_size=24), -6),
    (dict(page_size=256), -6),
    (dict(n_pages=0), -1),
    (dict(max_seqs=0), -1),
    (dict(max_tokens=0), -1),
    (dict(max_seq_len=-1), -1),
    (dict(dtype=2), -1),
    (dict(scale=float("nan")), -1),
    (dict(scale=-0.1), -1),
    (dict(swa_window=-1), -1),
    (dict(device=-1), -1),
    (dict(n_pages=2**30), -2),                                  # positions beyond 32 bits
    (dict(n_pages=2**20, n_layers=2**10), -2),                  # rows of storage beyond 32 bits
    (dict(max_tokens=2**30), -2),
    (dict(max_seqs=2**20), -2),
])
def test_create_rejects_bad_config_without_device(lib, kw, code):
    h = C.c_void_p()
    assert lib.l3p_paged_create(C.byref(_cfg(**kw)), C.byref(h)) == code
    assert not h.value


def test_null_arguments_are_errors(lib):
    n = C.c_int()
    assert lib.l3p_paged_create(None, None) == -1
    assert lib.l3p_paged_seq_new(None, C.byref(n)) == -1
    assert lib.l3p_paged_seq_fork(None, 0, -1, 1, C.byref(n)) == -1
    assert lib.l3p_paged_seq_copy(None, 0, None, None, None) == -1
    assert lib.l3p_paged_seq_truncate(None, 0, 0) == -1
    assert lib.l3p_paged_seq_free(None, 0, None) == -1
    assert lib.l3p_paged_seq_length(None, 0, C.byref(n)) == -1
    assert lib.l3p_paged_tables(None, 0, None, 0, None, None) == -1
    assert lib.l3p_paged_free_pages(None, C.byref(n)) == -1
    assert lib.l3p_paged_compact(None, C.byref(n), None) == -1
    assert lib.l3p_paged_begin(None, 0, None, None, None) == -1
    assert lib.l3p_paged_set_rope(None, None) == -1
    assert lib.l3p_paged_rope_append_dev(None, 0, None, 0, None, 0, None, 0, None, 0, None) == -1
    assert lib.l3p_paged_append_dev(None, 0, None, 0, None, 0, None) == -1
    assert lib.l3p_paged_attn_dev(None, 0, None, 0, None, 0, None) == -1
    assert lib.l3p_paged_check(None, None) == -1
    assert lib.l3p_paged_storage(None, None, None) == -1
    assert lib.l3p_paged_launch_count(None) == -1
    assert lib.l3p_paged_last_error(None) == b""
    lib.l3p_paged_destroy(None)


def test_warps_meet_with_the_outcome_of_their_waits():
    """The loop over key tiles of the fp32 chunk kernel has a barrier that some of a CTA's warps meet at.  A warp's bounded wait
    may give up where another's does not, so the barrier has to tell all of them: one that only counts threads would be waited
    for without a bound by the warps that go on."""
    with open(os.path.join(CSRC, "paged_f32.cuh")) as f:
        code = re.sub(r"//[^\n]*", "", f.read())
    assert not re.findall(r"bar(?:rier)?(?:\.cta)?\.sync", code)
    assert len(re.findall(r"bar\.red\.and\.pred", code)) == 1
    meets = re.findall(r"[^\n]*pg_meet\(ok\)[^\n]*", code)
    assert len(meets) == 2 and all(re.search(r"if \(!\(ok = pg_meet\(ok\)\)\) break;", m) for m in meets)


@pytest.mark.parametrize("kw,text", [
    (dict(n_heads=6, n_kv_heads=4), "n_heads"),
    (dict(head_dim=96), "head_dim"),
    (dict(page_size=24), "page_size"),
    (dict(dtype=2), "dtype"),
    (dict(scale=-0.1), "scale"),
    (dict(n_pages=2**30), "positions"),
    (dict(max_seqs=2**20), "max_seqs"),
    (dict(max_tokens=2**30), "max_tokens"),
    (dict(n_pages=2**20, n_layers=2**10), "rows"),
])
def test_a_refused_create_says_why(lib, kw, text):
    from llama3pure_b200.paged import PagedCache

    h = C.c_void_p()
    assert lib.l3p_paged_create(C.byref(_cfg(**kw)), C.byref(h)) < 0
    assert text in lib.l3p_paged_create_error().decode()
    base = dict(n_layers=2, n_heads=8, n_kv_heads=2, head_dim=128, page_size=16, n_pages=8, max_seqs=4, max_tokens=64) | kw
    if base.get("dtype", "f32") == "f32":  # the binding refuses names of types by itself
        with pytest.raises(attn.AttnError, match=text):
            PagedCache(**base, lib=lib)


@pytest.mark.parametrize("kw", [
    dict(n_pages=2**20, n_layers=2**30, n_heads=2**9, n_kv_heads=2**9, max_tokens=1),  # 2^64 rows: 0 in 64 bits
    dict(n_pages=2**26, n_layers=2**22, n_heads=2**12, n_kv_heads=2**12, max_tokens=1),  # 2^65
    dict(n_pages=2**22, n_layers=2**30 + 1, n_heads=2**12, n_kv_heads=2**12, max_tokens=1),
])
def test_sizes_whose_product_passes_64_bits_are_refused(lib, kw):
    h = C.c_void_p()
    assert lib.l3p_paged_create(C.byref(_cfg(**kw)), C.byref(h)) == -2
    assert not h.value


def test_the_binding_refuses_numbers_beyond_32_bits():
    """ctypes would cut them off: a cut at 2^32 positions would empty the sequence, a pool of 2^32 + 8 pages have 8."""
    from llama3pure_b200.paged import PagedCache

    class Lib:  # nothing may be called
        def __getattr__(self, name):
            def call(*args):
                raise AssertionError(f"{name}{args} was called")

            return call

    base = dict(n_layers=2, n_heads=8, n_kv_heads=2, head_dim=128, page_size=16, n_pages=8, max_seqs=4, max_tokens=64)
    for k in (*base, "max_seq_len", "swa_window", "device"):
        with pytest.raises(OverflowError):
            PagedCache(**(base | {k: 2**32 + 8}), lib=Lib())
    c = PagedCache.__new__(PagedCache)
    c.lib, c.h = Lib(), None
    for call in (lambda: c.truncate(0, 2**32), lambda: c.truncate(2**32, 0), lambda: c.fork(0, 1, 2**32), lambda: c.fork(2**32), lambda: c.fork(0, 2**32),
                 lambda: c.length(2**32), lambda: c.free([2**32]), lambda: c.begin([0], [2**32])):
        with pytest.raises(OverflowError):
            call()

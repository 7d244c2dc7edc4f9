"""Python binding of the paged KV cache (include/llama3pure_paged.h): many
sequences in one pool of pages, batched attention over them, rotary positions
written with the new rows, and forks, copies and compaction of pages.

    cache = PagedCache(n_layers=32, n_heads=32, n_kv_heads=8, head_dim=128, page_size=16,
                       n_pages=4096, max_seqs=64, max_tokens=2048, dtype="bf16")
    cache.set_rope(max_pos=8192, layout="interleaved")
    a, b = cache.new_seq(), cache.new_seq()
    cache.begin([a, b], [700, 1])            # a chunk of a's prompt, one token of b
    for layer in range(32):
        cache.rope_append_dev(layer, q, k, v, q)   # torch CUDA tensors [701, heads, 128]
        cache.attn_dev(layer, q, out)

There is no CPU fallback.  Kernels run on the given torch stream, by default
torch's current stream of the cache's device.
"""
from __future__ import annotations

import ctypes as C
from array import array

import numpy as np

from .attn import L3P_OK, AttnError, PagedConfig, PagedRopeConfig, load_library

DTYPES = {"f32": 0, "bf16": 1}
LAYOUTS = {"interleaved": 0, "half": 1}
SCALINGS = {"none": 0, "linear": 1, "bands": 2, "yarn": 3}


def _ints(x) -> tuple[int, int, array]:
    """Whole numbers of 32 bits: address, count, and the array that holds them (others raise)."""
    a = array("i", x.tolist() if hasattr(x, "tolist") else x)
    return *a.buffer_info(), a


def _int(x) -> int:
    """A whole number of 32 bits (others raise; ctypes would cut them off)."""
    return array("i", (x,))[0]


class _Memory:
    """A cache's storage for torch, which holds this object by its tensor: the cache lives as long as that.  No class of its own
    for every tensor: a class is part of a reference cycle, and the pool would stay until a garbage collection."""

    def __init__(self, owner, interface: dict):
        self.owner = owner
        self.__cuda_array_interface__ = interface


class PagedCache:
    """One l3p_paged_ctx."""

    def __init__(self, n_layers: int, n_heads: int, n_kv_heads: int, head_dim: int, page_size: int, n_pages: int,
                 max_seqs: int, max_tokens: int, max_seq_len: int = 0, dtype: str = "f32", scale: float = 0.0,
                 is_gemma3: int = 0, swa_window: int = 0, swa_pattern: int = 0, device: int = 0, lib=None):
        import torch

        self.torch = torch
        self.lib = lib or load_library()
        if dtype not in DTYPES:
            raise ValueError(f"dtype {dtype!r}: one of {sorted(DTYPES)}")
        self.cfg = PagedConfig(*map(_int, (n_layers, n_heads, n_kv_heads, head_dim, page_size, n_pages, max_seqs, max_tokens,
                                           max_seq_len, DTYPES[dtype])), scale, *map(_int, (is_gemma3, swa_window, swa_pattern, device)))
        self.dtype = torch.bfloat16 if dtype == "bf16" else torch.float32
        self.n_layers, self.n_heads, self.n_kv_heads, self.head_dim = n_layers, n_heads, n_kv_heads, head_dim
        self.device = device
        # the handle of torch's current stream, without a Stream object around it where torch offers that
        self._current_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                                       lambda d: torch.cuda.current_stream(d).cuda_stream)
        self.n_tokens = 0  # of the current batch
        self.h = None
        h = C.c_void_p()
        rc = self.lib.l3p_paged_create(C.byref(self.cfg), C.byref(h))
        if rc != L3P_OK:
            raise AttnError(rc, f"create: {self.lib.l3p_paged_create_error().decode()}")
        self.h = h

    @classmethod
    def for_shape(cls, shape, **kw) -> "PagedCache":
        kw.setdefault("n_layers", shape.n_layers)
        return cls(n_heads=shape.n_heads, n_kv_heads=shape.n_kv_heads, head_dim=shape.head_dim,
                   is_gemma3=shape.is_gemma3, swa_window=shape.swa_window, swa_pattern=shape.swa_pattern, **kw)

    # -- lifecycle -----------------------------------------------------------
    def close(self) -> None:
        if getattr(self, "h", None):
            self.lib.l3p_paged_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def _ok(self, rc: int, what: str) -> None:
        if rc != L3P_OK:
            msg = self.lib.l3p_paged_last_error(self.h)
            raise AttnError(rc, f"{what}: {msg.decode() if msg else ''}")

    def _stream(self, stream) -> int:
        if stream is None:
            return self._current_stream(self.device)
        return stream if isinstance(stream, int) else stream.cuda_stream

    def check(self, stream=None) -> None:
        """Waits for the stream and raises what its kernels recorded."""
        self._ok(self.lib.l3p_paged_check(self.h, self._stream(stream)), "check")

    def launch_count(self) -> int:
        return int(self.lib.l3p_paged_launch_count(self.h))

    def storage(self):
        """The pool as a tensor [n_pages][n_layers][2: K, V][n_kv_heads][page_size][head_dim] that shares its
        memory and keeps the cache alive; valid until close()."""
        base, size = C.c_void_p(), C.c_size_t()
        self._ok(self.lib.l3p_paged_storage(self.h, C.byref(base), C.byref(size)), "storage")
        c = self.cfg
        memory = _Memory(self, {  # bfloat16 has no array-interface type: 16-bit integers, viewed below
            "shape": (c.n_pages, c.n_layers, 2, c.n_kv_heads, c.page_size, c.head_dim),
            "typestr": "<f4" if c.dtype == 0 else "<i2", "data": (base.value, False), "version": 3, "stream": None,
        })
        t = self.torch.as_tensor(memory, device=f"cuda:{self.device}")
        return t if c.dtype == 0 else t.view(self.torch.bfloat16)

    # -- sequences and pages -----------------------------------------------------
    def new_seq(self) -> int:
        s = C.c_int()
        self._ok(self.lib.l3p_paged_seq_new(self.h, C.byref(s)), "new_seq")
        return s.value

    def fork(self, seq: int, n: int = 1, n_tokens: int = -1) -> list[int]:
        """n sequences that share the first n_tokens positions of `seq` (default: all of them)."""
        seq, n, n_tokens = map(_int, (seq, n, n_tokens))
        out = array("i", bytes(4 * max(n, 1)))
        self._ok(self.lib.l3p_paged_seq_fork(self.h, seq, n_tokens, n, out.buffer_info()[0]), "fork")
        return out.tolist()[:n]

    def copy(self, seqs, stream=None) -> list[int]:
        """Sequences with pages of their own and the rows of `seqs`."""
        p, n, ids = _ints(seqs)
        out = array("i", ids)
        self._ok(self.lib.l3p_paged_seq_copy(self.h, n, p, out.buffer_info()[0], self._stream(stream)), "copy")
        return out.tolist()

    def truncate(self, seq: int, n_tokens: int) -> None:
        self._ok(self.lib.l3p_paged_seq_truncate(self.h, _int(seq), _int(n_tokens)), "truncate")

    def free(self, seqs) -> None:
        p, n, ids = _ints(seqs)
        self._ok(self.lib.l3p_paged_seq_free(self.h, n, p), "free")

    def length(self, seq: int) -> int:
        n = C.c_int()
        self._ok(self.lib.l3p_paged_seq_length(self.h, _int(seq), C.byref(n)), "length")
        return n.value

    def tables(self, seqs) -> np.ndarray:
        """Page tables of `seqs`, int32 [n][widest], filled up with -1."""
        p, n, ids = _ints(seqs)
        need = array("i", [0])
        self._ok(self.lib.l3p_paged_tables(self.h, n, p, 0, None, need.buffer_info()[0]), "tables")
        out = np.empty((n, need[0]), np.int32)
        self._ok(self.lib.l3p_paged_tables(self.h, n, p, need[0], out.ctypes.data, None), "tables")
        return out

    def free_pages(self) -> int:
        n = C.c_int()
        self._ok(self.lib.l3p_paged_free_pages(self.h, C.byref(n)), "free_pages")
        return n.value

    def compact(self, stream=None) -> int:
        """Moves the pages in use to the front of the pool; returns how many there are."""
        n = C.c_int()
        self._ok(self.lib.l3p_paged_compact(self.h, C.byref(n), self._stream(stream)), "compact")
        return n.value

    # -- a step ----------------------------------------------------------------------
    def begin(self, seqs, n_new, stream=None) -> None:
        """Begins a batch: sequence seqs[i] grows by n_new[i] tokens."""
        p, n, ids = _ints(seqs)
        q, m, new = _ints(n_new)
        if n != m:
            raise ValueError("seqs and n_new differ in length")
        self._ok(self.lib.l3p_paged_begin(self.h, n, p, q, self._stream(stream)), "begin")
        self.n_tokens = sum(new)

    def set_rope(self, max_pos: int, layout: str = "interleaved", rotary_dim: int = 0, scaling: str = "none",
                 theta: float = 0.0, theta_swa: float = 0.0, factor: float = 1.0, low_freq: float = 0.0,
                 high_freq: float = 0.0, beta_fast: float = 0.0, beta_slow: float = 0.0, original_len: int = 0,
                 attn_factor: float = 0.0, rms_norm_eps: float = 0.0, q_norm=None, k_norm=None) -> None:
        """Rotary tables and norm weights ([n_layers][head_dim] float32) of rope_append_dev."""
        if layout not in LAYOUTS or scaling not in SCALINGS:
            raise ValueError(f"layout {layout!r}, scaling {scaling!r}")
        norms = []
        for w in (q_norm, k_norm):
            w = None if w is None else np.ascontiguousarray(w, np.float32)
            if w is not None and w.shape != (self.n_layers, self.head_dim):
                raise ValueError(f"norm weights of shape {w.shape}, not {(self.n_layers, self.head_dim)}")
            norms.append(w)
        rc = PagedRopeConfig(max_pos, LAYOUTS[layout], rotary_dim, SCALINGS[scaling], theta, theta_swa, factor, low_freq,
                             high_freq, beta_fast, beta_slow, original_len, attn_factor, rms_norm_eps,
                             *(None if w is None else w.ctypes.data for w in norms))
        self._ok(self.lib.l3p_paged_set_rope(self.h, C.byref(rc)), "set_rope")

    def _rows(self, t, heads: int, name: str) -> tuple[int, int]:
        """Address and token stride of rows [n_tokens or more][heads][head_dim]."""
        if t.dtype != self.dtype or t.get_device() != self.device:
            raise TypeError(f"{name}: a {self.dtype} tensor on cuda:{self.device}, not {t.dtype} on {t.device}")
        shape = t.shape
        if len(shape) != 3 or shape[0] < self.n_tokens or shape[1] != heads or shape[2] != self.head_dim:
            raise ValueError(f"{name}: shape {tuple(shape)}, not ({self.n_tokens}, {heads}, {self.head_dim})")
        stride, head, one = t.stride()
        if one != 1 or (heads > 1 and head != self.head_dim):
            raise ValueError(f"{name}: the heads of a token are not dense")
        if shape[0] < 2:
            stride = 0
        elif stride < heads * self.head_dim:
            raise ValueError(f"{name}: tokens {stride} values apart, rows of {heads * self.head_dim}")
        return t.data_ptr(), stride

    def rope_append_dev(self, layer, q, k, v, q_out, stream=None) -> None:
        """Rotates the batch's q (into q_out, which may be q) and k rows, and writes k and v into the pages."""
        self._ok(self.lib.l3p_paged_rope_append_dev(
            self.h, layer, *self._rows(q, self.n_heads, "q"), *self._rows(k, self.n_kv_heads, "k"),
            *self._rows(v, self.n_kv_heads, "v"), *self._rows(q_out, self.n_heads, "q_out"), self._stream(stream)),
            "rope_append_dev")

    def append_dev(self, layer, k, v, stream=None) -> None:
        """Writes the batch's k (already rotated) and v rows into the pages."""
        self._ok(self.lib.l3p_paged_append_dev(self.h, layer, *self._rows(k, self.n_kv_heads, "k"),
                                               *self._rows(v, self.n_kv_heads, "v"), self._stream(stream)), "append_dev")

    def attn_dev(self, layer, q, out, stream=None) -> None:
        """Attention of the batch's tokens over their sequences."""
        heads = self.n_heads
        qp, qs = self._rows(q, heads, "q")
        op, os_ = self._rows(out, heads, "out")
        rc = self.lib.l3p_paged_attn_dev(self.h, layer, qp, qs, op, os_, self._stream(stream))
        if rc:
            self._ok(rc, "attn_dev")

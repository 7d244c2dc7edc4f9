"""The paged cache on the GPU against a plain implementation in 64 bits.

Tolerances.  Scores of bf16 rows are sums of exact products in fp32; of fp32
rows, three TF32 products leave at most 2^-20 of each product.  A score that is
off by ds moves a softmax weight by a factor within 1 +- 2 ds, so an output by
2 ds sum(p |v|).  With bf16 pages the weights are rounded once (2^-8) ahead of
the second product and the output once (2^-8).  `ds` counts the accumulation too,
2^-23 per term of head_dim terms at the sum's size (far above what it is), and
2^-21 of the score for the scaling and the exponential.
"""
import math
import random

import numpy as np
import pytest

from llama3pure_b200.attn import AttnError

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch

    return torch


def _cache(**kw):
    from llama3pure_b200.paged import PagedCache

    base = dict(n_layers=2, n_heads=8, n_kv_heads=2, head_dim=128, page_size=16, n_pages=64, max_seqs=16, max_tokens=512)
    base.update(kw)
    return PagedCache(**base)


def _type(torch, dtype):
    return torch.bfloat16 if dtype == "bf16" else torch.float32


def _want(torch, q, k, v, past, window=0, scale=None):
    """Exact outputs of new tokens q [n][H][d] over k, v [past + n][Hkv][d], and their tolerance."""
    n, H, d = q.shape
    G = H // k.shape[1]
    scale = 1 / math.sqrt(d) if scale is None else scale
    out, tol = torch.empty(n, H, d, dtype=torch.float64, device=q.device), torch.empty(n, H, d, dtype=torch.float64, device=q.device)
    t = torch.arange(past, past + n, device=q.device)[:, None]
    j = torch.arange(k.shape[0], device=q.device)[None]
    seen = (j <= t) & ((j > t - window) if window else True)
    bf16 = q.dtype == torch.bfloat16
    for h in range(H):
        kh, vh, qh = k[:, h // G].double(), v[:, h // G].double(), q[:, h].double()
        s = (qh @ kh.T * scale).masked_fill(~seen, -math.inf)
        p = torch.softmax(s, -1)
        out[:, h] = p @ vh
        size = (qh.abs() @ kh.abs().T * abs(scale)).masked_fill(~seen, 0).amax(-1, keepdim=True)
        ds = size * ((0 if bf16 else 2**-20) + d * 2**-23 + 2**-21)
        pv = p @ vh.abs()
        tol[:, h] = 2 * ds * pv + 2**-22 * pv
        if bf16:
            tol[:, h] += 2**-8 * pv + 2**-8 * out[:, h].abs()
    return out, tol


def _near(got, want, tol, what=""):
    err = (got.double() - want).abs()
    assert bool((err <= tol + 1e-30).all()), f"{what}: {float((err / (tol + 1e-30)).max()):.3g} times the tolerance"


class Books:
    """What the cache should hold: every sequence's rows as lists of tensors, one per layer."""

    def __init__(self, torch, cache, seed=0):
        self.torch, self.c, self.rows = torch, cache, {}
        self.g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(self, *shape):
        return self.torch.randn(*shape, generator=self.g, device="cuda").to(self.c.dtype)

    def new(self):
        s = self.c.new_seq()
        self.rows[s] = [self.randn(0, 2, self.c.n_kv_heads, self.c.head_dim) for _ in range(self.c.n_layers)]
        return s

    def step(self, seqs, n_new, attend=True, window=lambda layer: 0, scale=None, stream=None):
        """One step over all layers: q, k, v lie in one tensor, as a projection leaves them."""
        torch, c = self.torch, self.c
        c.begin(seqs, n_new, stream)
        n, H, K, d = sum(n_new), c.n_heads, c.n_kv_heads, c.head_dim
        for layer in range(c.n_layers):
            qkv = self.randn(n, H + 2 * K, d)
            q, k, v = qkv[:, :H], qkv[:, H:H + K], qkv[:, H + K:]
            out = torch.full((n + 3, H, d), 7.0, device="cuda", dtype=c.dtype)
            if stream is not None:
                torch.cuda.synchronize()
            c.append_dev(layer, k, v, stream)
            if attend:
                c.attn_dev(layer, q, out, stream)
            c.check(stream)
            assert bool((out[n:] == 7.0).all()), "rows behind the last token"
            at = 0
            for s, m in zip(seqs, n_new):
                old = self.rows[s][layer]
                new = torch.stack([k[at:at + m], v[at:at + m]], 1)
                self.rows[s][layer] = torch.cat([old, new])
                if attend and m:
                    kv = self.rows[s][layer]
                    want, tol = _want(torch, q[at:at + m], kv[:, 0], kv[:, 1], len(old), window(layer), scale)
                    _near(out[at:at + m], want, tol, f"sequence {s}, {m} tokens on {len(old)}, layer {layer}")
                at += m

    def verify(self):
        """Lengths, tables and every row of every sequence."""
        c, st, seen = self.c, self.c.storage(), set()
        for s, rows in self.rows.items():
            n = len(rows[0])
            assert c.length(s) == n
            table = c.tables([s])[0]
            assert len(table) == -(-n // c.cfg.page_size) and len(set(table.tolist())) == len(table)
            seen |= set(table.tolist())
            if n:
                idx = self.torch.from_numpy(table).cuda().long()
                for layer in range(c.n_layers):
                    got = st[idx, layer].permute(0, 3, 1, 2, 4).reshape(-1, 2, c.n_kv_heads, c.head_dim)[:n]
                    assert bool((got == rows[layer]).all()), f"rows of sequence {s}"
        assert c.free_pages() == c.cfg.n_pages - len(seen)


SHAPES = [  # heads, KV heads, head_dim
    (32, 8, 64), (4, 4, 64), (8, 2, 128), (6, 2, 128), (5, 1, 128), (8, 8, 128), (16, 2, 128), (8, 1, 256), (6, 3, 256),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv,dim", SHAPES)
def test_single_tokens_ragged(torch, dtype, heads, kv, dim):
    """Lengths around tile and page ends, single tokens of every sequence and of some."""
    with _cache(n_heads=heads, n_kv_heads=kv, head_dim=dim, dtype=dtype, n_pages=160, n_layers=1) as c:
        b = Books(torch, c, heads)
        lengths = [0, 1, 14, 15, 16, 17, 31, 32, 100, 255, 256, 300]
        seqs = [b.new() for _ in lengths]
        for at in range(0, 300, 150):
            new = [max(0, min(n - at, 150)) for n in lengths]
            for i in range(0, len(seqs), 3):
                b.step(seqs[i:i + 3], new[i:i + 3], attend=False)
        b.step(seqs, [1] * len(seqs))
        b.step(seqs[::2], [1] * len(seqs[::2]))
        b.step(seqs, [i % 2 for i in range(len(seqs))])
        b.verify()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv,dim", SHAPES)
@pytest.mark.parametrize("page", [16, 128])
def test_chunks(torch, dtype, heads, kv, dim, page):
    """Chunks of every path: a few tokens, whole tiles, ragged ones, beside single tokens and none."""
    with _cache(n_heads=heads, n_kv_heads=kv, head_dim=dim, dtype=dtype, page_size=page, n_pages=2048 // page, n_layers=1,
                max_tokens=1024) as c:
        b = Books(torch, c, dim + page)
        seqs = [b.new() for _ in range(5)]
        b.step(seqs, [3, 0, 129, 1, 40])
        b.step(seqs, [257, 1, 2, 5, 0])
        b.step(seqs, [1, 8, 130, 64, 300])
        b.step(seqs[::-1], [7, 1, 1, 33, 63])
        b.verify()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("window", [1, 16, 50, 1000])
def test_sliding_window_layers(torch, dtype, dim, window):
    """Layers 0 and 1 of pattern 3 look back `window` positions, layer 2 sees everything."""
    with _cache(n_heads=4, n_kv_heads=1, head_dim=dim, dtype=dtype, n_layers=3, is_gemma3=1, swa_window=window, swa_pattern=3,
                n_pages=200, max_tokens=600) as c:
        b = Books(torch, c, window)
        seqs = [b.new() for _ in range(3)]
        win = lambda layer: window if layer % 3 < 2 else 0  # noqa: E731
        b.step(seqs, [390, 17, 0], window=win)
        b.step(seqs, [1, 1, 1], window=win)
        b.step(seqs, [150, 5, 260], window=win)
        b.step(seqs, [1, 4, 1], window=win)


@pytest.mark.parametrize("dtype,heads,kv,dim,lengths", [
    ("f32", 32, 8, 128, [9000, 3]), ("f32", 16, 8, 128, [66100]), ("bf16", 32, 8, 128, [20000]), ("bf16", 8, 1, 64, [33000]), ("f32", 8, 1, 256, [5000, 1]),
    ("bf16", 8, 1, 256, [7000]), ("bf16", 16, 8, 128, [40, 6000, 1, 2500, 777]),
])
def test_long_sequences_are_split_and_joined(torch, dtype, heads, kv, dim, lengths):
    with _cache(n_heads=heads, n_kv_heads=kv, head_dim=dim, dtype=dtype, n_layers=1, n_pages=sum(lengths) // 64 + 20, page_size=64,
                max_tokens=max(lengths)) as c:
        b = Books(torch, c, dim)
        seqs = []
        for n in lengths:
            seqs.append(b.new())
            b.step(seqs[-1:], [n], attend=False)
        b.step(seqs, [1] * len(seqs))
        b.step(seqs, [3] * len(seqs))
        b.step(seqs[:1], [70])
        for _ in range(3):  # tickets return to zero
            b.step(seqs, [1] * len(seqs))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_scale(torch, dtype):
    with _cache(dtype=dtype, scale=0.3, n_layers=1) as c:
        b = Books(torch, c)
        s = b.new()
        b.step([s], [60], scale=0.3)
        b.step([s], [1], scale=0.3)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_values_that_are_not_attended_never_matter(torch, dtype, dim, bad):
    """Pages full of `bad` behind and before the rows in use, and `bad` in K and V of later tokens of a chunk."""
    with _cache(n_heads=4, n_kv_heads=1, head_dim=dim, dtype=dtype, n_layers=2, is_gemma3=1, swa_window=40, swa_pattern=2, n_pages=64,
                max_tokens=700) as c:
        c.storage().fill_(bad)
        b = Books(torch, c)
        seqs = [b.new(), b.new()]
        win = lambda layer: 40 if layer == 0 else 0  # noqa: E731
        b.step(seqs, [201, 3], window=win)
        b.step(seqs, [1, 1], window=win)
        b.step(seqs, [4, 1], window=win)
        # the last three of 160 and of 5 new tokens are bad: the rows before them do not see it
        for n in (160, 5):
            past = len(b.rows[seqs[0]][1])
            c.begin(seqs[:1], [n])
            q, k, v = b.randn(n, 4, dim), b.randn(n, 1, dim), b.randn(n, 1, dim)
            k[-3:] = bad
            v[-3:, :, 5:9] = bad
            for layer in (0, 1):
                out = torch.empty_like(q)
                c.append_dev(layer, k, v)
                c.attn_dev(layer, q, out)
                c.check()
                rows = torch.cat([b.rows[seqs[0]][layer], torch.stack([k, v], 1)])[:past + n - 3]
                want, tol = _want(torch, q[:-3], rows[:, 0], rows[:, 1], past, win(layer))
                _near(out[:-3], want, tol, f"{n} tokens, layer {layer}")
            c.truncate(seqs[0], past)
        # V alone: rows that attend to it have it in its columns and nowhere else
        for n in (160, 5):
            past = len(b.rows[seqs[0]][1])
            c.begin(seqs[:1], [n])
            q, k, v = b.randn(n, 4, dim), b.randn(n, 1, dim), b.randn(n, 1, dim)
            v[-3, :, 5:9] = bad
            c.append_dev(1, k, v)
            out = torch.empty_like(q)
            c.attn_dev(1, q, out)
            c.check()
            rows = torch.cat([b.rows[seqs[0]][1], torch.stack([k, v], 1)])
            clean = rows.clone()
            clean[-3, 1, :, 5:9] = 0
            want, tol = _want(torch, q, clean[:, 0], clean[:, 1], past)
            assert bool(out[-3:, :, 5:9].float().isfinite().logical_not().all())
            keep = torch.ones(n, 1, dim, dtype=torch.bool, device="cuda").expand(n, 4, dim).clone()
            keep[-3:, :, 5:9] = False
            _near(out[keep], want[keep], tol[keep], f"columns beside, {n} tokens")
            c.truncate(seqs[0], past)


def test_empty_batches(torch):
    with _cache(n_layers=1) as c:
        b = Books(torch, c)
        c.begin([], [])
        e = torch.empty(0, 8, 128, device="cuda")
        kv = torch.empty(0, 2, 128, device="cuda")
        n0 = c.launch_count()
        c.append_dev(0, kv, kv)
        c.attn_dev(0, e, e)
        s = b.new()
        b.step([s], [0])
        assert c.launch_count() == n0
        b.step([s], [1])


@pytest.mark.parametrize("seed", range(4))
def test_pages_under_random_use(torch, seed):
    """Forks, copies, cuts, frees, compaction and steps in any order: every sequence keeps its rows."""
    rng = random.Random(seed)
    dtype = rng.choice(["f32", "bf16"])
    with _cache(n_heads=4, n_kv_heads=2, head_dim=64, n_pages=90, max_seqs=12, max_tokens=200, dtype=dtype, page_size=rng.choice([16, 32])) as c:
        b = Books(torch, c, seed)
        for i in range(60):
            live = sorted(b.rows)
            do = rng.choice(["new", "fork", "copy", "cut", "free", "compact", "step", "step", "step"])
            try:
                if do == "new" or not live:
                    b.new()
                elif do == "fork":
                    s = rng.choice(live)
                    n = rng.choice([-1, rng.randint(0, c.length(s))])
                    for ch in c.fork(s, rng.randint(1, 3), n):
                        b.rows[ch] = [r[:len(r) if n < 0 else n] for r in b.rows[s]]
                elif do == "copy":
                    some = rng.sample(live, rng.randint(1, len(live)))
                    for s, ch in zip(some, c.copy(some)):
                        b.rows[ch] = list(b.rows[s])
                elif do == "cut":
                    s = rng.choice(live)
                    n = rng.randint(0, c.length(s))
                    c.truncate(s, n)
                    b.rows[s] = [r[:n] for r in b.rows[s]]
                elif do == "free":
                    gone = rng.sample(live, rng.randint(1, max(1, len(live) // 2)))
                    c.free(gone)
                    for s in gone:
                        del b.rows[s]
                elif do == "compact":
                    used = c.compact()
                    assert used == c.cfg.n_pages - c.free_pages()
                    if b.rows:
                        assert int(c.tables(sorted(b.rows)).max(initial=-1)) < used
                else:
                    some = rng.sample(live, rng.randint(1, len(live)))
                    b.step(some, [rng.choice([0, 1, 1, 5, 30]) for _ in some], attend=i % 2 == 0)
            except AttnError as e:
                assert e.code == -4  # the pool or the sequence ids are used up: nothing has changed
            b.verify()


def test_last_holder_of_a_shared_page_keeps_it(torch):
    with _cache(n_layers=1, n_pages=20) as c:
        b = Books(torch, c)
        s = b.new()
        b.step([s], [20], attend=False)
        children = c.fork(s, 2)
        for ch in children:
            b.rows[ch] = list(b.rows[s])
        t = c.tables([s])[0].tolist()
        b.step([s] + children, [1, 2, 1])
        tables = c.tables([s] + children)
        assert tables[:, 0].tolist() == [t[0]] * 3
        assert sorted(tables[:, 1].tolist()) == [t[1], 2, 3] and tables[2, 1] == t[1]
        b.verify()


ROPES = [
    dict(layout="interleaved"), dict(layout="half"), dict(layout="half", rotary=32), dict(layout="interleaved", rotary=20),
    dict(layout="half", rotary=6, norm=True), dict(layout="interleaved", scaling="linear", factor=4.0), dict(layout="half", scaling="bands", factor=8.0, norm=True),
    dict(layout="half", scaling="yarn", factor=16.0, rotary=64), dict(layout="interleaved", scaling="yarn", factor=4.0, attn=1.25),
]


def _turned(torch, x, pos, dim, layout, rotary, scaling, factor, attn, theta, original, w=None):
    """Exact rotation of rows x [n][heads][dim]."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + 1e-5) * w.double()
    r = rotary or dim
    f, mult = [theta ** (-2 * i / r) for i in range(r // 2)], 1.0
    if scaling == "linear":
        f = [v / factor for v in f]
    elif scaling == "bands":
        g = []
        for v in f:
            wave = 2 * math.pi / v
            if wave < original / 4.0:
                g.append(v)
            elif wave > original / 1.0:
                g.append(v / factor)
            else:
                mix = (original / wave - 1.0) / 3.0
                g.append((1 - mix) * v / factor + mix * v)
        f = g
    elif scaling == "yarn":
        at = lambda n: r * math.log(original / (n * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        lo, hi = max(math.floor(at(32)), 0), min(math.ceil(at(1)), r - 1)
        ramp = [min(1.0, max(0.0, (i - lo) / ((hi - lo) or 0.001))) for i in range(r // 2)]
        f = [v * (1 - m) + v / factor * m for v, m in zip(f, ramp)]
        mult = attn or 0.1 * math.log(factor) + 1
    ang = pos[:, None].double() * torch.tensor(f, dtype=torch.float64, device=x.device)
    c, s = torch.cos(ang)[:, None] * mult, torch.sin(ang)[:, None] * mult
    y = x.clone()
    if layout == "half":
        a, b = x[..., :r // 2], x[..., r // 2:r]
        y[..., :r // 2], y[..., r // 2:r] = a * c - b * s, a * s + b * c
    else:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y[..., 0:r:2], y[..., 1:r:2] = a * c - b * s, a * s + b * c
    return y


def _rope_near(torch, got, want, dtype, what):
    # fp32: cosine and sine rounded (2^-24 each), two products and a sum, and with a norm a mean over the row, a square root, a
    # division and two products: within 2^-20 of a pair's size, which the row's largest value bounds.  bf16: and one rounding, 2^-8.
    size = want.abs().amax(-1, keepdim=True) * 2
    tol = size * 2**-20 + (want.abs() * 2**-8 if dtype == "bf16" else 0)
    _near(got, want, tol, what)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("kw", ROPES, ids=lambda k: "-".join(str(v) for v in k.values()))
def test_rotary_and_append(torch, dtype, dim, kw):
    kw = dict(rotary=0, scaling="none", factor=1.0, attn=0.0, norm=False) | kw
    original = 512
    with _cache(n_heads=6, n_kv_heads=2, head_dim=dim, dtype=dtype, n_layers=2, n_pages=400, max_tokens=3000) as c:
        b = Books(torch, c, dim)
        rng = np.random.default_rng(5)
        wq, wk = (1 + 0.1 * rng.standard_normal((2, dim))).astype(np.float32), (1 + 0.1 * rng.standard_normal((2, dim))).astype(np.float32)
        norm = dict(q_norm=wq, k_norm=wk) if kw["norm"] else {}
        c.set_rope(max_pos=4000, layout=kw["layout"], rotary_dim=kw["rotary"], scaling=kw["scaling"], factor=kw["factor"], theta=10000.0,
                   original_len=original, attn_factor=kw["attn"], **norm)
        seqs = [b.new() for _ in range(3)]
        c.begin(seqs, [2900, 0, 17])
        for new in ([5, 1, 0], [1, 1, 1], [700, 100, 30], [5, 900, 400]):
            past = [c.length(s) for s in seqs]
            c.begin(seqs, new)
            n = sum(new)
            pos = torch.cat([torch.arange(p, p + m, device="cuda") for p, m in zip(past, new)])
            for layer in (0, 1):
                qkv = b.randn(n, 10, dim)
                q, k, v = qkv[:, :6], qkv[:, 6:8], qkv[:, 8:]
                args = (pos, dim, kw["layout"], kw["rotary"], kw["scaling"], kw["factor"], kw["attn"], 10000.0, original)
                w = [torch.from_numpy(x[layer]).cuda() if kw["norm"] else None for x in (wq, wk)]
                want_q, want_k = _turned(torch, q, *args, w=w[0]), _turned(torch, k, *args, w=w[1])
                want_v = v.clone()
                out = torch.empty(n, 6, dim, device="cuda", dtype=c.dtype)
                c.rope_append_dev(layer, q, k, v, out)
                c.check()
                _rope_near(torch, out, want_q, dtype, "q")
                c.rope_append_dev(layer, q, k, v, q)  # in place
                c.check()
                assert bool((q == out).all())
                st, at = c.storage(), 0
                for s, p, m in zip(seqs, past, new):
                    if m:
                        t = torch.from_numpy(c.tables([s])[0]).cuda().long()
                        rows = st[t, layer].permute(0, 3, 1, 2, 4).reshape(-1, 2, 2, dim)[p:p + m]
                        _rope_near(torch, rows[:, 0], want_k[at:at + m], dtype, "k")
                        assert bool((rows[:, 1] == want_v[at:at + m]).all())
                    at += m


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_rotary_large_tokens(torch, dtype, layout):
    """Tokens of which two do not fit a CTA's shared memory."""
    with _cache(n_heads=96, n_kv_heads=8, head_dim=256, dtype=dtype, n_layers=1, n_pages=20, max_tokens=200) as c:
        b = Books(torch, c)
        wq, wk = (np.linspace(0.5, 1.5, 256, dtype=np.float32)[None] * f for f in (1, -1))
        c.set_rope(max_pos=200, layout=layout, theta=10000.0, q_norm=wq, k_norm=wk)
        s = b.new()
        for past, n in ((0, 1), (1, 130)):
            c.begin([s], [n])
            q, k, v = b.randn(n, 96, 256), b.randn(n, 8, 256), b.randn(n, 8, 256)
            out = torch.empty_like(q)
            c.rope_append_dev(0, q, k, v, out)
            c.check()
            pos = torch.arange(past, past + n, device="cuda")
            args = (pos, 256, layout, 0, "none", 1.0, 0.0, 10000.0, 0)
            _rope_near(torch, out, _turned(torch, q, *args, w=torch.from_numpy(wq[0]).cuda()), dtype, "q")
            t = torch.from_numpy(c.tables([s])[0]).cuda().long()
            rows = c.storage()[t, 0].permute(0, 3, 1, 2, 4).reshape(-1, 2, 8, 256)[past:past + n]
            _rope_near(torch, rows[:, 0], _turned(torch, k, *args, w=torch.from_numpy(wk[0]).cuda()), dtype, "k")
            assert bool((rows[:, 1] == v).all())


def test_rotary_far_positions_and_window_layers(torch):
    """Angles of far positions keep their precision; sliding-window layers use their own, unscaled table."""
    with _cache(n_heads=4, n_kv_heads=1, head_dim=64, n_layers=2, is_gemma3=1, swa_window=8, swa_pattern=2, page_size=128, n_pages=4100,
                max_tokens=600000) as c:
        b = Books(torch, c)
        c.set_rope(max_pos=524288, layout="half", scaling="linear", factor=8.0, theta=1e6, theta_swa=1e4)
        s = b.new()
        c.begin([s], [524280])
        c.begin([s], [8])
        pos = torch.arange(524280, 524288, device="cuda")
        for layer in (0, 1):
            q, k, v = b.randn(8, 4, 64), b.randn(8, 1, 64), b.randn(8, 1, 64)
            out = torch.empty_like(q)
            c.rope_append_dev(layer, q, k, v, out)
            c.check()
            args = ("none", 1.0, 0.0, 1e4) if layer == 0 else ("linear", 8.0, 0.0, 1e6)
            _rope_near(torch, out, _turned(torch, q, pos, 64, "half", 0, *args, 0), "f32", f"layer {layer}")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_serving_loop_on_another_stream(torch, dtype):
    """Prompts in chunks beside decoding sequences, forks of a prompt, frees and compaction, on a stream of the caller's: every
    output equals attention over the whole rotated history."""
    heads, kv, dim = 8, 2, 128
    s = torch.cuda.Stream()
    with _cache(n_heads=heads, n_kv_heads=kv, head_dim=dim, dtype=dtype, n_layers=2, n_pages=80, max_tokens=256) as c, torch.cuda.stream(s):
        c.set_rope(max_pos=1000, layout="interleaved", scaling="bands", factor=8.0, original_len=256)
        g = torch.Generator(device="cuda").manual_seed(1)
        hist = {}

        def step(seqs, new):
            c.begin(seqs, new)
            n = sum(new)
            for layer in range(2):
                qkv = torch.randn(n, heads + 2 * kv, dim, generator=g, device="cuda").to(c.dtype)
                q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
                qr, out = torch.empty(n, heads, dim, device="cuda", dtype=c.dtype), torch.empty(n, heads, dim, device="cuda", dtype=c.dtype)
                c.rope_append_dev(layer, q, k, v, qr)
                c.attn_dev(layer, qr, out)
                c.check()
                at = 0
                for x, m in zip(seqs, new):
                    past = len(hist[x][layer])
                    pos = torch.arange(past, past + m, device="cuda")
                    kr = _turned(torch, k[at:at + m], pos, dim, "interleaved", 0, "bands", 8.0, 0.0, 500000.0, 256)
                    # the rounded row that the page holds: the table's cosines are the oracle's within 2^-24, so take the page's own
                    t = torch.from_numpy(c.tables([x])[0]).cuda().long()
                    row = c.storage()[t, layer].permute(0, 3, 1, 2, 4).reshape(-1, 2, kv, dim)[past:past + m]
                    _rope_near(torch, row[:, 0], kr, dtype, "k")
                    hist[x][layer] = torch.cat([hist[x][layer], row.clone()])
                    if m:
                        h = hist[x][layer]
                        want, tol = _want(torch, qr[at:at + m], h[:, 0], h[:, 1], past)
                        _near(out[at:at + m], want, tol, f"sequence {x}")
                    at += m

        def new():
            x = c.new_seq()
            hist[x] = [torch.empty(0, 2, kv, dim, device="cuda", dtype=c.dtype) for _ in range(2)]
            return x

        a, b = new(), new()
        step([a, b], [100, 7])
        step([a, b], [1, 90])
        kids = c.fork(a, 3)
        for x in kids:
            hist[x] = list(hist[a])
        step([a, b] + kids, [1, 1, 1, 1, 4])
        step([b] + kids, [130, 1, 1, 1])
        c.free([a, kids[0]])
        c.compact()
        step([b] + kids[1:], [1, 60, 1])
        d = c.copy([b])[0]
        hist[d] = list(hist[b])
        c.truncate(b, 50)
        hist[b] = [x[:50] for x in hist[b]]
        step([b, d], [20, 1])


def test_captured_step_serves_later_batches(torch):
    """One graph of a decoding step, replayed on other sequences and lengths; a batch that it cannot serve is reported."""
    with _cache(n_heads=8, n_kv_heads=2, head_dim=64, dtype="bf16", n_layers=2, n_pages=600, max_tokens=4096, page_size=16) as c:
        b = Books(torch, c)
        c.set_rope(max_pos=6000, layout="half")
        seqs = [b.new() for _ in range(6)]
        for x, n in zip(seqs, [5, 900, 17, 64, 333, 2000]):
            c.begin([x], [n])
            for layer in range(2):
                k, v = b.randn(n, 2, 64), b.randn(n, 2, 64)
                c.append_dev(layer, k, v)
        c.begin(seqs, [1] * 6)
        q, k, v = b.randn(6, 8, 64), b.randn(6, 2, 64), b.randn(6, 2, 64)
        qr, outs = torch.empty_like(q), [torch.empty_like(q) for _ in range(2)]

        def layers():
            for layer in range(2):
                c.rope_append_dev(layer, q, k, v, qr)
                c.attn_dev(layer, qr, outs[layer])

        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            layers()
            c.check()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                layers()
            for some in (seqs, seqs[:2], seqs[::-1], seqs[5:], seqs[1:5]):
                c.begin(some, [1] * len(some))
                for t in (q, k, v):
                    t.copy_(b.randn(*t.shape))
                layers()
                want = [o.clone() for o in outs]
                for o in outs:
                    o.fill_(3.0)
                graph.replay()
                c.check()
                for o, w in zip(outs, want):
                    assert bool((o[:len(some)] == w[:len(some)]).all())
                    assert bool((o[len(some):] == 3.0).all())
            for some, new in ((seqs, [2, 1, 1, 1, 1, 1]), (seqs[:1], [200]), (seqs[:2], [4, 1])):
                c.begin(some, new)
                graph.replay()
                with pytest.raises(AttnError) as e:
                    c.check()
                assert e.value.code == -1
            c.begin(seqs, [1] * 6)
            graph.replay()
            c.check()
            del graph


@pytest.mark.parametrize("dtype,dim", [("f32", 64), ("f32", 128), ("bf16", 64), ("bf16", 128), ("bf16", 256)])
def test_captured_chunks(torch, dtype, dim):
    """A captured batch of chunks beside single tokens, replayed on smaller ones, with parts to be joined; one that is larger is
    reported and written nothing for."""
    with _cache(n_heads=8, n_kv_heads=2, head_dim=dim, dtype=dtype, n_layers=1, n_pages=800, max_tokens=6000, page_size=16) as c:
        b = Books(torch, c)
        seqs = [b.new() for _ in range(3)]
        for x, n in zip(seqs, [5000, 900, 17]):
            b.step([x], [n], attend=False)
        big, small = [200, 130, 1], [60, 40, 1]
        c.begin(seqs, big)
        q, out = b.randn(sum(big), 8, dim), torch.empty(sum(big), 8, dim, device="cuda", dtype=c.dtype)
        kv = [b.randn(sum(big), 2, dim) for _ in range(2)]
        s = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            c.append_dev(0, *kv)
            c.attn_dev(0, q, out)
            c.check()
            want = out.clone()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                c.append_dev(0, *kv)
                c.attn_dev(0, q, out)
            for new in (big, small):
                for x, n in zip(seqs, [5000, 900, 17]):
                    c.truncate(x, n)
                c.begin(seqs, new)
                out.fill_(9.0)
                graph.replay()
                c.check()
                got = out.clone()
                out.fill_(9.0)
                c.attn_dev(0, q, out)
                c.check()
                assert bool((got == out).all()) and bool((got[sum(new):] == 9.0).all())
                if new == big:
                    assert bool((got == want).all())
            for new in ([200, 131, 1], [600, 1, 1], [1, 1, 1]):
                c.begin(seqs, new)
                out.fill_(9.0)
                graph.replay()
                with pytest.raises(AttnError) as e:
                    c.check()
                assert e.value.code == -1
                if new != [1, 1, 1]:  # single tokens alone: the captured row launch meets no chunk, and neither writes
                    assert bool((out == 9.0).all())
            del graph


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 64), (32, 8, 128), (6, 3, 256), (71, 1, 64), (32, 1, 128), (20, 1, 256)])
def test_few_tokens_of_every_sequence(torch, dtype, heads, kv, dim):
    """As many sequences as the cache takes, with token counts around the ends of each path, alone and beside a long chunk."""
    with _cache(n_heads=heads, n_kv_heads=kv, head_dim=dim, dtype=dtype, n_layers=1, max_seqs=12, n_pages=400, max_tokens=420) as c:
        b = Books(torch, c, dim)
        seqs = [b.new() for _ in range(12)]
        b.step(seqs, [20 + i for i in range(12)])
        for n in (2, 3, 4, 5, 8, 9, 16, 17, 32, 33):
            b.step(seqs, [n] * 12)
            for x in seqs:
                c.truncate(x, 20)
                b.rows[x] = [r[:20] for r in b.rows[x]]
        b.step(seqs, [16] * 11 + [140])
        b.step(seqs, [1, 2, 3, 4, 5, 8, 9, 16, 17, 32, 33, 34])


@pytest.mark.parametrize("dtype,largest", [("f32", 16), ("bf16", 4)])
def test_captured_few_tokens(torch, dtype, largest):
    """A captured batch of few tokens serves up to the largest count of the same path."""
    with _cache(n_heads=8, n_kv_heads=2, head_dim=128, dtype=dtype, n_layers=1, max_seqs=8, n_pages=400, max_tokens=500) as c:
        b = Books(torch, c)
        seqs = [b.new() for _ in range(8)]
        past = [10 + 40 * i for i in range(8)]
        for x, n in zip(seqs, past):
            b.step([x], [n], attend=False)
        n = largest * 8
        q, out = b.randn(n, 8, 128), torch.empty(n, 8, 128, device="cuda", dtype=c.dtype)
        kv = [b.randn(n, 2, 128) for _ in range(2)]
        c.begin(seqs, [largest] * 8)
        s = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            c.append_dev(0, *kv)
            c.attn_dev(0, q, out)
            c.check()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                c.append_dev(0, *kv)
                c.attn_dev(0, q, out)
            for new in ([largest] * 8, [3] * 8, [largest, 1, 2, 3, 1, 1, 1, 1], [0, largest, 0, 1, 0, 2, 0, 3]):
                for x, m in zip(seqs, past):
                    c.truncate(x, m)
                c.begin(seqs, new)
                out.fill_(9.0)
                graph.replay()
                c.check()
                got = out.clone()
                out.fill_(9.0)
                c.attn_dev(0, q, out)
                c.check()
                assert bool((got == out).all()) and bool((got[sum(new):] == 9.0).all())
            del graph


def test_calls_during_capture_are_refused(torch):
    with _cache(n_layers=1) as c:
        b = Books(torch, c)
        s = b.new()
        b.step([s], [20], attend=False)
        stream = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        codes = []
        with torch.cuda.graph(graph, stream=stream):
            for call in (lambda: c.begin([s], [1]), lambda: c.copy([s]), lambda: c.compact()):
                with pytest.raises(AttnError) as e:
                    call()
                codes.append(e.value.code)
            torch.zeros(4, device="cuda")
        assert codes == [-1] * 3
        b.verify()
        b.step([s], [1])


def test_refusals_change_nothing(torch):
    with _cache(n_layers=1, n_pages=4, max_seqs=3, max_tokens=60, max_seq_len=50) as c:
        b = Books(torch, c)
        s, t = b.new(), b.new()
        q, kv = b.randn(8, 8, 128), b.randn(8, 2, 128)

        def code(f, *a, **k):
            with pytest.raises(AttnError) as e:
                f(*a, **k)
            return e.value.code

        assert code(c.attn_dev, 0, q, q) == -1  # no batch yet
        assert code(c.append_dev, 0, kv, kv) == -1
        assert code(c.begin, [s, s], [1, 1]) == -1
        assert code(c.begin, [s, 2], [1, 1]) == -2
        assert code(c.begin, [-1], [1]) == -2
        assert code(c.begin, [s], [-1]) == -1
        assert code(c.begin, [s], [51]) == -2       # max_seq_len
        assert code(c.begin, [s, t], [40, 21]) == -2  # max_tokens
        assert code(c.begin, [s, t], [33, 17]) == -4  # 3 + 2 pages of 4
        assert code(c.truncate, s, 1) == -2
        assert code(c.truncate, 2, 0) == -2
        assert code(c.fork, s, 1, 1) == -2
        assert code(c.fork, s, 2) == -4             # sequence ids
        assert code(c.free, [s, s]) == -1
        assert code(c.free, [7]) == -2
        assert code(c.copy, [s, s]) == -4
        assert code(c.copy, [2]) == -2
        assert code(c.length, 2) == -2
        b.verify()
        b.step([s], [8], attend=False)
        assert code(c.append_dev, 1, kv, kv) == -2
        assert code(c.attn_dev, -1, q, q) == -2
        assert code(c.rope_append_dev, 0, q, kv, kv, q) == -1  # no tables
        for bad in (dict(max_pos=0), dict(max_pos=9, rotary_dim=3), dict(max_pos=9, rotary_dim=130), dict(max_pos=9, theta=0.5),
                    dict(max_pos=9, scaling="linear", factor=0.5), dict(max_pos=9, scaling="bands", factor=2.0),
                    dict(max_pos=9, scaling="yarn", factor=2.0), dict(max_pos=9, scaling="bands", factor=2.0, original_len=9, low_freq=4.0, high_freq=2.0),
                    dict(max_pos=9, scaling="yarn", factor=float("nan"), original_len=9), dict(max_pos=9, q_norm=np.ones((1, 128), np.float32))):
            assert code(c.set_rope, **bad) == -1
        c.set_rope(max_pos=7)
        assert code(c.rope_append_dev, 0, q, kv, kv, q) == -2  # position 7
        lib, h = c.lib, c.h
        p = q.data_ptr()
        assert lib.l3p_paged_attn_dev(h, 0, p, 0, None, 0, None) == -1
        assert lib.l3p_paged_attn_dev(h, 0, p + 4, 0, p, 0, None) == -1      # alignment
        assert lib.l3p_paged_attn_dev(h, 0, p, 8 * 128 - 4, p, 0, None) == -1  # a stride below the row
        assert lib.l3p_paged_attn_dev(h, 0, p, 8 * 128 + 2, p, 0, None) == -1  # a stride off 16 bytes
        assert lib.l3p_paged_tables(h, 1, (np.array([s], np.int32)).ctypes.data, 0, np.zeros(1, np.int32).ctypes.data, None) == -2
        for bad in (q.half(), q.cpu(), q[:7], q[:, :4], q.transpose(0, 1), q[:1].expand(8, 8, 128)):
            with pytest.raises((TypeError, ValueError)):
                c.attn_dev(0, bad, q)
        with pytest.raises(ValueError):
            c.begin([s], [1, 1])
        b.verify()
        c.truncate(s, 8)
        assert code(c.attn_dev, 0, q, q) == -1  # the batch has ended
        b.step([s], [1])


def test_storage_keeps_the_cache(torch):
    import gc
    import weakref

    c = _cache(n_layers=1)
    gone = weakref.ref(c)
    st = c.storage()
    view = st[1:2]
    del c, st
    gc.collect()
    assert gone() is not None  # ahead of any use of the view
    assert not bool(view.any())
    del view
    gc.collect()
    assert gone() is None


def test_create_without_memory(torch):
    with pytest.raises(AttnError) as e:
        _cache(n_layers=64, n_heads=8, n_kv_heads=8, head_dim=256, page_size=128, n_pages=16000)  # 537 GB
    assert e.value.code == -4
    assert torch.zeros(4, device="cuda").sum().item() == 0


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("page", [32, 128])
@pytest.mark.parametrize("rotate", [False, True])
def test_rows_copied_for_a_fork_are_read_after_the_copy(torch, dtype, page, rotate):
    """begin, append and attention of many children of a prompt at once: whole tiles of each child's history are what begin
    copies.  The pool holds garbage before, so that a row read too early shows."""
    n, past, heads, kv, dim = 48, 3 * page + page - 1, 8, 2, 128
    with _cache(n_heads=heads, n_kv_heads=kv, head_dim=dim, dtype=dtype, page_size=page, n_layers=2, n_pages=n + 8, max_seqs=n + 1,
                max_tokens=past) as c:
        c.set_rope(max_pos=past + 8)
        b = Books(torch, c)
        s = b.new()
        b.step([s], [past], attend=False)
        for _ in range(5):
            kids = c.fork(s, n)
            own = torch.arange(4, n + 4, device="cuda")  # the children's own last pages
            c.storage()[own] = 1e30
            qkv = b.randn(n, heads + 2 * kv, dim)
            q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
            qr, outs = torch.empty(n, heads, dim, device="cuda", dtype=c.dtype), [torch.empty(n, heads, dim, device="cuda", dtype=c.dtype) for _ in range(2)]
            torch.cuda.synchronize()
            c.begin(kids, [1] * n)
            for layer in range(2):
                if rotate:
                    c.rope_append_dev(layer, q, k, v, qr)
                else:
                    c.append_dev(layer, k, v)
                c.attn_dev(layer, qr if rotate else q, outs[layer])
            c.check()
            last = c.tables(kids)[:, -1]
            assert sorted(last.tolist()) == own.tolist()
            for layer in range(2):
                new = c.storage()[torch.from_numpy(last).cuda().long(), layer, :, :, past % page]  # [n, 2, kv, dim]: the rows as they were appended
                for i in range(n):
                    rows = torch.cat([b.rows[s][layer], new[i:i + 1]])
                    want, tol = _want(torch, (qr if rotate else q)[i:i + 1], rows[:, 0], rows[:, 1], past)
                    _near(outs[layer][i:i + 1], want, tol, f"child {i}, layer {layer}")
            c.free(kids)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_that_the_caller_writes_ahead_of_attention(torch, dtype):
    """Old rows replaced through storage() right before append and attention, and right before attention."""
    with _cache(dtype=dtype, n_layers=1, page_size=64, n_pages=80, max_tokens=4000) as c:
        b = Books(torch, c)
        s = b.new()
        b.step([s], [3990], attend=False)
        table = torch.from_numpy(c.tables([s])[0]).cuda().long()
        for when in ("append", "attention"):
            past = c.length(s)
            rows = b.randn(past, 2, 2, 128)
            pages = torch.zeros(len(table) * 64, 2, 2, 128, device="cuda", dtype=c.dtype)
            pages[:past] = rows
            pages = pages.reshape(len(table), 64, 2, 2, 128).permute(0, 2, 3, 1, 4).contiguous()
            q, k, v = b.randn(1, 8, 128), b.randn(1, 2, 128), b.randn(1, 2, 128)
            out = torch.empty_like(q)
            c.begin([s], [1])
            torch.cuda.synchronize()
            if when == "append":
                c.storage()[table, 0] = pages
                c.append_dev(0, k, v)
            else:
                c.append_dev(0, k, v)
                new = c.storage()[table[-1], 0, :, :, past % 64].clone()
                c.storage()[table, 0] = pages
                c.storage()[table[-1], 0, :, :, past % 64] = new
            c.attn_dev(0, q, out)
            c.check()
            kv = torch.cat([rows, torch.stack([k, v], 1)])
            want, tol = _want(torch, q, kv[:, 0], kv[:, 1], past)
            _near(out, want, tol, when)
            b.rows[s] = [kv]


@pytest.mark.parametrize("dim", [64, 128])
def test_begin_makes_the_workspace_of_fp32_chunks(torch, dim):
    """A chunk whose workspace is larger than any before is captured without a call ahead of it, and a graph captured with
    smaller images keeps working when later batches need larger ones."""
    with _cache(n_heads=8, n_kv_heads=2, head_dim=dim, n_layers=1, n_pages=700, max_tokens=6000, max_seqs=3) as c:
        b = Books(torch, c, dim)
        s, t = b.new(), b.new()
        b.step([s], [300])  # loads the kernels
        graphs = []
        stream = torch.cuda.Stream()
        for x, past, n in ((t, 0, 2000), (s, 300, 4000)):
            q, out = b.randn(n, 8, dim), torch.empty(n, 8, dim, device="cuda")
            kv = [b.randn(n, 2, dim) for _ in range(2)]
            c.begin([x], [n])
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                c.append_dev(0, *kv)
                c.attn_dev(0, q, out)
            graphs.append((graph, x, past, n, q, out, kv))
            b.rows[x] = [torch.cat([b.rows[x][0], torch.stack(kv, 1)])]
            for graph, x, past, n, q, out, kv in graphs:  # the earlier graph too, on a batch of its own
                c.truncate(x, past)
                c.begin([x], [n])
                out.fill_(9.0)
                torch.cuda.synchronize()
                graph.replay()
                torch.cuda.synchronize()
                c.check()
                rows = b.rows[x][0]
                want, tol = _want(torch, q, rows[:, 0], rows[:, 1], past)
                _near(out, want, tol, f"{n} tokens on {past}")
        del graph, graphs


@pytest.mark.parametrize("original,theta,beta_slow,beta_fast,scaled", [
    (4, 10000.0, 1.0, 32.0, True), (6, 10000.0, 1.0, 32.0, True), (256, 500000.0, 64.0, 128.0, True),  # every pair turns less than beta_slow times
    (2**30, 50.0, 1.0, 32.0, False),                                    # every pair turns more than beta_fast times
])
def test_yarn_where_no_pair_is_on_the_ramp(torch, original, theta, beta_slow, beta_fast, scaled):
    turns = [original * theta ** (-2 * i / 128) / (2 * math.pi) for i in range(64)]
    assert max(turns) < beta_slow if scaled else min(turns) > beta_fast
    with _cache(n_layers=1) as c:
        b = Books(torch, c)
        c.set_rope(max_pos=600, layout="half", scaling="yarn", factor=8.0, original_len=original, theta=theta, beta_slow=beta_slow,
                   beta_fast=beta_fast, attn_factor=1.25)
        s = b.new()
        c.begin([s], [500])
        q, k, v = b.randn(500, 8, 128), b.randn(500, 2, 128), b.randn(500, 2, 128)
        out = torch.empty_like(q)
        c.rope_append_dev(0, q, k, v, out)
        c.check()
        pos = torch.arange(500, device="cuda")
        want = 1.25 * _turned(torch, q, pos, 128, "half", 0, "linear" if scaled else "none", 8.0, 0.0, theta, 0)
        _rope_near(torch, out, want, "f32", "q")


LONG = [("f32", 32, 8, 128, 9000, 64), ("f32", 16, 8, 128, 66100, 64), ("f32", 8, 1, 64, 20011, 16), ("f32", 8, 1, 256, 5000, 32),
        ("bf16", 32, 8, 128, 20000, 64), ("bf16", 8, 1, 64, 33000, 16), ("bf16", 8, 1, 256, 7000, 128), ("bf16", 16, 8, 128, 6000, 32)]


@pytest.mark.parametrize("dtype,heads,kv,dim,past,page", LONG)
def test_long_histories_by_the_norm_of_the_error(torch, dtype, heads, kv, dim, past, page):
    """The error of every output row by its norm, relative to the row's own.

    q, k and v are independent and normal, so that errors of the weights meet values of either sign: with a relative error e_j
    of weight j, an output's error is sum p_j e_j v_j, whose size is at most max |e| of the output's, sum p_j v_j.  bf16: a
    weight is rounded once (2^-8) and so is the output (2^-8): 2^-7 together; scores are exact products summed in fp32.
    fp32: scores are about 1 in size and their sums of head_dim products pass through at most 16 roundings and 48 truncations
    (2^-23 of a partial sum of that size each), mostly 6: 2^-18 with the split's rest (2^-21) and the exponential (2^-22);
    the second product's partial sums of 16 to 64 keys are cut off likewise (2^-20) and then added in fp32: 2^-17 together.
    A tile of 16 keys left out moves a row by sqrt(16 / past) of its norm, three times the tolerance and more."""
    tol = 2**-7 if dtype == "bf16" else 2**-17
    with _cache(n_heads=heads, n_kv_heads=kv, head_dim=dim, dtype=dtype, n_layers=1, n_pages=(past + 200) // page + 1, page_size=page,
                max_tokens=past) as c:
        b = Books(torch, c, past)
        s = b.new()
        b.step([s], [past], attend=False)
        rows = b.rows[s][0]
        for n in (1, 3, 8, 70, 200):
            c.begin([s], [n])
            q, k, v = b.randn(n, heads, dim), b.randn(n, kv, dim), b.randn(n, kv, dim)
            out = torch.empty_like(q)
            c.append_dev(0, k, v)
            c.attn_dev(0, q, out)
            c.check()
            full = torch.cat([rows, torch.stack([k, v], 1)])
            want, _ = _want(torch, q, full[:, 0], full[:, 1], past)
            size = want.norm(dim=-1)
            worst = float(((out.double() - want).norm(dim=-1) / size).max())
            assert worst <= tol, f"{n} tokens: {worst:.3g}, at most {tol:.3g}"
            if n == 1:  # the tolerance sees a lost tile, wherever it is
                for at in range(0, past - 16, past // 7):
                    less = torch.cat([full[:at], full[at + 16:]])
                    w, _ = _want(torch, q, less[:, 0], less[:, 1], past - 16)
                    assert float(((w - want).norm(dim=-1) / size).min()) > tol, at
            c.truncate(s, past)


@pytest.mark.parametrize("dtype,dim", [("f32", 64), ("f32", 128), ("f32", 256), ("bf16", 64), ("bf16", 128), ("bf16", 256)])
def test_strided_outputs(torch, dtype, dim):
    """Output rows further apart than a token's heads, by every kernel: single tokens, few, chunks with parts that are joined;
    the values between them stay."""
    heads, kv = 8, 2
    with _cache(n_heads=heads, n_kv_heads=kv, head_dim=dim, dtype=dtype, n_layers=1, n_pages=700, max_tokens=9000) as c:
        b = Books(torch, c, dim)
        seqs = [b.new() for _ in range(3)]
        b.step(seqs, [8000, 30, 77], attend=False)
        for new in ([1, 1, 1], [4, 2, 1], [100, 1, 3], [0, 0, 130]):
            past, n = [c.length(s) for s in seqs], sum(new)
            wide = torch.full((n, heads + 3, dim), 7.0, device="cuda", dtype=c.dtype)
            q = b.randn(n, heads + 1, dim)[:, 1:]
            k, v = b.randn(n, kv, dim), b.randn(n, kv, dim)
            c.begin(seqs, new)
            c.append_dev(0, k, v)
            c.attn_dev(0, q, wide[:, 2:2 + heads])
            c.check()
            assert bool((wide[:, :2] == 7.0).all()) and bool((wide[:, 2 + heads:] == 7.0).all())
            at = 0
            for s, p, m in zip(seqs, past, new):
                b.rows[s][0] = torch.cat([b.rows[s][0], torch.stack([k[at:at + m], v[at:at + m]], 1)])
                if m:
                    want, tol = _want(torch, q[at:at + m], b.rows[s][0][:, 0], b.rows[s][0][:, 1], p)
                    _near(wide[at:at + m, 2:2 + heads], want, tol, f"sequence {s}, {m} tokens")
                at += m


def test_for_shape(torch):
    """A cache of a model's geometry: heads, and sliding windows where the model has them."""
    from llama3pure_b200.paged import PagedCache
    from llama3pure_b200 import synth

    for shape in synth.CONFIGS.values():
        with PagedCache.for_shape(shape, n_layers=2, page_size=16, n_pages=40, max_seqs=2, max_tokens=600) as c:
            assert (c.n_heads, c.n_kv_heads, c.head_dim) == (shape.n_heads, shape.n_kv_heads, shape.head_dim)
            window = shape.swa_window if shape.is_gemma3 else 0
            assert (c.cfg.is_gemma3, c.cfg.swa_window, c.cfg.swa_pattern) == (shape.is_gemma3, shape.swa_window, shape.swa_pattern)
            b = Books(torch, c)
            s = b.new()
            win = lambda layer: window if window and layer % shape.swa_pattern < shape.swa_pattern - 1 else 0  # noqa: E731
            b.step([s], [560], window=win)
            b.step([s], [1], window=win)


@pytest.mark.parametrize("dtype,dim", [("f32", 64), ("f32", 128), ("bf16", 64), ("bf16", 128), ("bf16", 256)])
def test_a_replay_that_does_not_fit_writes_nothing(torch, dtype, dim):
    """A graph of chunks beside single tokens meets single tokens alone, and a graph of single tokens meets a chunk."""
    with _cache(n_heads=8, n_kv_heads=2, head_dim=dim, dtype=dtype, n_layers=1, n_pages=800, max_tokens=6000, page_size=16) as c:
        b = Books(torch, c)
        seqs = [b.new() for _ in range(3)]
        b.step(seqs, [5000, 900, 17], attend=False)
        kinds = {"chunks": [200, 130, 1], "single": [1, 1, 1], "few": [4, 3, 4] if dtype == "bf16" else [9, 4, 5]}
        q, out = b.randn(400, 8, dim), torch.empty(400, 8, dim, device="cuda", dtype=c.dtype)
        s = torch.cuda.Stream()
        graphs = {}

        def begin(new):
            for x, m in zip(seqs, (5000, 900, 17)):
                c.truncate(x, m)
            c.begin(seqs, new)

        for kind, new in kinds.items():
            begin(new)
            torch.cuda.synchronize()
            with torch.cuda.stream(s):
                c.attn_dev(0, q, out)
            s.synchronize()
            graphs[kind] = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graphs[kind], stream=s):
                c.attn_dev(0, q, out)
        for kind, new in kinds.items():
            for other, graph in graphs.items():
                begin(new)
                out.fill_(9.0)
                torch.cuda.synchronize()
                graph.replay()
                torch.cuda.synchronize()
                if other == kind:
                    c.check()
                    assert bool((out[:sum(new)] != 9.0).any(-1).all()) and bool((out[sum(new):] == 9.0).all())
                else:
                    with pytest.raises(AttnError) as e:
                        c.check()
                    assert e.value.code == -1
                    assert bool((out == 9.0).all()), f"a graph of {other} on {kind}"
        del graph, graphs


@pytest.mark.parametrize("dtype,dim", [("f32", 64), ("f32", 128), ("bf16", 64), ("bf16", 128)])
def test_a_replay_whose_row_part_does_not_fit_writes_nothing(torch, dtype, dim):
    """A graph of a chunk beside single tokens, of another row path than the batch that it meets: both parts stay out."""
    with _cache(n_heads=8, n_kv_heads=2, head_dim=dim, dtype=dtype, n_layers=1, n_pages=300, max_tokens=3000) as c:
        b = Books(torch, c)
        seqs = [b.new() for _ in range(3)]
        q, out = b.randn(600, 8, dim), torch.empty(600, 8, dim, device="cuda", dtype=c.dtype)
        kinds = [[300, 1, 1], [300, 4, 1] if dtype == "f32" else [300, 0, 2]]  # fp32: 16 rows per KV head, another kernel
        s = torch.cuda.Stream()
        graphs = []

        def begin(new):
            for x in seqs:
                c.truncate(x, 0)
            c.begin(seqs, new)

        for new in kinds:
            begin(new)
            torch.cuda.synchronize()
            with torch.cuda.stream(s):
                c.attn_dev(0, q, out)
            s.synchronize()
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=s):
                c.attn_dev(0, q, out)
        for i, new in enumerate(kinds):
            for j, graph in enumerate(graphs):
                begin(new)
                c.attn_dev(0, q, out)
                want = out.clone()
                out.fill_(9.0)
                torch.cuda.synchronize()
                graph.replay()
                torch.cuda.synchronize()
                try:
                    c.check()
                    assert bool((out[:sum(new)] == want[:sum(new)]).all()) and bool((out[sum(new):] == 9.0).all())
                except AttnError as e:
                    assert e.code == -1 and i != j
                    assert bool((out == 9.0).all()), f"a graph of {kinds[j]} on {new}"
        del graph, graphs


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_dropped_cache_is_gone_at_once(torch, dtype):
    """Not when the garbage collector comes: a pool is large, and freeing one in the middle of another's capture would end that."""
    import gc
    import weakref

    gc.collect()
    gc.disable()
    try:
        c = _cache(n_layers=1, dtype=dtype)
        gone = weakref.ref(c)
        st = c.storage()
        c.storage().zero_()
        view = st[1:2]
        del c, st
        assert gone() is not None and not bool(view.any())
        del view
        assert gone() is None
    finally:
        gc.enable()


def test_check_during_capture_leaves_the_capture(torch):
    with _cache(n_layers=1) as c:
        b = Books(torch, c)
        s = b.new()
        b.step([s], [20], attend=False)
        c.begin([s], [1])
        q, out = b.randn(1, 8, 128), torch.full((1, 8, 128), 9.0, device="cuda")
        k, v = b.randn(1, 2, 128), b.randn(1, 2, 128)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
            c.append_dev(0, k, v)
            with pytest.raises(AttnError) as e:
                c.check()
            c.attn_dev(0, q, out)
        assert e.value.code == -1
        graph.replay()
        torch.cuda.synchronize()
        c.check()
        rows = torch.cat([b.rows[s][0], torch.stack([k, v], 1)])
        want, tol = _want(torch, q, rows[:, 0], rows[:, 1], 20)
        _near(out, want, tol)
        del graph


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_pools_of_more_values_than_32_bits_count(torch, dtype):
    """Pages behind the 2^32nd value of a pool: rotation, append, copies, compaction, and every attention kernel."""
    with _cache(n_heads=8, n_kv_heads=8, head_dim=128, dtype=dtype, n_layers=32, page_size=128, n_pages=620, max_tokens=80000, max_seqs=4) as c:
        assert c.storage()[590].storage_offset() > 2**32
        c.set_rope(max_pos=600)
        b = Books(torch, c)
        full = c.new_seq()
        c.begin([full], [595 * 128])  # the pages before, without rows
        ids, rows = [c.new_seq() for _ in range(2)], [[], []]
        layer = 31

        def step(seqs, new):
            c.begin([ids[i] for i in seqs], new)
            n = sum(new)
            q, k, v = b.randn(n, 8, 128), b.randn(n, 8, 128), b.randn(n, 8, 128)
            qr, out = torch.empty_like(q), torch.empty_like(q)
            c.rope_append_dev(layer, q, k, v, qr)
            c.attn_dev(layer, qr, out)
            c.check()
            at = 0
            for i, m in zip(seqs, new):
                past = sum(len(x) for x in rows[i])
                t = torch.from_numpy(c.tables([ids[i]])[0]).cuda().long()
                pos = torch.arange(past, past + m, device="cuda")
                got = c.storage()[t[pos // 128], layer, :, :, pos % 128]
                kr = _turned(torch, k[at:at + m], pos, 128, "interleaved", 0, "none", 1.0, 0.0, 500000.0, 0)
                _rope_near(torch, got[:, 0], kr, dtype, "k")
                assert bool((got[:, 1] == v[at:at + m]).all())
                rows[i].append(got.clone())
                h = torch.cat(rows[i])
                want, tol = _want(torch, qr[at:at + m], h[:, 0], h[:, 1], past)
                _near(out[at:at + m], want, tol, f"{m} tokens on {past}")
                at += m

        step([0, 1], [300, 40])
        assert all(int(c.tables([i]).min()) >= 595 for i in ids)
        step([0, 1], [1, 1])
        step([0, 1], [3, 2])
        k, v = b.randn(1, 8, 128), b.randn(1, 8, 128)
        c.begin([ids[1]], [1])
        c.append_dev(layer, k, v)
        c.check()
        rows[1].append(torch.stack([k, v], 1))
        t = c.tables([ids[1]])[0]
        assert bool((c.storage()[int(t[-1]), layer, :, :, (c.length(ids[1]) - 1) % 128] == rows[1][-1][0]).all())
        kid = c.copy([ids[0]])[0]
        h = torch.cat(rows[0])
        for s in (kid, None):
            if s is None:  # moved to the front
                c.truncate(full, 0)
                assert c.compact() <= 10
                s = ids[0]
            t = torch.from_numpy(c.tables([s])[0]).cuda().long()
            pos = torch.arange(len(h), device="cuda")
            assert bool((c.storage()[t[pos // 128], layer, :, :, pos % 128] == h).all())
        step([0, 1], [1, 1])

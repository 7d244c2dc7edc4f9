"""What the paged-cache operators are measured on: their cases, their plain forms and their calls.

Three operators over one paged KV cache (llama3pure_b200/paged.py):
  attention   a batch of sequences, each with a chunk of new tokens (one token when decoding), attends causally to its pages;
  rotary      the new tokens' q and k are rotated (after an optional RMS norm of each head) and k, v are written into the pages;
  pages       sequences are forked, copied, freed and the pool is compacted.

The pages of a pool are one tensor [n_pages][n_layers][2: K, V][n_kv_heads][page_size][head_dim].  A new page is always the free page
of the lowest index, so the page tables follow from the order of the calls.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}

# Heads, KV heads and head size of the configurations this repository measures.
B1 = dict(heads=32, kv=8, dim=64)    # Llama 3.2 1B
B8 = dict(heads=32, kv=8, dim=128)   # Llama 3.1 8B
GM = dict(heads=8, kv=1, dim=256)    # Gemma 2B


def _attn(name, shape, type, seqs, past_lo, past_hi, new_lo, new_hi, page, layer=0, window=0):
    return dict(name=name, op="attention", type=type, seqs=seqs, past_lo=past_lo, past_hi=past_hi, new_lo=new_lo, new_hi=new_hi, page=page,
                layer=layer, window=window, **shape)


def _rot(name, shape, type, tokens, seqs, past, page, layout, rotary, scaling, norm):
    return dict(name=name, op="rotary", type=type, tokens=tokens, seqs=seqs, past=past, page=page, layout=layout, rotary=rotary, scaling=scaling, norm=norm,
                **shape)


def _pages(name, shape, type, kind, layers, seqs, tokens, page):
    return dict(name=name, op=kind, type=type, layers=layers, seqs=seqs, tokens=tokens, page=page, **shape)


def listed():
    return [
        # one user's next token after a short dialogue: latency is all
        _attn("one token 1B", B1, "bf16", 1, 1022, 1022, 1, 1, 16),
        # one user's next token at the end of a long document, fp32 cache: one long stream split over the whole card
        _attn("one token 128K 8B f32", B8, "f32", 1, 131071, 131071, 1, 1, 64),
        # a serving step: 64 users at lengths of their own, one token each
        _attn("64 sequences 8B", B8, "bf16", 64, 60, 8191, 1, 1, 16),
        # drafts being verified: a few tokens for each of 16 users
        _attn("16 drafts 8B", B8, "bf16", 16, 700, 6001, 3, 6, 32),
        # a fresh 2K prompt in fp32, nothing cached before it
        _attn("prompt 2K 8B f32", B8, "f32", 1, 0, 0, 2048, 2048, 64),
        # a chunk of a long document, alone on the card: few rows against many keys
        _attn("chunk 96 of 32K 8B", B8, "bf16", 1, 32001, 32001, 96, 96, 16),
        # prompts fed in chunks of 2K, each on what came before: the largest pass
        _attn("4 chunks 2K 8B", B8, "bf16", 4, 1, 6143, 1900, 2048, 64),
        # sliding-window layer, one prompt chunk among decoding users, head size 256
        _attn("window 256-dim", GM, "bf16", 8, 3, 4095, 1, 389, 32, window=512),
        # the rotation of one serving step
        _rot("rotary 64 tokens 8B", B8, "bf16", 64, 64, 4001, 16, "interleaved", 128, "bands", False),
        # the rotation of a long prompt: half layout, half of each head, long-context scaling
        _rot("rotary 8K tokens 8B f32", B8, "f32", 8191, 2, 120001, 64, "half", 64, "yarn", True),
        # one prompt answered 64 times: every answer takes a copy of the prompt's last page
        _pages("fork 64 8B", B8, "bf16", "fork", 32, 64, 1007, 16),
        # half of the users leave, the pool is compacted, then every user that stayed is copied
        _pages("compact 8B", B8, "bf16", "compact", 32, 8, 501, 16),
    ]


def draw(rng):
    while True:
        c = _draw(rng)
        w = work(c)
        if w["flops"] <= 5e11 and w["bytes"] <= 2e9:  # no more than the largest listed cases
            return c


def _draw(rng):
    def span(lo, hi):  # spread over the logarithm
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["attention", "attention", "attention", "rotary", "rotary", "fork", "compact"])
    type = rng.choice(["f32", "bf16"])
    dim = rng.choice([64, 128, 256])
    kv = rng.choice([1, 2, 3, 4, 8]) if dim < 256 else rng.choice([1, 2, 4])
    heads = kv * rng.choice([1, 2, 3, 4, 6, 8])
    page = rng.choice([16, 32, 64, 128])
    shape = dict(heads=heads, kv=kv, dim=dim)
    if op == "attention":
        new_hi = rng.choice([1, 1, span(2, 16), span(16, 1500)])
        new_lo = max(1, new_hi // rng.choice([1, 2, 50]))
        seqs = span(1, 64) if new_hi == 1 else span(1, 24) if new_hi <= 16 else span(1, 4)
        past_hi = span(1, 60000) if seqs == 1 and new_hi <= 16 else span(1, 6000)
        past_lo = past_hi // rng.choice([1, 3, 40])
        window = rng.choice([0, 0, span(1, 2000)])
        return _attn("", shape, type, seqs, past_lo, past_hi, new_lo, new_hi, page, window=window)
    if op == "rotary":
        tokens = span(1, 6000)
        rotary = rng.choice([dim, dim, dim // 2, dim // 4, 2 * rng.randrange(1, dim // 2)])
        return _rot("", shape, type, tokens, rng.randrange(1, min(tokens, 40) + 1), span(1, 120000), page, rng.choice(["interleaved", "half"]), rotary,
                    rng.choice(["none", "linear", "bands", "yarn"]), rng.random() < 0.5)
    return _pages("", shape, type, op, rng.choice([1, 4, 16, 32]), span(1, 48) if op == "fork" else span(1, 6), span(1, 900), page)


# ---- what a case holds ------------------------------------------------------------------------------------------------------------


def _lengths(c):
    """Cached tokens and new tokens of every sequence of an attention case: whole numbers spread over the case's ranges, the highest ones among them."""
    n = c["seqs"]
    past = [c["past_hi"] - (c["past_hi"] - c["past_lo"]) * ((i * 5) % n) // max(1, n - 1) for i in range(n)]
    new = [c["new_hi"] if i % 8 == 0 else c["new_lo"] + (i * 7) % (1 + min(c["new_hi"] - c["new_lo"], max(1, c["new_lo"] // 8))) for i in range(n)]
    return past, new


def _rot_lengths(c):
    n, t = c["seqs"], c["tokens"]
    return [max(0, c["past"] - 13 * i) for i in range(n)], [t // n + (i < t % n) for i in range(n)]


def _need(tokens, page):
    return -(-tokens // page)


def _grown(lengths, page):
    """Page tables of sequences that grew side by side, in eight steps each: the pages of one sequence lie apart, as in a pool in use."""
    tables, used = [[] for _ in lengths], 0
    for step in range(1, 9):
        for t, n in zip(tables, lengths):
            while len(t) < _need(n * step // 8, page):
                t.append(used)
                used += 1
    return tables, used


def _padded(tables):
    out = np.full((len(tables), max(len(t) for t in tables)), -1, np.int32)
    for i, t in enumerate(tables):
        out[i, :len(t)] = t
    return out


def _cache(c, n_layers, n_pages, seqs, tokens, **kw):
    from llama3pure_b200.paged import PagedCache

    return PagedCache(n_layers=n_layers, n_heads=c["heads"], n_kv_heads=c["kv"], head_dim=c["dim"], page_size=c["page"], n_pages=n_pages, max_seqs=seqs,
                      max_tokens=tokens, dtype=c["type"], **kw)


def _grow(cache, seqs, lengths):
    """The calls that lead to _grown's page tables."""
    done = [0] * len(lengths)
    for step in range(1, 9):
        new = [n * step // 8 - d for n, d in zip(lengths, done)]
        cache.begin(seqs, new)
        done = [d + x for d, x in zip(done, new)]


def _rows(g, *shape, type):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(TYPES[type])


def _keys(g, *shape, type):
    """Keys as a model has them: some channels of a head carry more than others."""
    gain = torch.exp(0.5 * torch.randn(shape[-1], generator=g, device="cuda"))
    return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * gain).to(TYPES[type])


def _attention_inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    past, new = _lengths(c)
    tables, used = _grown(past, c["page"])
    for t, p, n in zip(tables, past, new):  # the new tokens' pages
        while len(t) < _need(p + n, c["page"]):
            t.append(used)
            used += 1
    block = (used, 1, c["kv"], c["page"], c["dim"])
    store = torch.stack([_keys(g, *block, type=c["type"]), _rows(g, *block, type=c["type"])], 2)
    q = _rows(g, sum(new), c["heads"], c["dim"], type=c["type"])
    return past, new, tables, used, store, q


def _rotary_inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    past, new = _rot_lengths(c)
    tables, used = _grown(past, c["page"])
    for t, p, n in zip(tables, past, new):
        while len(t) < _need(p + n, c["page"]):
            t.append(used)
            used += 1
    t = sum(new)
    q, k, v = (_rows(g, t, h, c["dim"], type=c["type"]) for h in (c["heads"], c["kv"], c["kv"]))
    norm = None
    if c["norm"]:
        norm = [1 + 0.1 * torch.randn(c["dim"], generator=g, device="cuda") for _ in range(2)]
    return past, new, tables, used, q, k, v, norm


THETA, FACTOR, ORIGINAL = 500000.0, 8.0, 8192


def _rope_kw(c, max_pos):
    return dict(max_pos=max_pos, layout=c["layout"], rotary_dim=c["rotary"], theta=THETA, scaling=c["scaling"], factor=FACTOR, original_len=ORIGINAL, low_freq=1.0,
                high_freq=4.0, beta_fast=32.0, beta_slow=1.0)


def _page_inputs(c, seed):
    """The sequences of a page case before its pass, and the content of the whole pool."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    if c["op"] == "fork":
        lengths = [c["tokens"]]
    else:
        lengths = [c["tokens"] + 3 * (i % 5) for i in range(2 * c["seqs"])]
    tables, used = _grown(lengths, c["page"])
    n_pages = used + c["seqs"] if c["op"] == "fork" else max(used, 2 * sum(len(t) for t in tables[c["seqs"]:]))
    store = _rows(g, n_pages, c["layers"], 2, c["kv"], c["page"], c["dim"], type=c["type"])
    return lengths, tables, n_pages, store


def prepare(case, seed):
    c = case
    if c["op"] == "attention":
        past, new, tables, used, store, q = _attention_inputs(c, seed)
        s = dict(c=c, q=q)
        if own:  # the cache, its sequences grown to their lengths and the step begun, as a serving loop has them before the layers run
            cache = _cache(c, 1, used, len(past), max(sum(past) // 8 + len(past) * 2, sum(new)), is_gemma3=int(c["window"] > 0), swa_window=c["window"],
                           swa_pattern=2 if c["window"] else 0)
            seqs = [cache.new_seq() for _ in past]
            _grow(cache, seqs, past)
            cache.begin(seqs, new)
            cache.storage().copy_(store)
            s.update(cache=cache, out=torch.empty_like(q))
        else:  # what a program without the framework keeps: the pool, the tables and the lengths on the device
            n_new, n_kv = (torch.tensor(v, device="cuda") for v in (new, [p + n for p, n in zip(past, new)]))
            table = torch.from_numpy(_padded(tables)).cuda().long().clamp_min(0)
            s.update(store=store, table=table, n_new=n_new, n_kv=n_kv, max_new=max(new))
        return s
    if c["op"] == "rotary":
        past, new, tables, used, q, k, v, norm = _rotary_inputs(c, seed)
        s = dict(c=c, q=q, k=k, v=v)
        if own:
            cache = _cache(c, 1, used, len(past), max(sum(past) // 8 + len(past) * 2, sum(new)))
            seqs = [cache.new_seq() for _ in past]
            _grow(cache, seqs, past)
            cache.begin(seqs, new)
            kw = _rope_kw(c, max(p + n for p, n in zip(past, new)))
            if norm is not None:
                kw.update(q_norm=norm[0].cpu().numpy()[None], k_norm=norm[1].cpu().numpy()[None], rms_norm_eps=1e-5)
            cache.set_rope(**kw)
            cache.storage().zero_()
            s.update(cache=cache, store=cache.storage(), q_out=torch.empty_like(q))
        else:
            pos = torch.cat([torch.arange(p, p + n, device="cuda") for p, n in zip(past, new)])
            row = torch.repeat_interleave(torch.arange(len(new), device="cuda"), torch.tensor(new, device="cuda"))
            table = torch.from_numpy(_padded(tables)).cuda().long()
            store = torch.zeros(used, 1, 2, c["kv"], c["page"], c["dim"], device="cuda", dtype=TYPES[c["type"]])
            s.update(store=store, pos=pos, row=row, table=table, norm=norm)
        return s
    lengths, tables, n_pages, store = _page_inputs(c, seed)
    if own:
        cache = _cache(c, c["layers"], n_pages, c["seqs"] + len(lengths), sum(lengths) // 8 + 2 * len(lengths) + c["seqs"])
        seqs = [cache.new_seq() for _ in lengths]
        _grow(cache, seqs, lengths)
        cache.storage().copy_(store)
        return dict(c=c, cache=cache, seqs=seqs, store=cache.storage())
    return dict(c=c, store=store, tables=tables, lengths=lengths)


# ---- the plain forms --------------------------------------------------------------------------------------------------------------


def _plain_attention(s):
    c, q, store, table, n_new, n_kv = s["c"], s["q"], s["store"], s["table"], s["n_new"], s["n_kv"]
    b, w, kv, dim, group = len(n_new), s["max_new"], c["kv"], c["dim"], c["heads"] // c["kv"]
    kv_rows = store[table, 0]  # [b, pages, 2, kv, page, dim]
    k, v = (kv_rows[:, :, i].permute(0, 2, 1, 3, 4).reshape(b, kv, -1, dim).float() for i in (0, 1))
    first = torch.cumsum(n_new, 0) - n_new
    i = torch.arange(w, device="cuda")
    at = (first[:, None] + i).clamp_max(q.shape[0] - 1)
    qs = q[at].float().reshape(b, w, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(b, kv, group * w, dim)
    score = (qs @ k.transpose(-1, -2)).reshape(b, kv, group, w, -1) * (1 / math.sqrt(dim))
    t = (n_kv - n_new)[:, None] + i  # positions of the new tokens
    j = torch.arange(k.shape[2], device="cuda")
    seen = j <= t[..., None]
    if c["window"]:
        seen &= j > t[..., None] - c["window"]
    score = score.masked_fill_(~seen[:, None, None], float("-inf"))
    score = (score - score.amax(-1, keepdim=True)).exp_()
    score = score / score.sum(-1, keepdim=True)
    o = (score.reshape(b, kv, group * w, -1) @ v).reshape(b, kv, group, w, dim).permute(0, 3, 1, 2, 4).reshape(b, w, c["heads"], dim)
    return o[i < n_new[:, None]].to(q.dtype)


def _frequencies(c, dtype=torch.float64):
    """The angle of one position for every pair, after the case's scaling, and the factor on cosine and sine."""
    r = c["rotary"]
    i = torch.arange(r // 2, device="cuda", dtype=dtype)
    f = THETA ** (-2 * i / r)
    if c["scaling"] == "linear":
        return f / FACTOR, 1.0
    if c["scaling"] == "bands":
        turns = ORIGINAL * f / (2 * math.pi)
        mix = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return f * ((1 - mix) / FACTOR + mix), 1.0
    if c["scaling"] == "yarn":
        lo, hi = (r * math.log(ORIGINAL / (n * 2 * math.pi)) / (2 * math.log(THETA)) for n in (32.0, 1.0))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), r - 1)
        ramp = ((i - lo) / (hi - lo if hi != lo else 0.001)).clamp(0, 1)
        return f * (1 - ramp) + f / FACTOR * ramp, 0.1 * math.log(FACTOR) + 1
    return f, 1.0


def _plain_turn(c, x, cos, sin, weight):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5) * weight
    r = c["rotary"]
    if c["layout"] == "half":
        a, b = x[..., :r // 2], x[..., r // 2:r]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., r:]], -1)
    a, b = x[..., 0:r:2], x[..., 1:r:2]
    return torch.cat([torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2), x[..., r:]], -1)


def _plain_rotary(s):
    c, store, pos = s["c"], s["store"], s["pos"]
    f, factor = _frequencies(c)
    angle = pos[:, None].double() * f
    cos, sin = ((h(angle) * factor).float()[:, None] for h in (torch.cos, torch.sin))
    wq, wk = s["norm"] or (None, None)
    page, at = s["table"][s["row"], pos // c["page"]], pos % c["page"]
    store[page, 0, 0, :, at] = _plain_turn(c, s["k"], cos, sin, wk).to(store.dtype)
    store[page, 0, 1, :, at] = s["v"]
    return _plain_turn(c, s["q"], cos, sin, wq).to(s["q"].dtype), store


def _plain_copy(store, src, dst, rows, page):
    """Copies the first rows[i] rows of page src[i] to page dst[i]."""
    if src:
        src, dst, rows = (torch.tensor(v, device="cuda") for v in (src, dst, rows))
        keep = (torch.arange(page, device="cuda") < rows[:, None])[:, None, None, None, :, None]
        store[dst] = torch.where(keep, store[src], store[dst])


def _plain_fork(s):
    c, store, table = s["c"], s["store"], s["tables"][0]
    used, n, rows = len(table), c["seqs"], c["tokens"] % c["page"]
    new = list(range(used, used + n))
    if rows:  # every child's next token falls into the shared last page: it takes a copy of it
        _plain_copy(store, [table[-1]] * n, new, [rows] * n, c["page"])
    children = np.empty((n, len(table) + (0 if rows else 1)), np.int32)
    children[:, :len(table)] = table
    children[:, -1] = new
    return store, children


def _plain_compact(s):
    c, store, tables, lengths, half, page = s["c"], s["store"], s["tables"], s["lengths"], s["c"]["seqs"], s["c"]["page"]
    tables, lengths = tables[half:], lengths[half:]  # the first half leaves
    rows = {p: min(page, n - i * page) for t, n in zip(tables, lengths) for i, p in enumerate(t)}
    k = len(rows)
    src, dst = sorted(p for p in rows if p >= k), sorted(set(range(k)) - set(rows))
    _plain_copy(store, src, dst, [rows[p] for p in src], page)
    moved = dict(zip(src, dst))
    tables = [[moved.get(p, p) for p in t] for t in tables]
    copies, at = [], k
    for t in tables:
        copies.append(list(range(at, at + len(t))))
        at += len(t)
    flat = [(p, d, min(page, n - i * page)) for t, u, n in zip(tables, copies, lengths) for i, (p, d) in enumerate(zip(t, u))]
    _plain_copy(store, [x[0] for x in flat], [x[1] for x in flat], [x[2] for x in flat], page)
    s["tables"], s["lengths"] = tables + copies, lengths + lengths
    return store, _padded(s["tables"]), k


def run(state):
    s, c = state, state["c"]
    if not own:
        return {"attention": _plain_attention, "rotary": _plain_rotary, "fork": _plain_fork, "compact": _plain_compact}[c["op"]](s)
    cache = s["cache"]
    if c["op"] == "attention":
        cache.attn_dev(0, s["q"], s["out"])
        return s["out"]
    if c["op"] == "rotary":
        cache.rope_append_dev(0, s["q"], s["k"], s["v"], s["q_out"])
        return s["q_out"], s["store"]
    if c["op"] == "fork":
        children = cache.fork(s["seqs"][0], c["seqs"])
        cache.begin(children, [1] * c["seqs"])
        tables = cache.tables(children)
        cache.free(children)
        return s["store"], tables
    half = c["seqs"]
    cache.free(s["seqs"][:half])
    used = cache.compact()
    kept = s["seqs"][half:]
    s["seqs"] = kept + cache.copy(kept)
    return s["store"], cache.tables(s["seqs"]), used


# ---- the work of a pass, and its exact outputs --------------------------------------------------------------------------------------


def _seen(past, new, window):
    """Attended keys over all new tokens of a sequence, and the cache rows that they reach."""
    if not window:
        return sum(past + i + 1 for i in range(new)), past + new
    return sum(min(past + i + 1, window) for i in range(new)), past + new - max(0, past - window + 1)


def work(case):
    c, size = case, TYPES[case["type"]].itemsize
    if c["op"] == "attention":
        past, new = _lengths(c)
        seen = [_seen(p, n, c["window"]) for p, n in zip(past, new)]
        rows = sum(r for _, r in seen)
        return {"bytes": size * c["dim"] * (2 * rows * c["kv"] + 2 * sum(new) * c["heads"]), "flops": 4 * c["dim"] * c["heads"] * sum(k for k, _ in seen)}
    if c["op"] == "rotary":
        t = c["tokens"]
        return {"bytes": 2 * size * t * c["dim"] * (c["heads"] + 2 * c["kv"]), "flops": 3 * t * c["rotary"] * (c["heads"] + c["kv"])}
    row = 2 * c["layers"] * c["kv"] * c["dim"] * size
    if c["op"] == "fork":
        return {"bytes": max(2 * row * c["seqs"] * (c["tokens"] % c["page"]), 4 * c["seqs"]), "flops": 0}
    # after the first pass the sequences that stay are the copies of the pass before: all their pages move down, and are copied again
    lengths = [c["tokens"] + 3 * (i % 5) for i in range(2 * c["seqs"])][c["seqs"]:]
    return {"bytes": 4 * row * sum(lengths), "flops": 0}


def exact(case, seed):
    c = case
    if c["op"] == "attention":
        past, new, tables, used, store, q = _attention_inputs(c, seed)
        group, outs, first = c["heads"] // c["kv"], [], 0
        for p, n, t in zip(past, new, tables):
            idx = torch.tensor(t, device="cuda")
            out = torch.empty(n, c["heads"], c["dim"], device="cuda", dtype=torch.float64)
            for h in range(c["heads"]):
                k, v = (store[idx, 0, i, h // group].reshape(-1, c["dim"])[:p + n].double() for i in (0, 1))
                for a in range(0, n, 512):  # a block of rows at a time
                    m = min(512, n - a)
                    e = q[first + a:first + a + m, h].double() @ k.T / math.sqrt(c["dim"])
                    d = torch.arange(p + a, p + a + m, device="cuda")[:, None] - torch.arange(p + n, device="cuda")
                    off = d < 0
                    if c["window"]:
                        off |= d >= c["window"]
                    out[a:a + m, h] = torch.softmax(e.masked_fill(off, -math.inf), -1) @ v
            outs.append(out)
            first += n
        return torch.cat(outs)
    if c["op"] == "rotary":
        past, new, tables, used, q, k, v, norm = _rotary_inputs(c, seed)
        pos = torch.tensor([p + i for p, n in zip(past, new) for i in range(n)], device="cuda")
        f, factor = _frequencies(c)
        turn = torch.polar(torch.full_like(pos[:, None] * f, factor), pos[:, None] * f)[:, None]  # as complex numbers

        def rotate(x, w):
            x = x.double()
            if w is not None:
                x = x / (x.pow(2).sum(-1, keepdim=True) / c["dim"] + 1e-5).sqrt() * w.double()
            r, y = c["rotary"], x.clone()
            a, b = (slice(0, r // 2), slice(r // 2, r)) if c["layout"] == "half" else (slice(0, r, 2), slice(1, r, 2))
            z = torch.complex(x[..., a].contiguous(), x[..., b].contiguous()) * turn
            y[..., a], y[..., b] = z.real, z.imag
            return y

        store = torch.zeros(used, 1, 2, c["kv"], c["page"], c["dim"], device="cuda", dtype=torch.float64)
        wq, wk = norm or (None, None)
        kr, first = rotate(k, wk), 0
        for p, n, t in zip(past, new, tables):
            at = torch.arange(p, p + n, device="cuda")
            pages = torch.tensor(t, device="cuda")[at // c["page"]]
            store[pages, 0, 0, :, at % c["page"]] = kr[first:first + n]
            store[pages, 0, 1, :, at % c["page"]] = v[first:first + n].double()
            first += n
        return rotate(q, wq), store
    return None  # pages are moved, not computed

// l3p_paged.cu -- the paged cache: pool, sequences, pages, and the batch
// description of a step (llama3pure_paged.h).  Books are kept on the host;
// the device holds the storage and what the current step's kernels read.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstring>
#include <functional>
#include <new>

#include "paged.h"
#include "ptx.cuh"

using namespace l3p;
using namespace l3p_pg;

namespace {

using Ctx = l3p_paged_ctx;

int pages_for(const Ctx* ctx, int tokens) { return (tokens + ctx->cfg.page_size - 1) >> ctx->shift; }

int take_page(Ctx* ctx) {
  std::pop_heap(ctx->free_heap.begin(), ctx->free_heap.end(), std::greater<int>());
  const int p = ctx->free_heap.back();
  ctx->free_heap.pop_back();
  ctx->refs[p] = 1;
  ctx->fill[p] = 0;
  return p;
}

void drop_page(Ctx* ctx, int p) {
  if (--ctx->refs[p] == 0) {
    ctx->free_heap.push_back(p);
    std::push_heap(ctx->free_heap.begin(), ctx->free_heap.end(), std::greater<int>());
  }
}

// Room for n pages in all, without a change; grown by doubling.
void reserve_pages(std::vector<int>* pages, size_t n) {
  if (pages->capacity() < n) pages->reserve(std::max(n, 2 * pages->capacity()));
}

int check_seq(Ctx* ctx, int seq) {
  if (seq < 0 || seq >= (int)ctx->seqs.size() || !ctx->seqs[seq].live)
    return fail(ctx, L3P_E_RANGE, "there is no sequence %d", seq);
  return L3P_OK;
}

// Every id is a live sequence, and no id comes twice.
int check_seqs(Ctx* ctx, int n, const int* seqs) {
  std::vector<char> seen(ctx->seqs.size(), 0);
  for (int i = 0; i < n; ++i) {
    if (int rc = check_seq(ctx, seqs[i])) return rc;
    if (seen[seqs[i]]) return fail(ctx, L3P_E_INVAL, "sequence %d is given twice", seqs[i]);
    seen[seqs[i]] = 1;
  }
  return L3P_OK;
}

int free_seq_count(const Ctx* ctx) {
  int n = 0;
  for (const auto& s : ctx->seqs) n += !s.live;
  return n;
}

int new_seq(Ctx* ctx) {
  for (size_t i = 0; i < ctx->seqs.size(); ++i)
    if (!ctx->seqs[i].live) {
      ctx->seqs[i].live = true;
      ctx->seqs[i].len = 0;
      ctx->seqs[i].pages.clear();
      return (int)i;
    }
  return -1;
}

// A pinned staging slot of at least `words` words whose last upload is done.
int take_slot(Ctx* ctx, size_t words, Ctx::Slot** out) {
  Ctx::Slot& s = ctx->slots[ctx->slot_next++ % Ctx::kSlots];
  if (s.used) PG_CUDA(ctx, cudaEventSynchronize(s.done));
  s.used = false;
  if (s.words < words) {
    if (s.host) cudaFreeHost(s.host);
    s.host = nullptr;
    s.words = 0;
    const size_t want = std::max(words + words / 2, (size_t)16384);
    if (cudaHostAlloc(&s.host, want * 4, cudaHostAllocDefault) != cudaSuccess) {
      cudaGetLastError();
      return fail(ctx, L3P_E_NOMEM, "pinned staging of %zu bytes failed", want * 4);
    }
    s.words = want;
  }
  *out = &s;
  return L3P_OK;
}

int upload(Ctx* ctx, Ctx::Slot* s, int* dev, size_t words, cudaStream_t st) {
  PG_CUDA(ctx, cudaMemcpyAsync(dev, s->host, words * 4, cudaMemcpyHostToDevice, st));
  PG_CUDA(ctx, cudaEventRecord(s->done, st));
  s->used = true;
  return L3P_OK;
}

// Enqueues the page copies `jobs` (source, destination, rows, 0) from a slot that has room for them.
int copy_pages(Ctx* ctx, const std::vector<int4>& jobs, Ctx::Slot* s, cudaStream_t st) {
  if (jobs.empty()) return L3P_OK;
  memcpy(s->host, jobs.data(), jobs.size() * sizeof(int4));
  if (int rc = upload(ctx, s, ctx->jobs, jobs.size() * 4, st)) return rc;
  return launch_page_copy(ctx, ctx->jobs, (int)jobs.size(), st);
}

cudaStream_t as_stream(void* s) { return static_cast<cudaStream_t>(s); }

int refuse_capture(Ctx* ctx, cudaStream_t s, const char* what) {
  if (capturing(s)) return fail(ctx, L3P_E_INVAL, "%s moves host data: not during stream capture", what);
  return L3P_OK;
}

// ---- the batch description -----------------------------------------------------

struct BatchSeq {
  int q_row0, n_new, len, tbl;  // len: with the new tokens
  bool tc;                      // takes the tensor-core kernels
};

// Which kernels a sequence takes: the row kernel up to row_limit rows per KV head.  In bf16, sequences of 9 to row_limit
// rows go with the longer ones where there are some: two kernels, each with part of the batch, fill the GPU less than one
// (16 drafts of 12 to 24 rows on 3000 keys, 8B heads, layers in turn: 44.2 us, by two kernels 62.5).
void choose_paths(const Ctx* ctx, std::vector<BatchSeq>* bs) {
  const int limit = row_limit(ctx);
  bool any = false;
  for (const auto& b : *bs) any |= (long long)b.n_new * ctx->G > limit;
  for (auto& b : *bs) b.tc = (long long)b.n_new * ctx->G > (any && ctx->bf16 ? std::min(limit, 8) : limit);
}

// First key that the token at `pos` attends to.
int first_key(const Ctx* ctx, bool win, int pos) { return win ? std::max(0, pos - ctx->cfg.swa_window + 1) : 0; }

// Row kernel: units are (sequence, KV head, block of 8*nt rows), their cost the
// 16-key tiles they read.  Two ways to share them out:
//   laid end to end and cut into equal runs, one per CTA: every SM streams the
//     same number of tiles, but a CTA may begin, end and merge several units;
//   every unit cut into equal parts on CTAs of its own (with no more units than
//     CTAs): one segment per CTA, the longest part sets the time.
// A run or part is a multiple of the CTA's warps, which take its tiles in turn,
// so both are counted in rounds of one tile per warp.  A further segment of a CTA
// costs about kSegRounds rounds that its prefetched tiles do not hide (8B heads:
// one token on 8K keys 17.3 us end to end, 12.4 by units; 4 sequences x 3000 keys
// 18.0 and 14.3; with 128 units, 16 sequences x 4 tokens, 43 either way).
constexpr double kSegRounds = 1.5;
void plan_rows(Ctx* ctx, bool win, const std::vector<BatchSeq>& bs, int nt, std::vector<int>* first,
               std::vector<PgSeg>* segs) {
  const int rt = 8 * nt, warps = row_warps(ctx), G = ctx->G;
  std::vector<PgSeg>& units = ctx->row_units;
  units.clear();
  long long total = 0;
  int longest = 0;
  for (const auto& b : bs) {
    const long long rows = (long long)b.n_new * G;
    if (rows == 0 || b.tc) continue;
    const int pos0 = b.len - b.n_new;
    for (int h = 0; h < ctx->cfg.n_kv_heads; ++h)
      for (int r0 = 0; r0 < rows; r0 += rt) {
        PgSeg u{};
        u.tbl = b.tbl;
        u.q_row0 = b.q_row0;
        u.pos0 = pos0;
        u.r0 = r0;
        u.n_rows = (int)std::min<long long>(rt, rows - r0);
        u.kvh = h;
        u.key_lo = first_key(ctx, win, pos0 + r0 / G);
        u.key_hi = pos0 + (r0 + u.n_rows - 1) / G + 1;
        u.tile0 = u.key_lo / kPgTile;
        u.tile1 = (u.key_hi + kPgTile - 1) / kPgTile;
        total += u.tile1 - u.tile0;
        longest = std::max(longest, u.tile1 - u.tile0);
        units.push_back(u);
      }
  }
  if (units.empty()) return;
  segs->reserve(units.size() + kPgMaxCtas);
  const int max_ctas = std::min(ctx->num_sms, kPgMaxCtas);
  auto rounds = [&](long long tiles) { return (tiles + warps - 1) / warps; };
  const long long run = rounds((total + max_ctas - 1) / max_ctas) * warps;
  long long part = 0;  // tiles of a part at most, when every CTA has one
  if ((int)units.size() <= max_ctas) {
    auto ctas = [&](long long r) {
      long long n = 0;
      for (const auto& u : units) n += (u.tile1 - u.tile0 + r * warps - 1) / (r * warps);
      return n;
    };
    long long lo = std::max<long long>(1, run / warps), hi = rounds(longest);  // rounds; ctas(hi) is the number of units
    while (lo < hi) {
      const long long mid = (lo + hi) / 2;
      if (ctas(mid) <= max_ctas)
        hi = mid;
      else
        lo = mid + 1;
    }
    const double more = std::ceil((double)units.size() * run / total);  // segments of a CTA behind its first, end to end
    if (hi <= run / warps + kSegRounds * more) part = hi * warps;
  }
  first->assign(1, 0);
  if (part > 0) {
    int cta = 0;
    for (const auto& u : units) {
      const int n = u.tile1 - u.tile0, k = (int)((n + part - 1) / part);
      const long long each = rounds((n + k - 1) / k) * warps;
      for (int i = 0; i < k; ++i) {
        PgSeg g = u;
        g.tile0 = (int)std::min<long long>(u.tile1, u.tile0 + i * each);
        g.tile1 = (int)std::min<long long>(u.tile1, g.tile0 + each);
        g.part = i;
        g.n_parts = k;
        g.cta0 = cta;
        segs->push_back(g);
        first->push_back((int)segs->size());
      }
      cta += k;
    }
    return;
  }
  const int n_cta = (int)((total + run - 1) / run);
  long long at = 0;  // tiles laid so far
  for (auto& u : units) {
    const int n = u.tile1 - u.tile0, t_begin = u.tile0, t_end = u.tile1;
    const int c0 = (int)(at / run), c1 = (int)((at + n - 1) / run);
    int t = t_begin;
    for (int c = c0; c <= c1; ++c) {
      const int end = (int)std::min<long long>(t_end, t_begin + ((long long)(c + 1) * run - at));
      PgSeg g = u;
      g.tile0 = t;
      g.tile1 = end;
      g.part = c - c0;
      g.n_parts = c1 - c0 + 1;
      g.cta0 = c0;
      while ((int)first->size() <= c) first->push_back((int)segs->size());
      segs->push_back(g);
      t = end;
    }
    at += n;
  }
  while ((int)first->size() <= n_cta) first->push_back((int)segs->size());
}

// Tensor-core kernels: units (sequence, KV head, block of rows); with too few
// of them for the GPU, long key ranges are cut into parts of equal size, which a
// second kernel merges.  Longest parts first.  fp32 pools: also the list of the
// key tiles that the units read.
void plan_tc(Ctx* ctx, bool win, const std::vector<BatchSeq>& bs, std::vector<PgPart>* parts,
             std::vector<PgPart>* merges, std::vector<PgPrep>* prep) {
  const int tile = ctx->bf16 ? tc_tile(ctx) : 128, G = ctx->G;
  const int rt = ctx->bf16 ? tc_rows(ctx) : f32_rows(ctx);
  // CTAs (or CTA pairs) that run at once
  const int wide = !ctx->bf16 && rt == 256 ? ctx->num_sms / 2 : ctx->num_sms;
  std::vector<PgPart>& units = ctx->tc_units;
  units.clear();
  for (const auto& b : bs) {
    const long long rows = (long long)b.n_new * G;
    if (!b.tc) continue;
    const int pos0 = b.len - b.n_new;
    int img0 = 0;
    if (!ctx->bf16) {
      const int t0 = first_key(ctx, win, pos0) / tile, t1 = (b.len + tile - 1) / tile;
      img0 = (int)prep->size() - t0;
      for (int t = t0; t < t1; ++t) prep->push_back({b.tbl, t * tile, b.len, img0 + t});
    }
    for (long long r0 = 0; r0 < rows; r0 += rt)
      for (int h = 0; h < ctx->cfg.n_kv_heads; ++h) {
        PgPart u{};
        u.tbl = b.tbl;
        u.q_row0 = b.q_row0;
        u.pos0 = pos0;
        u.r0 = (int)r0;
        u.n_rows = (int)std::min<long long>(rt, rows - r0);
        u.kvh = h;
        u.key_hi = pos0 + (int)((r0 + u.n_rows - 1) / G) + 1;
        u.tile0 = first_key(ctx, win, pos0 + (int)(r0 / G)) / tile;
        u.tile1 = (u.key_hi + tile - 1) / tile;
        u.img = img0;
        units.push_back(u);
      }
  }
  // A part's time is its tiles times what a tile costs: of bf16 blocks of more than 128 rows 3.8K cycles, of up to 128
  // rows (two streams of tiles) about half of that, more where small pages bound the loads.
  auto weight = [&](const PgPart& u) { return ctx->bf16 && rt == 256 ? (u.n_rows > 128 ? 5 : 3) : 1; };
  // no part is shorter than 1024 keys: below that the merge's launch costs more than the split saves
  const int least = 1024 / tile;
  auto parts_of = [&](const PgPart& u, long long share) {
    const int n = u.tile1 - u.tile0, w = weight(u), cap = (int)std::max<long long>(least, (share + w - 1) / w);
    return (n + cap - 1) / cap;
  };
  // The share of a part.  Candidates: the smallest with which all parts run at once, and fractions of an SM's part of
  // everything, whose parts come in more than one wave but even out ragged lengths; each is judged by laying its parts,
  // longest first, on the SMs that are free first.  A part's start costs about 4.5K cycles, the merge's launch 5K.
  const double start = ctx->bf16 ? (rt == 256 ? 6 : 2) : 1, join = start;
  long long total = 0, longest = 0;
  for (const auto& u : units) {
    const long long c = (long long)weight(u) * (u.tile1 - u.tile0);
    total += c;
    longest = std::max(longest, c);
  }
  const long long even = std::max<long long>(1, (total + wide - 1) / wide);
  long long share = even;
  if ((int)units.size() <= 2 * wide) {
    auto count = [&](long long s) {
      long long n = 0;
      for (const auto& u : units) n += parts_of(u, s);
      return n;
    };
    auto makespan = [&](long long s) {
      std::vector<double> cost;
      bool split = false;
      for (const auto& u : units) {
        const int k = parts_of(u, s);
        split |= k > 1;
        cost.insert(cost.end(), k, start + (double)weight(u) * (u.tile1 - u.tile0) / k);
      }
      std::sort(cost.begin(), cost.end(), std::greater<double>());
      std::vector<double> sm(wide, 0.0);  // a min-heap of the times at which SMs are free
      double end = 0;
      for (double c : cost) {
        std::pop_heap(sm.begin(), sm.end(), std::greater<double>());
        sm.back() += c;
        end = std::max(end, sm.back());
        std::push_heap(sm.begin(), sm.end(), std::greater<double>());
      }
      return end + (split ? join : 0);
    };
    std::vector<long long> tries;
    if ((int)units.size() <= wide) {
      long long lo = even, hi = std::max(longest, lo);
      while (lo < hi) {
        const long long mid = (lo + hi) / 2;
        if (count(mid) <= wide)
          hi = mid;
        else
          lo = mid + 1;
      }
      tries.push_back(hi);
    }
    for (int f = 1; f <= 3; ++f) tries.push_back(std::max<long long>(1, even / f));
    double best = 1e300;
    for (long long s : tries) {
      if (count(s) > 2 * wide) continue;  // the workspace's parts
      const double m = makespan(s);
      if (m < best) best = m, share = s;
    }
  }
  int slot = 0;
  for (const auto& u : units) {
    const int n = u.tile1 - u.tile0, k = parts_of(u, share);
    for (int i = 0; i < k; ++i) {
      PgPart p = u;
      p.tile0 = u.tile0 + (int)((long long)n * i / k);
      p.tile1 = u.tile0 + (int)((long long)n * (i + 1) / k);
      p.part = i;
      p.n_parts = k;
      p.slot = slot;  // of part 0
      parts->push_back(p);
    }
    if (k > 1) {
      PgPart m = u;
      m.n_parts = k;
      m.slot = slot;
      merges->push_back(m);
      slot += k;
    }
  }
  std::stable_sort(parts->begin(), parts->end(), [&](const PgPart& a, const PgPart& b) {
    return weight(a) * (a.tile1 - a.tile0) > weight(b) * (b.tile1 - b.tile0);
  });
}

// Plans a batch: the lists of the kernels (the context's vectors, so that a step allocates nothing), the header, the words of
// the description, and where in it the n_jobs page copies are.  Reads lengths and page counts from bs, not the books.
int plan_batch(Ctx* ctx, const std::vector<BatchSeq>& bs, int n_tokens, size_t tbl_words, size_t n_jobs, PgHeader* out, size_t* words,
               size_t* jobs_at) {
  PgHeader h{};
  h.n_tokens = n_tokens;
  h.n_seqs = (int)bs.size();
  int max_rows = 0;
  for (const auto& b : bs)
    if (!b.tc) max_rows = std::max(max_rows, b.n_new * ctx->G);
  h.row_nt = std::min(max_rows <= 8 ? 1 : 2, row_max_nt(ctx));
  size_t at = kPgHdrWords;
  auto place = [&](size_t bytes) {
    at = (at + 3) & ~(size_t)3;  // records are read 16 bytes at a time
    const size_t here = at;
    at += bytes / 4;
    return here;
  };
  const int n_lists = ctx->swa ? 2 : 1;
  for (int v = 0; v < n_lists; ++v) {
    auto& p = ctx->plan[v];
    p.first.clear(), p.segs.clear(), p.parts.clear(), p.merges.clear(), p.prep.clear();
    plan_rows(ctx, v == 1, bs, h.row_nt, &p.first, &p.segs);
    plan_tc(ctx, v == 1, bs, &p.parts, &p.merges, &p.prep);
    PgLists& l = h.lists[v];
    l.row_ctas = p.first.empty() ? 0 : (int)p.first.size() - 1;
    l.row_first = (int)place(p.first.size() * 4);
    l.row_segs = (int)place(p.segs.size() * sizeof(PgSeg));
    l.n_tc = (int)p.parts.size();
    l.tc_parts = (int)place(p.parts.size() * sizeof(PgPart));
    l.n_merge = (int)p.merges.size();
    l.merges = (int)place(p.merges.size() * sizeof(PgPart));
    l.n_prep = (int)p.prep.size();
    l.prep = (int)place(p.prep.size() * sizeof(PgPrep));
  }
  h.tok = (int)place((size_t)n_tokens * sizeof(int2));
  h.tbl = (int)place(tbl_words * 4);
  *jobs_at = place(n_jobs * sizeof(int4));
  if (at > ctx->batch_words) return fail(ctx, L3P_E_RANGE, "batch description of %zu words", at);
  *out = h;
  *words = at;
  return L3P_OK;
}

// Writes the planned batch to `w`, its tables and token rows from the books.
void write_batch(const Ctx* ctx, const PgHeader& h, const std::vector<BatchSeq>& bs, const int* seqs, const std::vector<int4>& jobs,
                 size_t jobs_at, int* w) {
  auto put = [&](size_t where, const void* p, size_t bytes) {
    if (bytes) memcpy(w + where, p, bytes);
  };
  memset(w, 0, kPgHdrWords * 4);
  memcpy(w, &h, sizeof h);
  for (int v = 0; v < (ctx->swa ? 2 : 1); ++v) {
    const auto& p = ctx->plan[v];
    const PgLists& l = h.lists[v];
    put(l.row_first, p.first.data(), p.first.size() * 4);
    put(l.row_segs, p.segs.data(), p.segs.size() * sizeof(PgSeg));
    put(l.tc_parts, p.parts.data(), p.parts.size() * sizeof(PgPart));
    put(l.merges, p.merges.data(), p.merges.size() * sizeof(PgPart));
    put(l.prep, p.prep.data(), p.prep.size() * sizeof(PgPrep));
  }
  int* tbl = w + h.tbl;
  for (size_t i = 0; i < bs.size(); ++i) {
    const auto& s = ctx->seqs[seqs[i]];
    const auto& b = bs[i];
    for (int t = 0; t < b.n_new; ++t) {
      const int pos = b.len - b.n_new + t;
      int* tok = w + h.tok + 2 * (b.q_row0 + t);
      tok[0] = s.pages[pos >> ctx->shift] * ctx->cfg.page_size + (pos & (ctx->cfg.page_size - 1));
      tok[1] = pos;
    }
    put(tbl - w, s.pages.data(), s.pages.size() * 4);
    tbl += s.pages.size();
  }
  put(jobs_at, jobs.data(), jobs.size() * sizeof(int4));
}

// Words of the largest batch block: bounds on what plan_batch lays out.
size_t batch_capacity(const Ctx* ctx) {
  const auto& c = ctx->cfg;
  const size_t max_len = c.max_seq_len, rows = (size_t)c.max_tokens * ctx->G, kv = c.n_kv_heads, seqs = c.max_seqs;
  const bool only_rows = row_limit(ctx) == INT_MAX;
  // units of the row kernel: blocks of at least 8 rows; segments: one more per CTA at most
  const size_t row_units = only_rows ? kv * (rows / 8 + seqs) : kv * (row_limit(ctx) / 8) * seqs;
  // units of the tensor-core kernels: blocks of at least 128 rows; parts: 3 num_sms more at most, as many merged units
  const size_t tc_units = only_rows ? 0 : kv * (rows / 128 + seqs);
  const size_t tiles = only_rows || ctx->bf16 ? 0 : 4 * seqs * ((max_len + 127) / 128 + 1);
  const size_t list = (row_units + kPgMaxCtas) * 16 + kPgMaxCtas + 1 + (tc_units + 6 * (size_t)ctx->num_sms) * 16 + tiles + 5 * 4;
  const size_t table = seqs * ((max_len + c.page_size - 1) / c.page_size);
  return kPgHdrWords + (ctx->swa ? 2 : 1) * list + 2 * (size_t)c.max_tokens + table + 4 * seqs + 64;
}

void release(Ctx* ctx) {
  cudaFree(ctx->storage);
  cudaFree(ctx->batch);
  cudaFree(ctx->jobs);
  for (auto& s : ctx->slots) {
    if (s.host) cudaFreeHost(s.host);
    if (s.done) cudaEventDestroy(s.done);
  }
  cudaFree(ctx->ws_o);
  cudaFree(ctx->ws_ml);
  cudaFree(ctx->tickets);
  cudaFree(ctx->tc_o);
  cudaFree(ctx->tc_ml);
  cudaFree(ctx->img);
  cudaFree(ctx->v_flags);
  if (ctx->rope_tab_swa != ctx->rope_tab) cudaFree(ctx->rope_tab_swa);
  cudaFree(ctx->rope_tab);
  cudaFree(ctx->qk_norm);
  for (void* p : ctx->retired) cudaFree(p);
  if (ctx->err_host) cudaFreeHost(ctx->err_host);
}

// Runs `f`, turning a host allocation failure into L3P_E_NOMEM: no C++
// exception leaves the C ABI.
template <typename F>
int guarded(Ctx* ctx, F f) {
  try {
    return f();
  } catch (const std::bad_alloc&) {
    return fail(ctx, L3P_E_NOMEM, "host memory is exhausted");
  } catch (...) {
    return fail(ctx, L3P_E_NOMEM, "host library failure");
  }
}

// Why the last create of this thread failed: its context is gone by then.
thread_local char g_create_error[512] = "";

int refuse(int code, const char* text) {
  snprintf(g_create_error, sizeof g_create_error, "%s", text);
  return code;
}

int create(const l3p_paged_config& in, Ctx** out) {
  l3p_paged_config c = in;
  if (c.n_layers <= 0 || c.n_heads <= 0 || c.n_kv_heads <= 0) return refuse(L3P_E_INVAL, "n_layers, n_heads and n_kv_heads are positive");
  if (c.n_heads % c.n_kv_heads != 0) return refuse(L3P_E_INVAL, "n_heads is a multiple of n_kv_heads");
  if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256) return refuse(L3P_E_UNSUPPORTED, "head_dim is 64, 128 or 256");
  if (c.page_size != 16 && c.page_size != 32 && c.page_size != 64 && c.page_size != 128)
    return refuse(L3P_E_UNSUPPORTED, "page_size is 16, 32, 64 or 128");
  if (c.n_pages <= 0 || c.max_seqs <= 0 || c.max_tokens <= 0 || c.max_seq_len < 0)
    return refuse(L3P_E_INVAL, "n_pages, max_seqs and max_tokens are positive, max_seq_len is not negative");
  if (c.dtype != L3P_PAGED_F32 && c.dtype != L3P_PAGED_BF16) return refuse(L3P_E_INVAL, "dtype is L3P_PAGED_F32 or L3P_PAGED_BF16");
  if (!std::isfinite(c.scale) || c.scale < 0.f) return refuse(L3P_E_INVAL, "scale is finite and not negative");
  if (c.swa_window < 0 || c.swa_pattern < 0 || c.device < 0)
    return refuse(L3P_E_INVAL, "swa_window, swa_pattern and device are not negative");
  // positions, storage rows and query rows are counted in 32 bits
  const long long pool_pos = (long long)c.n_pages * c.page_size;
  if (pool_pos > INT_MAX / 2) return refuse(L3P_E_RANGE, "the pool has more than 2^30 positions");
  if (c.max_seqs > 65536) return refuse(L3P_E_RANGE, "max_seqs is above 65536");
  if (c.max_seq_len == 0 || c.max_seq_len > pool_pos) c.max_seq_len = (int)pool_pos;
  if ((long long)c.max_tokens * c.n_heads > INT_MAX / 2) return refuse(L3P_E_RANGE, "max_tokens * n_heads is above 2^30");
  // rows of the tensor map; by division, since the product may pass 64 bits
  if (c.n_layers > INT_MAX / pool_pos || c.n_kv_heads > INT_MAX / (2 * pool_pos * c.n_layers))
    return refuse(L3P_E_RANGE, "the pool has more than 2^31 rows");
  Ctx* ctx = new Ctx;
  ctx->cfg = c;
  ctx->hd = c.head_dim;
  ctx->G = c.n_heads / c.n_kv_heads;
  ctx->bf16 = c.dtype == L3P_PAGED_BF16;
  ctx->es = ctx->bf16 ? 2 : 4;
  while ((1 << ctx->shift) < c.page_size) ++ctx->shift;
  ctx->swa = c.is_gemma3 && c.swa_window > 0 && c.swa_pattern > 0;
  ctx->scale = c.scale != 0.f ? c.scale : 1.0f / sqrtf((float)c.head_dim);
  *out = ctx;
  DeviceScope dev(c.device);
  ctx->block_bytes = (size_t)c.page_size * c.head_dim * ctx->es;
  ctx->page_bytes = ctx->block_bytes * c.n_kv_heads * 2 * c.n_layers;
  cudaDeviceProp prop;
  PG_CUDA(ctx, cudaGetDeviceProperties(&prop, c.device));
  ctx->num_sms = prop.multiProcessorCount;
  ctx->batch_words = batch_capacity(ctx);
  if (ctx->batch_words > (1u << 29))
    return fail(ctx, L3P_E_RANGE, "max_seqs, max_tokens and max_seq_len make a batch description of %zu words",
                ctx->batch_words);
  const size_t bytes = ctx->page_bytes * c.n_pages;
  ctx->jobs_cap = (size_t)c.n_pages;
  if (cudaMalloc(&ctx->storage, bytes) != cudaSuccess || cudaMalloc(&ctx->batch, ctx->batch_words * 4) != cudaSuccess ||
      cudaMalloc(&ctx->jobs, ctx->jobs_cap * sizeof(int4)) != cudaSuccess) {
    cudaGetLastError();
    return fail(ctx, L3P_E_NOMEM, "a pool of %zu bytes does not fit on the device", bytes);
  }
  PG_CUDA(ctx, cudaMemset(ctx->storage, 0, bytes));
  PG_CUDA(ctx, cudaHostAlloc(&ctx->err_host, sizeof(int), cudaHostAllocMapped));
  *ctx->err_host = 0;
  PG_CUDA(ctx, cudaHostGetDevicePointer(&ctx->err_dev, ctx->err_host, 0));
  for (auto& s : ctx->slots) PG_CUDA(ctx, cudaEventCreateWithFlags(&s.done, cudaEventDisableTiming));
  ctx->seqs.resize(c.max_seqs);
  ctx->refs.assign(c.n_pages, 0);
  ctx->fill.assign(c.n_pages, 0);
  ctx->free_heap.resize(c.n_pages);
  for (int i = 0; i < c.n_pages; ++i) ctx->free_heap[i] = i;  // ascending: a min-heap already
  if (int rc = init_kv(ctx)) return rc;
  if (int rc = init_rows(ctx)) return rc;
  if (int rc = ctx->bf16 ? init_tc(ctx) : init_f32(ctx)) return rc;
  PG_CUDA(ctx, cudaDeviceSynchronize());  // the storage is zero before any stream of the caller's writes it
  return L3P_OK;
}

int begin(Ctx* ctx, int n_seqs, const int* ids, const int* n_new, cudaStream_t s) {
  if (int rc = check_seqs(ctx, n_seqs, ids)) return rc;
  long long tokens = 0, need = 0;
  for (int i = 0; i < n_seqs; ++i) {
    const auto& q = ctx->seqs[ids[i]];
    if (n_new[i] < 0) return fail(ctx, L3P_E_INVAL, "sequence %d grows by %d tokens", ids[i], n_new[i]);
    if ((long long)q.len + n_new[i] > ctx->cfg.max_seq_len)
      return fail(ctx, L3P_E_RANGE, "sequence %d would hold %lld of at most %d positions", ids[i],
                  (long long)q.len + n_new[i], ctx->cfg.max_seq_len);
    tokens += n_new[i];
    need += pages_for(ctx, q.len + n_new[i]) - (int)q.pages.size();
  }
  if (tokens > ctx->cfg.max_tokens)
    return fail(ctx, L3P_E_RANGE, "%lld new tokens, at most %d", tokens, ctx->cfg.max_tokens);
  // shared last pages that a sequence grows into: the holder that finds others
  // beside it takes a copy; a page all of whose holders grow stays with the last one
  std::vector<std::pair<int, int>> cow;  // (index in the batch, page)
  for (int i = 0; i < n_seqs; ++i) {
    const auto& q = ctx->seqs[ids[i]];
    if (n_new[i] == 0 || (q.len & (ctx->cfg.page_size - 1)) == 0) continue;
    const int p = q.pages.back();
    if (ctx->refs[p] > 1) cow.push_back({i, p});
  }
  {
    std::vector<std::pair<int, int>> take;
    std::vector<int> count(cow.empty() ? 0 : ctx->cfg.n_pages, 0);
    for (const auto& x : cow)
      if (ctx->refs[x.second] - count[x.second] > 1) {
        ++count[x.second];
        take.push_back(x);
      }
    cow.swap(take);
  }
  need += (long long)cow.size();
  if (need > (long long)ctx->free_heap.size())
    return fail(ctx, L3P_E_NOMEM, "the batch needs %lld pages, %zu are free", need, ctx->free_heap.size());
  if (int rc = refuse_capture(ctx, s, "begin")) return rc;

  // Everything that may find no memory comes before the books move: the plan, a slot for it, room in the lists.
  std::vector<int4> jobs;
  jobs.reserve(cow.size());
  std::vector<BatchSeq> bs(n_seqs);
  int row = 0, tbl = 0, max_pos = 0;
  for (int i = 0; i < n_seqs; ++i) {
    auto& q = ctx->seqs[ids[i]];
    const int len = q.len + n_new[i], n_pages = pages_for(ctx, len);
    reserve_pages(&q.pages, n_pages);
    bs[i] = {row, n_new[i], len, tbl, false};
    row += n_new[i];
    if (n_new[i] > 0) max_pos = std::max(max_pos, len);
    tbl += n_pages;
  }
  choose_paths(ctx, &bs);
  PgHeader hdr;
  size_t words, jobs_at;
  if (int rc = plan_batch(ctx, bs, row, tbl, cow.size(), &hdr, &words, &jobs_at)) return rc;
  Ctx::Slot* slot;
  if (int rc = take_slot(ctx, words, &slot)) return rc;
  if (int rc = prepare_f32(ctx, hdr)) return rc;

  // Give out pages, in batch order, a sequence's copy first.
  ctx->batch_valid = false;
  size_t next = 0;
  for (int i = 0; i < n_seqs; ++i) {
    auto& q = ctx->seqs[ids[i]];
    if (next < cow.size() && cow[next].first == i) {
      const int src = q.pages.back(), dst = take_page(ctx), rows = q.len & (ctx->cfg.page_size - 1);
      jobs.push_back(make_int4(src, dst, rows, 0));
      drop_page(ctx, src);
      ctx->fill[dst] = rows;
      q.pages.back() = dst;
      ++next;
    }
    const int len = bs[i].len, n_pages = pages_for(ctx, len);
    while ((int)q.pages.size() < n_pages) q.pages.push_back(take_page(ctx));
    for (int pos = q.len; pos < len; pos = (pos | (ctx->cfg.page_size - 1)) + 1) {
      const int p = q.pages[pos >> ctx->shift];
      ctx->fill[p] = std::max(ctx->fill[p], std::min(ctx->cfg.page_size, len - (pos & ~(ctx->cfg.page_size - 1))));
    }
    q.len = len;
  }
  ctx->hdr = hdr;
  ctx->max_pos_in_batch = max_pos;
  write_batch(ctx, hdr, bs, ids, jobs, jobs_at, slot->host);
  if (int rc = upload(ctx, slot, ctx->batch, words, s)) return rc;
  if (!jobs.empty())
    if (int rc = launch_page_copy(ctx, ctx->batch + jobs_at, (int)jobs.size(), s)) return rc;
  ctx->batch_valid = true;
  return L3P_OK;
}

int copy_seqs(Ctx* ctx, int n, const int* ids, int* children, cudaStream_t s) {
  for (int i = 0; i < n; ++i)
    if (int rc = check_seq(ctx, ids[i])) return rc;
  if (n > free_seq_count(ctx))
    return fail(ctx, L3P_E_NOMEM, "%d sequences more than max_seqs = %d allows", n, ctx->cfg.max_seqs);
  long long need = 0;
  for (int i = 0; i < n; ++i) need += ctx->seqs[ids[i]].pages.size();
  if (need > (long long)ctx->free_heap.size())
    return fail(ctx, L3P_E_NOMEM, "the copies need %lld pages, %zu are free", need, ctx->free_heap.size());
  if (int rc = refuse_capture(ctx, s, "copy")) return rc;
  // everything that may find no memory comes before the books move
  std::vector<int4> jobs;
  jobs.reserve(need);
  std::vector<std::vector<int>> pages(n);
  for (int i = 0; i < n; ++i) pages[i].reserve(ctx->seqs[ids[i]].pages.size());
  Ctx::Slot* slot = nullptr;
  if (need > 0)
    if (int rc = take_slot(ctx, need * 4, &slot)) return rc;
  for (int i = 0; i < n; ++i) {
    const int child = new_seq(ctx);
    auto& dst = ctx->seqs[child];
    const auto& src = ctx->seqs[ids[i]];
    dst.len = src.len;
    dst.pages.swap(pages[i]);
    for (size_t k = 0; k < src.pages.size(); ++k) {
      const int p = take_page(ctx), rows = std::min(ctx->cfg.page_size, src.len - (int)k * ctx->cfg.page_size);
      ctx->fill[p] = rows;
      dst.pages.push_back(p);
      jobs.push_back(make_int4(src.pages[k], p, rows, 0));
    }
    children[i] = child;
  }
  return copy_pages(ctx, jobs, slot, s);
}

int compact(Ctx* ctx, int* n_used, cudaStream_t s) {
  if (int rc = refuse_capture(ctx, s, "compact")) return rc;
  const int k = ctx->cfg.n_pages - (int)ctx->free_heap.size();
  std::vector<int4> jobs;
  jobs.reserve(std::min(k, ctx->cfg.n_pages - k));
  std::vector<int> moved(ctx->cfg.n_pages, -1);
  int dst = 0;
  for (int p = k; p < ctx->cfg.n_pages; ++p) {
    if (ctx->refs[p] == 0) continue;
    while (ctx->refs[dst] != 0) ++dst;  // fewer used pages below k than k, so dst stays below k
    moved[p] = dst;
    jobs.push_back(make_int4(p, dst, ctx->fill[p], 0));
    ++dst;
  }
  if (!jobs.empty()) {
    Ctx::Slot* slot;
    if (int rc = take_slot(ctx, jobs.size() * 4, &slot)) return rc;
    ctx->batch_valid = false;
    if (int rc = copy_pages(ctx, jobs, slot, s)) return rc;
    for (const auto& j : jobs) {
      ctx->refs[j.y] = ctx->refs[j.x];
      ctx->fill[j.y] = ctx->fill[j.x];
      ctx->refs[j.x] = 0;
    }
    for (auto& q : ctx->seqs)
      for (auto& p : q.pages)
        if (moved[p] >= 0) p = moved[p];
    ctx->free_heap.clear();
    for (int p = k; p < ctx->cfg.n_pages; ++p) ctx->free_heap.push_back(p);
  }
  if (n_used) *n_used = k;
  return L3P_OK;
}

}  // namespace

L3P_API const char* l3p_paged_create_error(void) { return g_create_error; }

L3P_API int l3p_paged_create(const l3p_paged_config* cfg, l3p_paged_ctx** out) {
  if (!cfg || !out) return refuse(L3P_E_INVAL, "null pointer");
  *out = nullptr;
  g_create_error[0] = 0;
  Ctx* ctx = nullptr;
  const int rc = guarded(nullptr, [&] { return create(*cfg, &ctx); });
  if (rc != L3P_OK) {
    if (ctx && ctx->last_error[0]) refuse(rc, ctx->last_error);
    if (!g_create_error[0]) refuse(rc, "host memory is exhausted");
    if (ctx) {
      DeviceScope dev(ctx->cfg.device);
      release(ctx);
      delete ctx;
    }
    return rc;
  }
  *out = ctx;
  return L3P_OK;
}

L3P_API void l3p_paged_destroy(l3p_paged_ctx* ctx) {
  if (!ctx) return;
  DeviceScope dev(ctx->cfg.device);
  cudaDeviceSynchronize();
  release(ctx);
  delete ctx;
}

L3P_API const char* l3p_paged_last_error(const l3p_paged_ctx* ctx) { return ctx ? ctx->last_error : ""; }

L3P_API long long l3p_paged_launch_count(const l3p_paged_ctx* ctx) { return ctx ? ctx->launches : L3P_E_INVAL; }

L3P_API int l3p_paged_check(l3p_paged_ctx* ctx, void* stream) {
  if (!ctx) return L3P_E_INVAL;
  DeviceScope dev(ctx->cfg.device);
  if (capturing(as_stream(stream))) return fail(ctx, L3P_E_INVAL, "check waits for the stream: not during stream capture");
  PG_CUDA(ctx, cudaStreamSynchronize(as_stream(stream)));
  const int e = *ctx->err_host;
  *ctx->err_host = 0;
  if (e == kErrTimeout) return fail(ctx, L3P_E_TIMEOUT, "a bounded wait in a kernel gave up");
  if (e != 0) return fail(ctx, L3P_E_INVAL, "a captured launch met a batch that it does not serve");
  return L3P_OK;
}

L3P_API int l3p_paged_storage(l3p_paged_ctx* ctx, void** base, size_t* bytes) {
  if (!ctx || !base || !bytes) return ctx ? fail(ctx, L3P_E_INVAL, "null pointer") : L3P_E_INVAL;
  *base = ctx->storage;
  *bytes = ctx->page_bytes * ctx->cfg.n_pages;
  return L3P_OK;
}

L3P_API int l3p_paged_seq_new(l3p_paged_ctx* ctx, int* seq) {
  if (!ctx || !seq) return ctx ? fail(ctx, L3P_E_INVAL, "null pointer") : L3P_E_INVAL;
  return guarded(ctx, [&] {
    const int id = new_seq(ctx);
    if (id < 0) return fail(ctx, L3P_E_NOMEM, "max_seqs = %d sequences exist", ctx->cfg.max_seqs);
    *seq = id;
    return (int)L3P_OK;
  });
}

L3P_API int l3p_paged_seq_fork(l3p_paged_ctx* ctx, int seq, int n_tokens, int n, int* children) {
  if (!ctx || !children || n < 0) return ctx ? fail(ctx, L3P_E_INVAL, "bad argument") : L3P_E_INVAL;
  return guarded(ctx, [&]() -> int {
    if (int rc = check_seq(ctx, seq)) return rc;
    const int len = n_tokens < 0 ? ctx->seqs[seq].len : n_tokens;
    if (len > ctx->seqs[seq].len)
      return fail(ctx, L3P_E_RANGE, "sequence %d has %d positions, not %d", seq, ctx->seqs[seq].len, len);
    if (n > free_seq_count(ctx))
      return fail(ctx, L3P_E_NOMEM, "%d sequences more than max_seqs = %d allows", n, ctx->cfg.max_seqs);
    const int n_pages = pages_for(ctx, len);
    const auto& shared = ctx->seqs[seq].pages;
    std::vector<std::vector<int>> pages(n);  // before the books move
    for (auto& p : pages) p.assign(shared.begin(), shared.begin() + n_pages);
    for (int i = 0; i < n; ++i) {
      const int id = new_seq(ctx);
      ctx->seqs[id].pages.swap(pages[i]);
      ctx->seqs[id].len = len;
      for (int p : ctx->seqs[id].pages) ++ctx->refs[p];
      children[i] = id;
    }
    return L3P_OK;
  });
}

L3P_API int l3p_paged_seq_copy(l3p_paged_ctx* ctx, int n, const int* seqs, int* children, void* stream) {
  if (!ctx || n < 0 || (n > 0 && (!seqs || !children))) return ctx ? fail(ctx, L3P_E_INVAL, "bad argument") : L3P_E_INVAL;
  DeviceScope dev(ctx->cfg.device);
  return guarded(ctx, [&] { return copy_seqs(ctx, n, seqs, children, as_stream(stream)); });
}

L3P_API int l3p_paged_seq_truncate(l3p_paged_ctx* ctx, int seq, int n_tokens) {
  if (!ctx || n_tokens < 0) return ctx ? fail(ctx, L3P_E_INVAL, "bad argument") : L3P_E_INVAL;
  return guarded(ctx, [&]() -> int {
    if (int rc = check_seq(ctx, seq)) return rc;
    auto& q = ctx->seqs[seq];
    if (n_tokens > q.len) return fail(ctx, L3P_E_RANGE, "sequence %d has %d positions, not %d", seq, q.len, n_tokens);
    ctx->batch_valid = false;
    while ((int)q.pages.size() > pages_for(ctx, n_tokens)) {
      drop_page(ctx, q.pages.back());
      q.pages.pop_back();
    }
    q.len = n_tokens;
    return L3P_OK;
  });
}

L3P_API int l3p_paged_seq_free(l3p_paged_ctx* ctx, int n, const int* seqs) {
  if (!ctx || n < 0 || (n > 0 && !seqs)) return ctx ? fail(ctx, L3P_E_INVAL, "bad argument") : L3P_E_INVAL;
  return guarded(ctx, [&]() -> int {
    if (int rc = check_seqs(ctx, n, seqs)) return rc;
    if (n > 0) ctx->batch_valid = false;
    for (int i = 0; i < n; ++i) {
      auto& q = ctx->seqs[seqs[i]];
      for (int p : q.pages) drop_page(ctx, p);
      q.pages.clear();
      q.len = 0;
      q.live = false;
    }
    return L3P_OK;
  });
}

L3P_API int l3p_paged_seq_length(l3p_paged_ctx* ctx, int seq, int* n_tokens) {
  if (!ctx || !n_tokens) return ctx ? fail(ctx, L3P_E_INVAL, "null pointer") : L3P_E_INVAL;
  if (int rc = check_seq(ctx, seq)) return rc;
  *n_tokens = ctx->seqs[seq].len;
  return L3P_OK;
}

L3P_API int l3p_paged_tables(l3p_paged_ctx* ctx, int n, const int* seqs, int width, int* table, int* need) {
  if (!ctx || n < 0 || (n > 0 && !seqs) || width < 0) return ctx ? fail(ctx, L3P_E_INVAL, "bad argument") : L3P_E_INVAL;
  int widest = 0;
  for (int i = 0; i < n; ++i) {
    if (int rc = check_seq(ctx, seqs[i])) return rc;
    widest = std::max(widest, (int)ctx->seqs[seqs[i]].pages.size());
  }
  if (need) *need = widest;
  if (!table) return L3P_OK;
  if (width < widest) return fail(ctx, L3P_E_RANGE, "tables of %d pages, rows of %d", widest, width);
  for (int i = 0; i < n; ++i) {
    const auto& p = ctx->seqs[seqs[i]].pages;
    int* row = table + (size_t)i * width;
    std::copy(p.begin(), p.end(), row);
    std::fill(row + p.size(), row + width, -1);
  }
  return L3P_OK;
}

L3P_API int l3p_paged_free_pages(l3p_paged_ctx* ctx, int* n_free) {
  if (!ctx || !n_free) return ctx ? fail(ctx, L3P_E_INVAL, "null pointer") : L3P_E_INVAL;
  *n_free = (int)ctx->free_heap.size();
  return L3P_OK;
}

L3P_API int l3p_paged_compact(l3p_paged_ctx* ctx, int* n_used, void* stream) {
  if (!ctx) return L3P_E_INVAL;
  DeviceScope dev(ctx->cfg.device);
  return guarded(ctx, [&] { return compact(ctx, n_used, as_stream(stream)); });
}

L3P_API int l3p_paged_begin(l3p_paged_ctx* ctx, int n_seqs, const int* seqs, const int* n_new, void* stream) {
  if (!ctx || n_seqs < 0 || (n_seqs > 0 && (!seqs || !n_new)))
    return ctx ? fail(ctx, L3P_E_INVAL, "bad argument") : L3P_E_INVAL;
  DeviceScope dev(ctx->cfg.device);
  return guarded(ctx, [&] { return begin(ctx, n_seqs, seqs, n_new, as_stream(stream)); });
}

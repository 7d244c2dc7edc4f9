// l3p_paged_kv.cu -- entry points that write the paged cache: rotary tables,
// rotate-and-append, append, and the launcher of page copies.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <vector>

#include "paged_kv.cuh"

using namespace l3p;
using namespace l3p_pg;

namespace l3p_pg {

int launch_page_copy(l3p_paged_ctx* ctx, const int* jobs, int n_jobs, cudaStream_t s) {
  const int blocks = ctx->cfg.n_layers * 2 * ctx->cfg.n_kv_heads;
  const int want = std::max(1, 8 * ctx->num_sms / n_jobs);  // CTAs of a job: a few per SM over all jobs
  const int gx = std::min((blocks + 7) / 8, want);
  for (int at = 0; at < n_jobs; at += 65535) {  // grid y
    const int n = std::min(n_jobs - at, 65535);
    paged_copy_kernel<<<dim3(gx, n), 256, 0, s>>>(reinterpret_cast<const int4*>(jobs) + at,
                                                  static_cast<char*>(ctx->storage), (long long)ctx->page_bytes, blocks,
                                                  (int)ctx->block_bytes, ctx->hd * ctx->es);
    ++ctx->launches;
  }
  PG_CUDA(ctx, cudaGetLastError());
  return L3P_OK;
}

}  // namespace l3p_pg

namespace {

constexpr int kRingBytes = 100 * 1024;  // of a CTA of the streaming rotation: two CTAs per SM

template <typename T>
auto ring_kernel(int hd) {
  return hd == 64 ? paged_rope_ring_kernel<T, 64> : hd == 128 ? paged_rope_ring_kernel<T, 128> : paged_rope_ring_kernel<T, 256>;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Rows of one token at `p`, `stride` values apart (0: dense): a multiple of 16
// bytes, and at least the row.
int check_rows(l3p_paged_ctx* ctx, const char* name, const void* p, long long* stride, int heads) {
  const long long row = (long long)heads * ctx->hd;
  if (!p) return fail(ctx, L3P_E_INVAL, "%s is null", name);
  if (!aligned16(p)) return fail(ctx, L3P_E_INVAL, "%s is not 16-byte aligned", name);
  if (*stride == 0) *stride = row;
  if (*stride < row || *stride * ctx->es % 16 != 0)
    return fail(ctx, L3P_E_INVAL, "%s: a stride of %lld values for rows of %lld", name, *stride, row);
  return L3P_OK;
}

int check_call(l3p_paged_ctx* ctx, int layer) {
  if (layer < 0 || layer >= ctx->cfg.n_layers) return fail(ctx, L3P_E_RANGE, "layer %d of %d", layer, ctx->cfg.n_layers);
  if (!ctx->batch_valid)
    return fail(ctx, L3P_E_INVAL, "there is no current batch: call l3p_paged_begin (freeing, truncating and compacting end a batch)");
  return L3P_OK;
}

// The layer's fields of a launch that writes pages.
PgKvArgs kv_args(l3p_paged_ctx* ctx, int layer) {
  PgKvArgs a{};
  a.batch = ctx->batch;
  a.n_tokens = ctx->hdr.n_tokens;
  a.storage = static_cast<char*>(ctx->storage) + (size_t)layer * 2 * ctx->cfg.n_kv_heads * ctx->block_bytes;
  a.page_elems = (long long)(ctx->page_bytes / ctx->es);
  a.v_off = (long long)(ctx->block_bytes / ctx->es) * ctx->cfg.n_kv_heads;
  a.page_size = ctx->cfg.page_size;
  a.shift = ctx->shift;
  a.n_heads = ctx->cfg.n_heads;
  a.n_kv = ctx->cfg.n_kv_heads;
  a.max_pos = ctx->rope_max;
  a.err = ctx->err_dev;
  return a;
}

template <typename T>
int launch_rope(l3p_paged_ctx* ctx, const PgKvArgs& a, int grid, cudaStream_t s) {
  auto kernel = ctx->hd == 64 ? paged_rope_kernel<T, 64> : ctx->hd == 128 ? paged_rope_kernel<T, 128> : paged_rope_kernel<T, 256>;
  return launch(ctx, kernel, dim3(grid), kPgKvWarps * 32, 0, s, 1, a);
}

template <typename T>
int launch_rope_ring(l3p_paged_ctx* ctx, const PgKvArgs& a, cudaStream_t s) {
  PgRingArgs g{};
  g.q_bytes = ctx->cfg.n_heads * ctx->hd * ctx->es;
  g.kv_bytes = ctx->cfg.n_kv_heads * ctx->hd * ctx->es;
  g.tab_bytes = ctx->rotary_dim / 2 * (int)sizeof(float2);
  g.stage_bytes = (g.q_bytes + 2 * g.kv_bytes + g.tab_bytes + 127) / 128 * 128;
  g.stages = std::min(kPgRingStages, kRingBytes / g.stage_bytes);
  return launch(ctx, ring_kernel<T>(ctx->hd), dim3(std::min(a.n_tokens, 2 * ctx->num_sms)), kPgRingThreads, g.stages * g.stage_bytes, s, 1, a, g);
}

int set_rope(l3p_paged_ctx* ctx, const l3p_paged_rope_config& in) {
  l3p_paged_rope_config r = in;
  const int hd = ctx->hd;
  if (r.rotary_dim == 0) r.rotary_dim = hd;
  if (r.rotary_dim < 2 || r.rotary_dim > hd || r.rotary_dim % 2 != 0)
    return fail(ctx, L3P_E_INVAL, "rotary_dim %d of head_dim %d", r.rotary_dim, hd);
  if (r.layout != L3P_ROPE_INTERLEAVED && r.layout != L3P_ROPE_HALF) return fail(ctx, L3P_E_INVAL, "layout %d", r.layout);
  if (r.scaling < L3P_ROPE_SCALE_NONE || r.scaling > L3P_ROPE_SCALE_YARN)
    return fail(ctx, L3P_E_INVAL, "scaling %d", r.scaling);
  if (r.max_pos <= 0) return fail(ctx, L3P_E_INVAL, "max_pos %d", r.max_pos);
  if ((r.q_norm == nullptr) != (r.k_norm == nullptr)) return fail(ctx, L3P_E_INVAL, "q_norm and k_norm go together");
  auto or_default = [](float v, float d) { return v == 0.f ? d : v; };
  r.theta = or_default(r.theta, 500000.f);
  r.theta_swa = or_default(r.theta_swa, 10000.f);
  r.low_freq = or_default(r.low_freq, 1.f);
  r.high_freq = or_default(r.high_freq, 4.f);
  r.beta_fast = or_default(r.beta_fast, 32.f);
  r.beta_slow = or_default(r.beta_slow, 1.f);
  r.rms_norm_eps = or_default(r.rms_norm_eps, 1e-5f);
  if (!(r.theta > 1.f) || !(r.theta_swa > 1.f) || !std::isfinite(r.theta) || !std::isfinite(r.theta_swa) ||
      !(r.rms_norm_eps > 0.f) || !std::isfinite(r.rms_norm_eps))
    return fail(ctx, L3P_E_INVAL, "theta and theta_swa are above 1, rms_norm_eps above 0");
  if (r.scaling != L3P_ROPE_SCALE_NONE && (!(r.factor >= 1.f) || !std::isfinite(r.factor)))
    return fail(ctx, L3P_E_INVAL, "factor %g is not at least 1", r.factor);
  if (r.scaling >= L3P_ROPE_SCALE_BANDS && r.original_len <= 0) return fail(ctx, L3P_E_INVAL, "original_len %d", r.original_len);
  if (r.scaling == L3P_ROPE_SCALE_BANDS && !(r.low_freq > 0.f && r.high_freq > r.low_freq))
    return fail(ctx, L3P_E_INVAL, "low_freq %g, high_freq %g", r.low_freq, r.high_freq);
  if (r.scaling == L3P_ROPE_SCALE_YARN && !(r.beta_slow > 0.f && r.beta_fast > r.beta_slow))
    return fail(ctx, L3P_E_INVAL, "beta_slow %g, beta_fast %g", r.beta_slow, r.beta_fast);
  if (!std::isfinite(r.attn_factor) || r.attn_factor < 0.f) return fail(ctx, L3P_E_INVAL, "attn_factor %g", r.attn_factor);

  const int dim = r.rotary_dim, half = dim / 2;
  const double pi = 3.14159265358979323846;
  std::vector<double> freq(half), freq_swa(half);
  double mult = 1.0;
  for (int i = 0; i < half; ++i) {
    freq[i] = pow((double)r.theta, -2.0 * i / dim);
    freq_swa[i] = pow((double)r.theta_swa, -2.0 * i / dim);
  }
  if (r.scaling == L3P_ROPE_SCALE_LINEAR)
    for (double& f : freq) f /= r.factor;
  if (r.scaling == L3P_ROPE_SCALE_BANDS)
    for (double& f : freq) {
      const double turns = r.original_len * f / (2 * pi);  // original_len / wavelength
      const double mix = std::min(1.0, std::max(0.0, (turns - r.low_freq) / ((double)r.high_freq - r.low_freq)));
      f *= (1.0 - mix) / r.factor + mix;
    }
  if (r.scaling == L3P_ROPE_SCALE_YARN) {
    // pair at which a head turns n times over original_len
    auto pair_of = [&](double n) { return dim * log(r.original_len / (n * 2 * pi)) / (2 * log((double)r.theta)); };
    const double from = floor(pair_of(r.beta_fast)), to = ceil(pair_of(r.beta_slow));
    const double lo = std::max(from, 0.0), hi = std::min(to, dim - 1.0);
    for (int i = 0; i < half; ++i) {
      // the ramp's ends are moved to the head's values; where all of it lies before the first or behind the last, its side counts
      const double ramp = to <= 0 ? 1.0 : from > dim - 1.0 ? 0.0 : std::min(1.0, std::max(0.0, (i - lo) / (hi == lo ? 0.001 : hi - lo)));
      freq[i] = freq[i] * (1.0 - ramp) + freq[i] / r.factor * ramp;
    }
    mult = r.attn_factor > 0.f ? r.attn_factor : 0.1 * log((double)r.factor) + 1.0;
  }

  // everything new is built before anything old goes
  ctx->retired.reserve(ctx->retired.size() + 3);
  const size_t n = (size_t)r.max_pos * half;
  float2 *tab = nullptr, *tab_swa = nullptr;
  float* norm = nullptr;
  double* dfreq = nullptr;
  const size_t n_norm = (size_t)ctx->cfg.n_layers * hd;
  auto drop = [&] {
    cudaFree(tab);
    cudaFree(tab_swa);
    cudaFree(norm);
    cudaFree(dfreq);
  };
  if (cudaMalloc(&tab, n * sizeof(float2)) != cudaSuccess || (ctx->swa && cudaMalloc(&tab_swa, n * sizeof(float2)) != cudaSuccess) ||
      (r.q_norm && cudaMalloc(&norm, 2 * n_norm * sizeof(float)) != cudaSuccess) ||
      cudaMalloc(&dfreq, 2 * half * sizeof(double)) != cudaSuccess) {
    cudaGetLastError();
    drop();
    return fail(ctx, L3P_E_NOMEM, "rotary tables of %zu bytes do not fit on the device", n * sizeof(float2) * (ctx->swa ? 2 : 1));
  }
  cudaError_t e = cudaMemcpy(dfreq, freq.data(), half * sizeof(double), cudaMemcpyHostToDevice);
  if (e == cudaSuccess) e = cudaMemcpy(dfreq + half, freq_swa.data(), half * sizeof(double), cudaMemcpyHostToDevice);
  const int grid = (int)std::min<size_t>((n + 255) / 256, (size_t)ctx->num_sms * 16);
  if (e == cudaSuccess) {
    paged_rope_table_kernel<<<grid, 256>>>(tab, dfreq, half, r.max_pos, mult);
    ++ctx->launches;
    if (ctx->swa) {
      paged_rope_table_kernel<<<grid, 256>>>(tab_swa, dfreq + half, half, r.max_pos, 1.0);
      ++ctx->launches;
    }
    e = cudaGetLastError();
  }
  if (e == cudaSuccess && norm) e = cudaMemcpy(norm, r.q_norm, n_norm * sizeof(float), cudaMemcpyHostToDevice);
  if (e == cudaSuccess && norm) e = cudaMemcpy(norm + n_norm, r.k_norm, n_norm * sizeof(float), cudaMemcpyHostToDevice);
  if (e == cudaSuccess) e = cudaDeviceSynchronize();  // also: no kernel still reads the old tables
  if (e != cudaSuccess) {
    drop();
    return fail(ctx, L3P_E_CUDA, "rotary tables: %s", cudaGetErrorString(e));
  }
  cudaFree(dfreq);
  if (ctx->rope_tab_swa != ctx->rope_tab) retire(ctx, ctx->rope_tab_swa, ctx->rope_captured);
  retire(ctx, ctx->rope_tab, ctx->rope_captured);
  retire(ctx, ctx->qk_norm, ctx->rope_captured);
  ctx->rope_captured = false;
  ctx->rope_tab = tab;
  ctx->rope_tab_swa = ctx->swa ? tab_swa : tab;
  ctx->qk_norm = norm;
  ctx->rope_max = r.max_pos;
  ctx->rope_layout = r.layout;
  ctx->rotary_dim = dim;
  ctx->rms_eps = r.rms_norm_eps;
  return L3P_OK;
}

}  // namespace

namespace l3p_pg {

int init_kv(l3p_paged_ctx* ctx) {
  if (ctx->bf16)
    PG_CUDA(ctx, cudaFuncSetAttribute(ring_kernel<__nv_bfloat16>(ctx->hd), cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes));
  else
    PG_CUDA(ctx, cudaFuncSetAttribute(ring_kernel<float>(ctx->hd), cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes));
  return L3P_OK;
}

}  // namespace l3p_pg

L3P_API int l3p_paged_set_rope(l3p_paged_ctx* ctx, const l3p_paged_rope_config* rope) {
  if (!ctx || !rope) return ctx ? fail(ctx, L3P_E_INVAL, "null pointer") : L3P_E_INVAL;
  DeviceScope dev(ctx->cfg.device);
  try {
    return set_rope(ctx, *rope);
  } catch (...) {
    return fail(ctx, L3P_E_NOMEM, "host memory is exhausted");
  }
}

L3P_API int l3p_paged_rope_append_dev(l3p_paged_ctx* ctx, int layer, const void* q, long long q_stride, const void* k,
                                      long long k_stride, const void* v, long long v_stride, void* q_out,
                                      long long q_out_stride, void* stream) {
  if (!ctx) return L3P_E_INVAL;
  if (int rc = check_call(ctx, layer)) return rc;
  if (!ctx->rope_tab) return fail(ctx, L3P_E_INVAL, "l3p_paged_set_rope has not been called on this context");
  if (ctx->max_pos_in_batch > ctx->rope_max)
    return fail(ctx, L3P_E_RANGE, "the batch reaches position %d, the rotary tables %d", ctx->max_pos_in_batch - 1, ctx->rope_max - 1);
  const auto& c = ctx->cfg;
  if (ctx->hdr.n_tokens == 0) return L3P_OK;
  if (int rc = check_rows(ctx, "q", q, &q_stride, c.n_heads)) return rc;
  if (int rc = check_rows(ctx, "k", k, &k_stride, c.n_kv_heads)) return rc;
  if (int rc = check_rows(ctx, "v", v, &v_stride, c.n_kv_heads)) return rc;
  if (int rc = check_rows(ctx, "q_out", q_out, &q_out_stride, c.n_heads)) return rc;
  DeviceScope dev(c.device);
  PgKvArgs a = kv_args(ctx, layer);
  a.q = q, a.k = k, a.v = v, a.q_out = q_out;
  a.q_stride = q_stride, a.k_stride = k_stride, a.v_stride = v_stride, a.q_out_stride = q_out_stride;
  const bool win = windowed(ctx, layer);
  ctx->rope_captured |= capturing(static_cast<cudaStream_t>(stream));
  a.tab = win ? ctx->rope_tab_swa : ctx->rope_tab;
  if (ctx->qk_norm) {
    a.q_norm = ctx->qk_norm + (size_t)layer * ctx->hd;
    a.k_norm = ctx->qk_norm + ((size_t)c.n_layers + layer) * ctx->hd;
  }
  a.eps = ctx->rms_eps;
  a.rotary = ctx->rotary_dim;
  a.interleaved = ctx->rope_layout == L3P_ROPE_INTERLEAVED;
  // Tokens stream through shared memory where two of them fit a CTA's ring and a table row is whole 16-byte pieces (8B
  // heads, bf16, call after call: 64 tokens 2.7 us, 8192 tokens 39.3 us; by the kernel below 3.6 and 103 us).
  const int token_bytes = (c.n_heads + 2 * c.n_kv_heads) * ctx->hd * ctx->es + ctx->rotary_dim * 4 + 128;
  if (2 * token_bytes <= kRingBytes && ctx->rotary_dim % 4 == 0)
    return ctx->bf16 ? launch_rope_ring<__nv_bfloat16>(ctx, a, static_cast<cudaStream_t>(stream))
                     : launch_rope_ring<float>(ctx, a, static_cast<cudaStream_t>(stream));
  // few tokens: four rows a warp, so that all of them are in flight at once;
  // many: twelve, so that the cosines are read once for more rows
  const int rows = c.n_heads + 2 * c.n_kv_heads;
  a.rows_per_warp = (long long)ctx->hdr.n_tokens * rows <= 64LL * ctx->num_sms * 4 ? 4 : 12;
  const long long items = (long long)ctx->hdr.n_tokens * ((rows + a.rows_per_warp - 1) / a.rows_per_warp);
  const int grid = (int)((items + kPgKvWarps - 1) / kPgKvWarps);
  if (ctx->bf16) return launch_rope<__nv_bfloat16>(ctx, a, grid, static_cast<cudaStream_t>(stream));
  return launch_rope<float>(ctx, a, grid, static_cast<cudaStream_t>(stream));
}

L3P_API int l3p_paged_append_dev(l3p_paged_ctx* ctx, int layer, const void* k, long long k_stride, const void* v,
                                 long long v_stride, void* stream) {
  if (!ctx) return L3P_E_INVAL;
  if (int rc = check_call(ctx, layer)) return rc;
  if (ctx->hdr.n_tokens == 0) return L3P_OK;
  if (int rc = check_rows(ctx, "k", k, &k_stride, ctx->cfg.n_kv_heads)) return rc;
  if (int rc = check_rows(ctx, "v", v, &v_stride, ctx->cfg.n_kv_heads)) return rc;
  DeviceScope dev(ctx->cfg.device);
  PgKvArgs a = kv_args(ctx, layer);
  a.k = k, a.v = v;
  a.k_stride = k_stride, a.v_stride = v_stride;
  const int vecs = ctx->hd * ctx->es / 16;
  const long long n = (long long)ctx->hdr.n_tokens * 2 * ctx->cfg.n_kv_heads * vecs;
  const int grid = (int)std::min<long long>((n + 255) / 256, (long long)ctx->num_sms * 16);
  return launch(ctx, paged_append_kernel, dim3(grid), 256, 0, static_cast<cudaStream_t>(stream), 1, a, vecs, ctx->es);
}

// Checked here with the other row arguments; the kernels are launched by path.
L3P_API int l3p_paged_attn_dev(l3p_paged_ctx* ctx, int layer, const void* q, long long q_stride, void* out,
                               long long out_stride, void* stream) {
  if (!ctx) return L3P_E_INVAL;
  if (int rc = check_call(ctx, layer)) return rc;
  if (ctx->hdr.n_tokens == 0) return L3P_OK;
  if (int rc = check_rows(ctx, "q", q, &q_stride, ctx->cfg.n_heads)) return rc;
  if (int rc = check_rows(ctx, "out", out, &out_stride, ctx->cfg.n_heads)) return rc;
  DeviceScope dev(ctx->cfg.device);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const PgLists& l = ctx->hdr.lists[windowed(ctx, layer) ? 1 : 0];
  if (l.n_tc > 0)
    if (int rc = ctx->bf16 ? launch_tc(ctx, layer, q, q_stride, out, out_stride, s)
                           : launch_f32(ctx, layer, q, q_stride, out, out_stride, s))
      return rc;
  if (l.row_ctas > 0)
    if (int rc = launch_rows(ctx, layer, q, q_stride, out, out_stride, s)) return rc;
  return launch_merge(ctx, l, windowed(ctx, layer), out, out_stride, s);
}

// l3p_paged_rows.cu -- launcher of the row kernel (paged_rows.cuh).
#include <cuda_runtime.h>

#include <climits>

#include "paged_rows.cuh"

using namespace l3p;

namespace l3p_pg {

// Sequences with more query rows per KV head take the tensor-core kernels.  16 sequences of 3000 keys, 8B heads, layers in
// turn, by the row kernel and by the tensor-core kernel: bf16 16 rows 43.8 and 44.0 us (one such sequence 12.4 and 18.4), 32
// rows, blocks of 16, 77.6 and 45.2; fp32, whose tensor-core kernel first splits every key tile, 64 rows 397 and 472 us (34.1
// and 65.0), 128 rows 778 and 489.  fp32 with head_dim 256 has none: Q and O of a key tile of 128 would fill tensor memory.
int row_limit(const l3p_paged_ctx* ctx) {
  return ctx->bf16 ? 16 : ctx->hd == 256 ? INT_MAX : 64;
}

// Blocks of 8 rows whose Q and O fit a thread's registers.
int row_max_nt(const l3p_paged_ctx* ctx) {
  return !ctx->bf16 && ctx->hd == 256 ? 1 : 2;
}

int row_warps(const l3p_paged_ctx* ctx) {
  return ctx->hd == 256 ? PgRowCfg<float, 256>::kWarps : PgRowCfg<float, 128>::kWarps;
}

// Calls f with the kernel of the context's type and head size for blocks of nt * 8 rows.
template <typename F>
static int with_kernel(const l3p_paged_ctx* ctx, int nt, F f) {
  using B = __nv_bfloat16;
#define PG_ROW(T, HD, NT) f(paged_rows_kernel<T, HD, NT>, PgRowCfg<T, HD>::kWarps * 32, PgRowCfg<T, HD>::kSmem)
  if (ctx->bf16) {
    if (ctx->hd == 64) return nt == 1 ? PG_ROW(B, 64, 1) : PG_ROW(B, 64, 2);
    if (ctx->hd == 128) return nt == 1 ? PG_ROW(B, 128, 1) : PG_ROW(B, 128, 2);
    return nt == 1 ? PG_ROW(B, 256, 1) : PG_ROW(B, 256, 2);
  }
  if (ctx->hd == 64) return nt == 1 ? PG_ROW(float, 64, 1) : PG_ROW(float, 64, 2);
  if (ctx->hd == 128) return nt == 1 ? PG_ROW(float, 128, 1) : PG_ROW(float, 128, 2);
  return PG_ROW(float, 256, 1);
#undef PG_ROW
}

int init_rows(l3p_paged_ctx* ctx) {
  const int max_nt = row_max_nt(ctx);
  for (int nt = 1; nt <= max_nt; nt *= 2) {
    const int rc = with_kernel(ctx, nt, [&](auto kernel, int, int smem) {
      PG_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
      return (int)L3P_OK;
    });
    if (rc) return rc;
  }
  const size_t slots = 2 * (size_t)ctx->num_sms + 2, rows = slots * 8 * max_nt;
  if (cudaMalloc(&ctx->ws_o, rows * ctx->hd * sizeof(float)) != cudaSuccess ||
      cudaMalloc(&ctx->ws_ml, rows * 2 * sizeof(float)) != cudaSuccess ||
      cudaMalloc(&ctx->tickets, (size_t)kPgMaxCtas * sizeof(unsigned)) != cudaSuccess) {
    cudaGetLastError();
    return fail(ctx, L3P_E_NOMEM, "the split workspace does not fit on the device");
  }
  PG_CUDA(ctx, cudaMemset(ctx->tickets, 0, (size_t)kPgMaxCtas * sizeof(unsigned)));
  return L3P_OK;
}

int launch_rows(l3p_paged_ctx* ctx, int layer, const void* q, long long qs, void* out, long long os, cudaStream_t s) {
  const bool win = windowed(ctx, layer);
  const PgLists& l = ctx->hdr.lists[win ? 1 : 0];
  PgRowArgs a{};
  a.batch = ctx->batch;
  a.q = q;
  a.out = out;
  a.q_stride = qs;
  a.out_stride = os;
  a.storage = static_cast<char*>(ctx->storage) + (size_t)layer * 2 * ctx->cfg.n_kv_heads * ctx->block_bytes;
  a.page_elems = (long long)(ctx->page_bytes / ctx->es);
  a.v_off = (long long)(ctx->block_bytes / ctx->es) * ctx->cfg.n_kv_heads;
  a.shift = ctx->shift;
  a.G = ctx->G;
  a.win = win ? 1 : 0;
  a.window = ctx->cfg.swa_window;
  a.lim = limits(ctx, l);
  a.late = l.n_tc > 0;
  a.scale_log2 = ctx->scale * kLog2e;
  a.ws_o = ctx->ws_o;
  a.ws_ml = ctx->ws_ml;
  a.tickets = ctx->tickets;
  a.err = ctx->err_dev;
  // a captured launch may meet a batch that uses more CTAs, of which plan_rows makes no more than SMs
  const int grid = capturing(s) ? ctx->num_sms : l.row_ctas;
  return with_kernel(ctx, ctx->hdr.row_nt,
                     [&](auto kernel, int threads, int smem) { return launch(ctx, kernel, dim3(grid), threads, smem, s, 1, a); });
}

}  // namespace l3p_pg

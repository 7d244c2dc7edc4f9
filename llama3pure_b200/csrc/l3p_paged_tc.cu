// l3p_paged_tc.cu -- launcher of the bf16 tensor-core kernel (paged_tc.cuh).
#include <cuda_runtime.h>

#include <cstring>

#include "paged_tc.cuh"

using namespace l3p;

namespace l3p_pg {

int tc_tile(const l3p_paged_ctx* ctx) { return ctx->hd == 256 ? 64 : 128; }
int tc_rows(const l3p_paged_ctx* ctx) { return ctx->hd == 256 ? 128 : 256; }

template <typename F>
static int with_kernel(const l3p_paged_ctx* ctx, F f) {
  if (ctx->hd == 64) return f(paged_tc_kernel<64>, PgTcCfg<64>::kThreads, PgTcCfg<64>::kSmem);
  if (ctx->hd == 128) return f(paged_tc_kernel<128>, PgTcCfg<128>::kThreads, PgTcCfg<128>::kSmem);
  return f(paged_tc_kernel<256>, PgTcCfg<256>::kThreads, PgTcCfg<256>::kSmem);
}

int init_tc(l3p_paged_ctx* ctx) {
  const auto& c = ctx->cfg;
  // the storage as a matrix of rows: boxes of a page's (at most a tile's) keys by 64 columns
  static_assert(sizeof(CUtensorMap) == sizeof(ctx->tmap), "tensor map");
  void* fn = nullptr;
  cudaDriverEntryPointQueryResult found;
  PG_CUDA(ctx, cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found));
  if (found != cudaDriverEntryPointSuccess || !fn) return fail(ctx, L3P_E_CUDA, "the driver has no cuTensorMapEncodeTiled");
  const cuuint64_t rows = (cuuint64_t)c.n_pages * c.n_layers * 2 * c.n_kv_heads * c.page_size;
  const cuuint64_t dims[2] = {(cuuint64_t)c.head_dim, rows};
  const cuuint64_t strides[1] = {(cuuint64_t)c.head_dim * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)(c.page_size < tc_tile(ctx) ? c.page_size : tc_tile(ctx))};
  const cuuint32_t ones[2] = {1, 1};
  const CUresult r = reinterpret_cast<decltype(&cuTensorMapEncodeTiled)>(fn)(
      reinterpret_cast<CUtensorMap*>(ctx->tmap), CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, ctx->storage, dims, strides, box, ones,
      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(ctx, L3P_E_CUDA, "cuTensorMapEncodeTiled: %d", (int)r);
  if (int rc = with_kernel(ctx, [&](auto kernel, int, int smem) {
        PG_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        return (int)L3P_OK;
      }))
    return rc;
  // plan_tc makes at most 2 num_sms parts of the units that it splits
  const size_t rows_ws = 2 * (size_t)ctx->num_sms * tc_rows(ctx);
  if (cudaMalloc(&ctx->tc_o, rows_ws * ctx->hd * sizeof(float)) != cudaSuccess ||
      cudaMalloc(&ctx->tc_ml, rows_ws * 2 * sizeof(float)) != cudaSuccess) {
    cudaGetLastError();
    return fail(ctx, L3P_E_NOMEM, "the split workspace does not fit on the device");
  }
  return L3P_OK;
}

int launch_tc(l3p_paged_ctx* ctx, int layer, const void* q, long long qs, void* out, long long os, cudaStream_t s) {
  const auto& c = ctx->cfg;
  const bool win = windowed(ctx, layer);
  const PgLists& l = ctx->hdr.lists[win ? 1 : 0];
  PgTcArgs a{};
  a.batch = ctx->batch;
  a.q = q;
  a.out = out;
  a.q_stride = qs;
  a.out_stride = os;
  a.storage = static_cast<const __nv_bfloat16*>(ctx->storage);
  a.page_elems = (long long)(ctx->page_bytes / ctx->es);
  a.row_k = layer * 2 * c.n_kv_heads * c.page_size;
  a.page_rows = c.n_layers * 2 * c.n_kv_heads * c.page_size;
  a.n_kv = c.n_kv_heads;
  a.shift = ctx->shift;
  a.G = ctx->G;
  a.win = win ? 1 : 0;
  a.window = c.swa_window;
  a.lim = limits(ctx, l);
  a.scale_log2 = ctx->scale * kLog2e;
  a.ws_o = ctx->tc_o;
  a.ws_ml = ctx->tc_ml;
  a.err = ctx->err_dev;
  CUtensorMap map;
  memcpy(&map, ctx->tmap, sizeof map);
  return with_kernel(ctx, [&](auto kernel, int threads, int smem) {
    return launch(ctx, kernel, dim3(l.n_tc), threads, smem, s, 1, a, map);
  });
}

template <typename T, int HD>
static int merge(l3p_paged_ctx* ctx, const PgLists& l, bool win, int rows, void* out, long long os, cudaStream_t s) {
  return launch(ctx, paged_merge_kernel<T, HD>, dim3(l.n_merge, rows / 8), 256, 0, s, 1, (const int*)ctx->batch, win ? 1 : 0,
                limits(ctx, l), rows, (const float*)ctx->tc_o, (const float*)ctx->tc_ml, static_cast<T*>(out), os, ctx->G);
}

int launch_merge(l3p_paged_ctx* ctx, const PgLists& l, bool win, void* out, long long os, cudaStream_t s) {
  const int rows = ctx->bf16 ? tc_rows(ctx) : f32_rows(ctx);
  if (l.n_merge == 0) return L3P_OK;
  if (ctx->bf16)
    return ctx->hd == 64    ? merge<__nv_bfloat16, 64>(ctx, l, win, rows, out, os, s)
           : ctx->hd == 128 ? merge<__nv_bfloat16, 128>(ctx, l, win, rows, out, os, s)
                            : merge<__nv_bfloat16, 256>(ctx, l, win, rows, out, os, s);
  return ctx->hd == 64 ? merge<float, 64>(ctx, l, win, rows, out, os, s) : merge<float, 128>(ctx, l, win, rows, out, os, s);
}

}  // namespace l3p_pg

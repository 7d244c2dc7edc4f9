// l3p_paged_f32.cu -- launcher of the fp32 tensor-core kernels (paged_f32.cuh).
#include <cuda_runtime.h>

#include <algorithm>

#include "paged_f32.cuh"

using namespace l3p;

namespace l3p_pg {

// Images of more than this are made for some KV heads at a time, at least one: its images are twice its K and V.
static constexpr size_t kImageBytes = 1ull << 30;

int f32_rows(const l3p_paged_ctx* ctx) { return ctx->hd == 64 ? 128 : 256; }

int init_f32(l3p_paged_ctx* ctx) {
  if (ctx->hd == 256) return L3P_OK;  // rows of 256 values take the row kernel
  if (ctx->hd == 64)
    PG_CUDA(ctx, cudaFuncSetAttribute(paged_f32_kernel<1, 64>, cudaFuncAttributeMaxDynamicSharedMemorySize, PgF32Cfg<1, 64>::kSmem));
  else
    PG_CUDA(ctx, cudaFuncSetAttribute(paged_f32_kernel<2, 128>, cudaFuncAttributeMaxDynamicSharedMemorySize, PgF32Cfg<2, 128>::kSmem));
  const size_t rows = 2 * (size_t)ctx->num_sms * f32_rows(ctx);  // as in init_tc
  if (cudaMalloc(&ctx->tc_o, rows * ctx->hd * sizeof(float)) != cudaSuccess ||
      cudaMalloc(&ctx->tc_ml, rows * 2 * sizeof(float)) != cudaSuccess) {
    cudaGetLastError();
    return fail(ctx, L3P_E_NOMEM, "the split workspace does not fit on the device");
  }
  return L3P_OK;
}

static size_t tile_floats(const l3p_paged_ctx* ctx) { return ctx->hd == 64 ? PfGeom<64>::kTileFloats : PfGeom<128>::kTileFloats; }

// KV heads whose images of n_prep tiles are made at a time.
static int image_heads(const l3p_paged_ctx* ctx, int n_prep) {
  const size_t fit = std::max<size_t>(1, kImageBytes / (tile_floats(ctx) * sizeof(float) * n_prep));
  return (int)std::min<size_t>(fit, ctx->cfg.n_kv_heads);
}

// The image buffer for a batch, as part of begin: attention then has nothing to allocate, in a capture or out of it.  It grows
// by half at least, since a prompt fed in chunks needs a little more at every step.
int prepare_f32(l3p_paged_ctx* ctx, const PgHeader& h) {
  size_t tiles = 0;  // of all heads at a time
  for (const PgLists& l : h.lists)
    if (l.n_prep > 0) tiles = std::max(tiles, (size_t)l.n_prep * image_heads(ctx, l.n_prep));
  if (tiles <= ctx->img_tiles) return L3P_OK;
  const size_t tile = tile_floats(ctx) * sizeof(float);
  ctx->retired.reserve(ctx->retired.size() + 2);
  float* img = nullptr;
  int* flags = nullptr;
  size_t want = std::max(tiles, ctx->img_tiles + ctx->img_tiles / 2);
  auto get = [&] {
    if (cudaMalloc(&img, want * tile) == cudaSuccess && cudaMalloc(&flags, want * 4 * sizeof(int)) == cudaSuccess) return true;
    cudaGetLastError();
    cudaFree(img);
    img = nullptr;
    return false;
  };
  if (!get() && (want == tiles || (want = tiles, !get())))
    return fail(ctx, L3P_E_NOMEM, "the fp32 chunks' workspace of %zu bytes does not fit on the device", want * tile);
  if (ctx->img) PG_CUDA(ctx, cudaDeviceSynchronize());  // earlier calls' kernels read the old ones
  retire(ctx, ctx->img, ctx->img_captured);
  retire(ctx, ctx->v_flags, ctx->img_captured);
  ctx->img_captured = false;
  ctx->img = img;
  ctx->v_flags = flags;
  ctx->img_tiles = want;
  return L3P_OK;
}

template <int CG, int HD>
static int chunks(l3p_paged_ctx* ctx, PgF32Args a, const PgLists& l, cudaStream_t s) {
  const int n_kv = ctx->cfg.n_kv_heads, group = image_heads(ctx, l.n_prep);
  ctx->img_captured |= capturing(s);
  a.img = ctx->img;
  a.flags = ctx->v_flags;
  for (int h = 0; h < n_kv; h += group) {
    a.kvh0 = h;
    a.n_kv = n_kv;
    a.n_kvh = std::min(group, n_kv - h);
    if (int rc = launch(ctx, paged_prep_kernel<CG, HD>, dim3(l.n_prep, a.n_kvh, 4), 256, 0, s, 1, a)) return rc;
    if (int rc = launch(ctx, paged_f32_kernel<CG, HD>, dim3(l.n_tc * CG), 512, PgF32Cfg<CG, HD>::kSmem, s, CG, a)) return rc;
  }
  return L3P_OK;
}

int launch_f32(l3p_paged_ctx* ctx, int layer, const void* q, long long qs, void* out, long long os, cudaStream_t s) {
  const bool win = windowed(ctx, layer);
  const PgLists& l = ctx->hdr.lists[win ? 1 : 0];
  PgF32Args a{};
  a.batch = ctx->batch;
  a.q = static_cast<const float*>(q);
  a.out = static_cast<float*>(out);
  a.q_stride = qs;
  a.out_stride = os;
  a.storage = reinterpret_cast<const float*>(static_cast<char*>(ctx->storage) + (size_t)layer * 2 * ctx->cfg.n_kv_heads * ctx->block_bytes);
  a.page_elems = (long long)(ctx->page_bytes / ctx->es);
  a.v_off = (long long)(ctx->block_bytes / ctx->es) * ctx->cfg.n_kv_heads;
  a.shift = ctx->shift;
  a.G = ctx->G;
  a.win = win ? 1 : 0;
  a.window = ctx->cfg.swa_window;
  a.lim = limits(ctx, l);
  a.scale_log2 = ctx->scale * kLog2e;
  a.ws_o = ctx->tc_o;
  a.ws_ml = ctx->tc_ml;
  a.err = ctx->err_dev;
  return ctx->hd == 64 ? chunks<1, 64>(ctx, a, l, s) : chunks<2, 128>(ctx, a, l, s);
}

}  // namespace l3p_pg

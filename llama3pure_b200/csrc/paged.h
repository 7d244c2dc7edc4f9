// paged.h -- the paged cache's context and the batch description that its
// kernels read (l3p_paged.cu, l3p_paged_kv.cu, l3p_paged_rows.cu,
// l3p_paged_tc.cu, l3p_paged_f32.cu).  Private: not part of the C ABI.
#pragma once
#include <cuda_runtime.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <vector>

#include "llama3pure_paged.h"

#define L3P_API extern "C" __attribute__((visibility("default")))

namespace l3p {

// ---- the batch on the device: one block of 32-bit words ----------------------
// [0, kPgHdrWords) header, then the arrays at the word offsets that the header
// names.  Everything that depends on the batch is read from here, so that a
// captured launch serves the batch that is current when it is replayed.
constexpr int kPgMaxCtas = 160;   // CTAs of the row kernel at most
constexpr int kPgTile = 16;       // keys of a warp tile of the row kernel

// Lists of one kind of layer: [0] layers that attend to everything, [1] sliding-window layers.
struct PgLists {
  int row_ctas;    // CTAs of the row kernel that have segments (0: no sequence takes that path)
  int row_first;   // word offset: int[row_ctas + 1], first segment of each
  int row_segs;    // word offset: PgSeg[]
  int n_tc;        // parts of the tensor-core kernels (0: none)
  int tc_parts;    // word offset: PgPart[]
  int n_merge;     // units that are cut into parts
  int merges;      // word offset: PgPart[], one for each of them
  int n_prep;      // fp32 pools: key tiles to split
  int prep;        // word offset: PgPrep[]
};
struct PgHeader {
  int n_tokens, n_seqs, row_nt, tok;  // tok: word offset of int2[n_tokens] (storage row, position)
  int tbl;                            // word offset: the sequences' page tables, one after the other
  int pad[3];
  PgLists lists[2];
};
constexpr int kPgHdrWords = 64;
static_assert(sizeof(PgHeader) <= kPgHdrWords * 4, "batch header");

// Keys [tile0*16, tile1*16) of the rows r0 .. r0+n_rows-1 of one sequence and
// KV head.  Row r is query head kvh*G + r % G of new token r / G.
struct __align__(16) PgSeg {
  int tbl;             // the sequence's table starts here (index into the tables)
  int key_lo, key_hi;  // keys that any of the rows attends to
  int tile0, tile1;
  int q_row0, pos0;    // batch row and position of the sequence's first new token
  int r0, n_rows, kvh;
  int part, n_parts;   // split of the rows' key range; the merge's ticket and slots go by
  int cta0;            //   the CTA that holds part 0
  int pad[3];
};
static_assert(sizeof(PgSeg) == 64, "segment");

// Key tiles [tile0, tile1) of 128 (64 for head_dim 256) keys for the rows
// r0 .. r0+n_rows-1 on the tensor cores.
struct __align__(16) PgPart {
  int tbl, key_hi, tile0, tile1;
  int q_row0, pos0, r0, n_rows;
  int kvh, part, n_parts, slot;
  int img, pad[3];  // slot: workspace of part 0; img: image of tile 0 (fp32 pools)
};
static_assert(sizeof(PgPart) == 64, "part");

// What a call's launches were made for: a batch that they meet when they are
// replayed must not exceed it (fits), else nothing is written and the error word
// is set.  All launches of a call decide alike.
struct PgLimits {
  int n_tokens, n_tc, n_merge, n_prep, with_tc;
  int with_rows;  // blocks of 8 rows that the row kernel's instance takes; 0: no row kernel
};
#ifdef __CUDACC__
__device__ __forceinline__ bool pg_fits(const PgHeader* h, const PgLists& l, const PgLimits& m) {
  return h->n_tokens <= m.n_tokens && l.n_tc <= m.n_tc && l.n_merge <= m.n_merge && l.n_prep <= m.n_prep &&
         (l.row_ctas != 0 ? h->row_nt : 0) == m.with_rows && (l.n_tc != 0) == (m.with_tc != 0);
}
#endif

struct PgPrep {
  int tbl, key0, key_hi, img;  // keys [key0, key0+128) below key_hi, to image tile img
};

}  // namespace l3p

struct l3p_paged_ctx {
  l3p_paged_config cfg{};
  int hd = 0, G = 1, es = 4, shift = 4;  // head size, heads per KV head, bytes of a value, log2(page_size)
  bool bf16 = false, swa = false;
  float scale = 1.f;
  int num_sms = 148;
  void* storage = nullptr;
  size_t page_bytes = 0;       // one page: all layers, K and V, all heads
  size_t block_bytes = 0;      // one head's rows of one layer's K or V in a page
  int* batch = nullptr;        // device batch block
  size_t batch_words = 0;
  int* jobs = nullptr;         // device page-copy jobs (int4 each)
  size_t jobs_cap = 0;
  // pinned staging of uploads, used in turn; an event says when a slot's copy is done
  static constexpr int kSlots = 4;
  struct Slot {
    int* host = nullptr;
    size_t words = 0;
    cudaEvent_t done = nullptr;
    bool used = false;
  } slots[kSlots];
  unsigned slot_next = 0;

  // books
  struct Seq {
    bool live = false;
    int len = 0;
    std::vector<int> pages;
  };
  std::vector<Seq> seqs;
  std::vector<int> refs;       // holders of each page
  std::vector<int> fill;       // rows of each page that any holder has used since it was given out
  std::vector<int> free_heap;  // free pages, the lowest index on top

  // current batch
  bool batch_valid = false;
  l3p::PgHeader hdr{};
  struct Plan {
    std::vector<int> first;
    std::vector<l3p::PgSeg> segs;
    std::vector<l3p::PgPart> parts, merges;
    std::vector<l3p::PgPrep> prep;
  } plan[2];
  std::vector<l3p::PgSeg> row_units;
  std::vector<l3p::PgPart> tc_units;
  int max_pos_in_batch = 0;  // one more than the highest position of a new token

  // split workspace: partial rows, (m, l) pairs, tickets (0 between launches)
  float* ws_o = nullptr;
  float* ws_ml = nullptr;
  unsigned* tickets = nullptr;
  float* tc_o = nullptr;
  float* tc_ml = nullptr;
  // fp32 pools on the tensor cores: K/V tile images, flags of tiles with values that are not finite (l3p_paged_f32.cu)
  float* img = nullptr;
  int* v_flags = nullptr;
  size_t img_tiles = 0;
  alignas(64) unsigned char tmap[128] = {};  // bf16 pools: the storage as rows of head_dim values (CUtensorMap)

  float2* rope_tab = nullptr;      // (cos, sin) [max_pos][rotary_dim/2]
  float2* rope_tab_swa = nullptr;  // sliding-window layers (the same array without them)
  float* qk_norm = nullptr;        // [2][n_layers][hd]
  int rope_max = 0, rope_layout = 0, rotary_dim = 0;
  float rms_eps = 1e-5f;

  // buffers that captured launches name: kept until the context ends when they are replaced
  bool img_captured = false, rope_captured = false;
  std::vector<void*> retired;

  int* err_host = nullptr;
  int* err_dev = nullptr;
  long long launches = 0;
  char last_error[512] = "";  // written without an allocation: a refusal may be for want of memory
};

namespace l3p_pg {

// Lets a replaced device buffer go: at once, or with the context when a captured launch names it.
inline void retire(l3p_paged_ctx* ctx, void* p, bool captured) {
  if (!p) return;
  if (captured)
    ctx->retired.push_back(p);
  else
    cudaFree(p);
}

inline int fail(l3p_paged_ctx* ctx, int code, const char* fmt, ...) noexcept {
  if (ctx) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(ctx->last_error, sizeof ctx->last_error, fmt, ap);
    va_end(ap);
  }
  return code;
}

#define PG_CUDA(ctx, call)                                                                                      \
  do {                                                                                                          \
    cudaError_t e_ = (call);                                                                                    \
    if (e_ != cudaSuccess)                                                                                      \
      return l3p_pg::fail((ctx), L3P_E_CUDA, "%s: %s (%s:%d)", #call, cudaGetErrorString(e_), __FILE__, __LINE__); \
  } while (0)

// Makes the context's device current for an entry point and restores the caller's.
struct DeviceScope {
  int prev = -1;
  bool changed = false;
  explicit DeviceScope(int dev) {
    if (cudaGetDevice(&prev) == cudaSuccess && prev != dev) changed = cudaSetDevice(dev) == cudaSuccess;
  }
  ~DeviceScope() {
    if (changed) cudaSetDevice(prev);
  }
};

// Whether `s` captures; of the null stream: or a stream that work on it would wait for.
inline bool capturing(cudaStream_t s) {
  cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
  const cudaError_t e = cudaStreamIsCapturing(s, &st);
  if (e != cudaSuccess) cudaGetLastError();
  return e == cudaErrorStreamCaptureImplicit || (e == cudaSuccess && st != cudaStreamCaptureStatusNone);
}

inline bool windowed(const l3p_paged_ctx* ctx, int layer) {
  return ctx->swa && layer % ctx->cfg.swa_pattern < ctx->cfg.swa_pattern - 1;
}

// Launches a kernel that may start while the one before it on the stream ends:
// ahead of its griddep_wait every such kernel reads only the batch description,
// which a copy brought.  (The row kernel beside a tensor-core kernel of the same
// call starts behind that kernel's own wait, and waits for it at its end.)
template <typename... P, typename... A>
int launch(l3p_paged_ctx* ctx, void (*kernel)(P...), dim3 grid, int threads, int smem, cudaStream_t s, int cluster, A... args) {
  cudaLaunchConfig_t lc{};
  lc.gridDim = grid;
  lc.blockDim = dim3(threads, 1, 1);
  lc.dynamicSmemBytes = smem;
  lc.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  lc.attrs = attr;
  lc.numAttrs = cluster > 1 ? 2 : 1;
  PG_CUDA(ctx, cudaLaunchKernelEx(&lc, kernel, args...));
  ++ctx->launches;
  return L3P_OK;
}

inline l3p::PgLimits limits(const l3p_paged_ctx* ctx, const l3p::PgLists& l) {
  return {ctx->hdr.n_tokens, l.n_tc, l.n_merge, l.n_prep, l.n_tc > 0, l.row_ctas > 0 ? ctx->hdr.row_nt : 0};
}

// Rows per KV head up to which a sequence takes the row kernel, and the key
// tile of the tensor-core kernel (l3p_paged_rows.cu, l3p_paged_tc.cu).
int row_limit(const l3p_paged_ctx* ctx);
int row_max_nt(const l3p_paged_ctx* ctx);  // blocks of 8 rows that one CTA takes at most
int row_warps(const l3p_paged_ctx* ctx);
int tc_tile(const l3p_paged_ctx* ctx);
int tc_rows(const l3p_paged_ctx* ctx);  // rows of a part, bf16 pools
int f32_rows(const l3p_paged_ctx* ctx);  // rows of a part, fp32 pools

// Set-up of the kernels at create: shared-memory attributes, tensor map, workspaces.
int init_kv(l3p_paged_ctx* ctx);
int init_rows(l3p_paged_ctx* ctx);
int init_tc(l3p_paged_ctx* ctx);
int init_f32(l3p_paged_ctx* ctx);

// Part of begin, before the books move: the workspace of a planned batch's fp32 chunks.
int prepare_f32(l3p_paged_ctx* ctx, const l3p::PgHeader& h);

int launch_rows(l3p_paged_ctx* ctx, int layer, const void* q, long long qs, void* out, long long os, cudaStream_t s);
int launch_tc(l3p_paged_ctx* ctx, int layer, const void* q, long long qs, void* out, long long os, cudaStream_t s);
int launch_f32(l3p_paged_ctx* ctx, int layer, const void* q, long long qs, void* out, long long os, cudaStream_t s);
// Joins the parts of the split units of the tensor-core kernels (l3p_paged_tc.cu).
int launch_merge(l3p_paged_ctx* ctx, const l3p::PgLists& l, bool win, void* out, long long os, cudaStream_t s);
// Copies rows of pages: jobs (source page, destination page, rows, 0) in device memory.
int launch_page_copy(l3p_paged_ctx* ctx, const int* jobs, int n_jobs, cudaStream_t s);

}  // namespace l3p_pg

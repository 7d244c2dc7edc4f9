// paged_books.cpp -- the paged cache's books without a GPU: l3p_paged.cu linked
// with a CUDA runtime of this file's own, whose device memory is host memory.
// Every host allocation (operator new, pinned, device) can be made to fail.
//
//     paged_books <test> [rest]      exits 0, or prints what is wrong and exits 1
#include <cuda_runtime_api.h>

#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <new>
#include <string>
#include <vector>

#include "paged.h"

// ---- allocations that fail on demand ------------------------------------------
static long g_fail_in = -1;  // the allocation that fails, counted down; -1: none, -2: it has failed
static bool g_fail_rest = false;  // and every one after it
static bool fails() {
  if (g_fail_in < 0) return g_fail_rest && g_fail_in == -2;
  if (g_fail_in-- > 0) return false;
  g_fail_in = -2;
  return true;
}
static bool g_watch = false;  // only the calls under test
void* operator new(size_t n) {
  if (g_watch && fails()) throw std::bad_alloc();
  if (void* p = malloc(n ? n : 1)) return p;
  throw std::bad_alloc();
}
void operator delete(void* p) noexcept { free(p); }
void operator delete(void* p, size_t) noexcept { free(p); }

// ---- the CUDA runtime that l3p_paged.cu calls -----------------------------------
static cudaError_t give(void** p, size_t n) {
  if (g_watch && fails()) return cudaErrorMemoryAllocation;
  *p = calloc(n ? n : 1, 1);
  return *p ? cudaSuccess : cudaErrorMemoryAllocation;
}
static bool g_capturing = false;  // the stream
static bool g_implicit = false;   // another stream, which work on the null stream would wait for
extern "C" {
cudaError_t cudaGetDevice(int* d) { return *d = 0, cudaSuccess; }
cudaError_t cudaSetDevice(int) { return cudaSuccess; }
cudaError_t cudaGetDeviceProperties_v2(cudaDeviceProp* p, int) {
  memset(p, 0, sizeof *p);
  p->multiProcessorCount = 148;
  return cudaSuccess;
}
cudaError_t cudaMalloc(void** p, size_t n) { return give(p, n); }
cudaError_t cudaFree(void* p) { return free(p), cudaSuccess; }
cudaError_t cudaHostAlloc(void** p, size_t n, unsigned) { return give(p, n); }
cudaError_t cudaFreeHost(void* p) { return free(p), cudaSuccess; }
cudaError_t cudaHostGetDevicePointer(void** d, void* h, unsigned) { return *d = h, cudaSuccess; }
cudaError_t cudaMemset(void* p, int v, size_t n) { return memset(p, v, n), cudaSuccess; }
cudaError_t cudaMemcpyAsync(void* d, const void* s, size_t n, cudaMemcpyKind, cudaStream_t) {
  if (g_capturing || g_implicit) return cudaErrorStreamCaptureImplicit;
  return memcpy(d, s, n), cudaSuccess;
}
cudaError_t cudaEventCreateWithFlags(cudaEvent_t* e, unsigned) { return give(reinterpret_cast<void**>(e), 1); }
cudaError_t cudaEventRecord(cudaEvent_t, cudaStream_t) { return cudaSuccess; }
cudaError_t cudaEventSynchronize(cudaEvent_t) { return cudaSuccess; }
cudaError_t cudaEventDestroy(cudaEvent_t e) { return free(e), cudaSuccess; }
cudaError_t cudaDeviceSynchronize() { return cudaSuccess; }
cudaError_t cudaStreamSynchronize(cudaStream_t) { return cudaSuccess; }
cudaError_t cudaStreamIsCapturing(cudaStream_t, cudaStreamCaptureStatus* s) {
  *s = g_capturing ? cudaStreamCaptureStatusActive : cudaStreamCaptureStatusNone;
  return g_implicit ? cudaErrorStreamCaptureImplicit : cudaSuccess;
}
cudaError_t cudaGetLastError() { return cudaSuccess; }
const char* cudaGetErrorString(cudaError_t) { return "planted"; }
// what nvcc's registration of device code calls
void** __cudaRegisterFatBinary(void*) { return nullptr; }
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
}

// ---- the parts of the library that launch kernels --------------------------------
namespace l3p_pg {
int init_kv(l3p_paged_ctx*) { return L3P_OK; }
int init_rows(l3p_paged_ctx*) { return L3P_OK; }
int init_tc(l3p_paged_ctx*) { return L3P_OK; }
int init_f32(l3p_paged_ctx*) { return L3P_OK; }
int prepare_f32(l3p_paged_ctx* ctx, const l3p::PgHeader&) {
  return g_watch && fails() ? fail(ctx, L3P_E_NOMEM, "planted") : (int)L3P_OK;
}
int row_limit(const l3p_paged_ctx* ctx) { return ctx->bf16 ? 16 : 64; }
int row_max_nt(const l3p_paged_ctx*) { return 2; }
int row_warps(const l3p_paged_ctx*) { return 8; }
int tc_tile(const l3p_paged_ctx*) { return 128; }
int tc_rows(const l3p_paged_ctx*) { return 256; }
int f32_rows(const l3p_paged_ctx*) { return 256; }
int launch_page_copy(l3p_paged_ctx* ctx, const int* jobs, int n, cudaStream_t) {
  char* base = static_cast<char*>(ctx->storage);
  for (int i = 0; i < n; ++i, jobs += 4)
    for (size_t b = 0; b < ctx->page_bytes; b += ctx->block_bytes)
      memcpy(base + jobs[1] * ctx->page_bytes + b, base + jobs[0] * ctx->page_bytes + b, (size_t)jobs[2] * ctx->hd * ctx->es);
  return L3P_OK;
}
}  // namespace l3p_pg

// ---- tests ---------------------------------------------------------------------------
static int g_bad = 0;
#define EXPECT(x)                                                \
  do {                                                           \
    if (!(x)) {                                                  \
      printf("%s:%d: %s\n", __FILE__, __LINE__, #x);             \
      if (++g_bad > 10) exit(1);                                 \
    }                                                            \
  } while (0)

constexpr int kPages = 400, kSeqs = 24;

static l3p_paged_ctx* make(int dtype) {
  l3p_paged_config c{};
  c.n_layers = 1, c.n_heads = 8, c.n_kv_heads = 2, c.head_dim = 64, c.page_size = 16, c.n_pages = kPages;
  c.max_seqs = kSeqs, c.max_tokens = 4000, c.dtype = dtype;
  l3p_paged_ctx* ctx = nullptr;
  EXPECT(l3p_paged_create(&c, &ctx) == L3P_OK && ctx);
  return ctx;
}

// All that a caller sees of the books: live sequences, lengths, tables, free pages, the batch, and all rows.
struct Seen {
  std::vector<int> words;
  std::vector<char> rows;
  bool operator==(const Seen& o) const { return words == o.words && rows == o.rows; }
};
static Seen look(l3p_paged_ctx* ctx) {
  Seen s;
  for (int i = 0; i < kSeqs; ++i) {
    int n = -1, table[kPages], need = 0;
    s.words.push_back(l3p_paged_seq_length(ctx, i, &n));
    s.words.push_back(n);
    if (n < 0) continue;
    EXPECT(l3p_paged_tables(ctx, 1, &i, kPages, table, &need) == L3P_OK);
    s.words.insert(s.words.end(), table, table + need);
  }
  int n_free = 0;
  l3p_paged_free_pages(ctx, &n_free);
  s.words.push_back(n_free);
  s.words.push_back(ctx->batch_valid);
  s.words.push_back(ctx->hdr.n_tokens);
  s.words.insert(s.words.end(), ctx->refs.begin(), ctx->refs.end());
  s.words.insert(s.words.end(), ctx->fill.begin(), ctx->fill.end());
  const char* p = static_cast<char*>(ctx->storage);
  s.rows.assign(p, p + ctx->page_bytes * kPages);
  return s;
}

// Sequences of 37, 20 and 700 positions; two children of the first, so that its last page is shared.
static void fill(l3p_paged_ctx* ctx, int* ids) {
  for (int i = 0; i < 3; ++i) EXPECT(l3p_paged_seq_new(ctx, ids + i) == L3P_OK);
  const int n[3] = {37, 20, 700};
  EXPECT(l3p_paged_begin(ctx, 3, ids, n, nullptr) == L3P_OK);
  for (size_t i = 0; i < ctx->page_bytes * kPages / 4; ++i) static_cast<int*>(ctx->storage)[i] = (int)i;
  EXPECT(l3p_paged_seq_fork(ctx, ids[0], -1, 2, ids + 3) == L3P_OK);
  const int one[1] = {1};
  EXPECT(l3p_paged_begin(ctx, 1, ids + 1, one, nullptr) == L3P_OK);
}

// Fails every allocation of `call` in turn (and with g_fail_rest all behind it too): the call returns L3P_E_NOMEM and nothing has
// changed, or it does without the memory.  A further call has the outcome that it has where nothing failed.
template <typename F>
static void fail_everywhere(const char* name, int dtype, F call, bool holes = false) {
  int ids[8];
  auto set_up = [&](l3p_paged_ctx* ctx) {
    fill(ctx, ids);
    if (holes) EXPECT(l3p_paged_seq_free(ctx, 1, ids + 1) == L3P_OK);
    const int none[1] = {0};  // there is a batch
    EXPECT(l3p_paged_begin(ctx, 1, ids, none, nullptr) == L3P_OK);
  };
  l3p_paged_ctx* ctx = make(dtype);
  set_up(ctx);
  const Seen before = look(ctx);
  EXPECT(call(ctx, ids) == L3P_OK);
  const Seen want = look(ctx);
  l3p_paged_destroy(ctx);
  int refused = 0;
  for (long at = 0, reached = 1; reached; ++at) {
    ctx = make(dtype);
    set_up(ctx);
    g_watch = true, g_fail_in = at;
    int rc = call(ctx, ids);
    g_watch = false;
    reached = g_fail_in < 0;
    g_fail_in = -1;
    if (rc != L3P_OK) {
      ++refused;
      EXPECT(reached && rc == L3P_E_NOMEM && l3p_paged_last_error(ctx)[0] != 0);
      const bool same = look(ctx) == before;
      if (!same) printf("%s: allocation %ld failed and the books changed\n", name, at);
      EXPECT(same);
      EXPECT(call(ctx, ids) == L3P_OK);
    }
    EXPECT(look(ctx) == want);
    l3p_paged_destroy(ctx);
  }
  EXPECT(refused > 0);
}

static int begin_call(l3p_paged_ctx* ctx, const int* ids) {
  const int n_new[5] = {1, 1400, 40, 2, 1};  // shared pages copied, a description that outgrows the first pinned slots
  return l3p_paged_begin(ctx, 5, ids, n_new, nullptr);
}
static int copy_call(l3p_paged_ctx* ctx, const int* ids) {
  int children[3];
  return l3p_paged_seq_copy(ctx, 3, ids, children, nullptr);
}
static int fork_call(l3p_paged_ctx* ctx, const int* ids) {
  int children[6];
  return l3p_paged_seq_fork(ctx, ids[2], 333, 6, children);
}
static int compact_call(l3p_paged_ctx* ctx, const int*) {
  int used;
  return l3p_paged_compact(ctx, &used, nullptr);
}

// Every allocation of create fails in turn: it returns L3P_E_NOMEM, says why, and leaves no context.
static void create_everywhere(int dtype) {
  l3p_paged_config c{};
  c.n_layers = 1, c.n_heads = 8, c.n_kv_heads = 2, c.head_dim = 64, c.page_size = 16, c.n_pages = kPages;
  c.max_seqs = kSeqs, c.max_tokens = 4000, c.dtype = dtype;
  int refused = 0;
  for (long at = 0, reached = 1; reached; ++at) {
    l3p_paged_ctx* ctx = nullptr;
    g_watch = true, g_fail_in = at;
    const int rc = l3p_paged_create(&c, &ctx);
    g_watch = false;
    reached = g_fail_in < 0;
    g_fail_in = -1;
    EXPECT((rc == L3P_OK) == (l3p_paged_create_error()[0] == 0) && (rc == L3P_OK) == (ctx != nullptr));
    EXPECT(reached ? rc == L3P_E_NOMEM || rc == L3P_E_CUDA : rc == L3P_OK);
    refused += rc != L3P_OK;
    l3p_paged_destroy(ctx);
  }
  EXPECT(refused > 5);
}

// Calls that move host data, on a stream that captures and on the null stream while another one does.
static void refused_in_capture(int dtype) {
  int ids[8], free_id[1];
  l3p_paged_ctx* ctx = make(dtype);
  fill(ctx, ids);
  free_id[0] = ids[1];
  EXPECT(l3p_paged_seq_free(ctx, 1, free_id) == L3P_OK);  // holes for compact
  const int one[1] = {1};
  EXPECT(l3p_paged_begin(ctx, 1, ids + 2, one, nullptr) == L3P_OK);
  const Seen before = look(ctx);
  for (bool* how : {&g_capturing, &g_implicit}) {
    *how = true;
    int children[1], used;
    EXPECT(l3p_paged_begin(ctx, 1, ids, one, nullptr) == L3P_E_INVAL);
    EXPECT(l3p_paged_seq_copy(ctx, 1, ids, children, nullptr) == L3P_E_INVAL);
    EXPECT(l3p_paged_compact(ctx, &used, nullptr) == L3P_E_INVAL);
    EXPECT(l3p_paged_check(ctx, nullptr) == L3P_E_INVAL);  // a wait would end the capture
    *how = false;
    EXPECT(look(ctx) == before);
  }
  l3p_paged_destroy(ctx);
}

int main(int argc, char** argv) {
  const std::string test = argc > 1 ? argv[1] : "";
  g_fail_rest = argc > 2 && std::string(argv[2]) == "rest";
  for (int dtype : {L3P_PAGED_F32, L3P_PAGED_BF16}) {
    if (test == "capture") {
      refused_in_capture(dtype);
    } else if (test == "create") {
      create_everywhere(dtype);
    } else if (test == "begin") {
      fail_everywhere("begin", dtype, begin_call);
    } else if (test == "copy") {
      fail_everywhere("copy", dtype, copy_call);
    } else if (test == "fork") {
      fail_everywhere("fork", dtype, fork_call);
    } else if (test == "compact") {
      fail_everywhere("compact", dtype, compact_call, true);
    } else {
      printf("no test %s\n", test.c_str());
      return 1;
    }
  }
  return g_bad != 0;
}

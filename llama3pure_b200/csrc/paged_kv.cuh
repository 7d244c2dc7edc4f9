// paged_kv.cuh -- what writes the paged cache: rotation and write of a batch's
// new rows, copies of page rows, and the cosine / sine tables (sm_100a).
#pragma once
#include <cuda_bf16.h>

#include "paged.h"
#include "ptx.cuh"

namespace l3p {

// ---- rows of either type as fp32 registers: lane l holds the HD/32
// consecutive values from l * HD/32 on ---------------------------------------
template <int N>
__device__ __forceinline__ void pg_load(const float* __restrict__ p, float (&x)[N]) {
  if constexpr (N == 2) {
    const float2 t = *reinterpret_cast<const float2*>(p);
    x[0] = t.x, x[1] = t.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 t = *reinterpret_cast<const float4*>(p + i);
      x[i] = t.x, x[i + 1] = t.y, x[i + 2] = t.z, x[i + 3] = t.w;
    }
  }
}
template <int N>
__device__ __forceinline__ void pg_load(const __nv_bfloat16* __restrict__ p, float (&x)[N]) {
  uint32_t w[N / 2];
  if constexpr (N == 2)
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  else if constexpr (N == 4)
    *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(p);
  else
    *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(p);
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
template <int N>
__device__ __forceinline__ void pg_store(float* __restrict__ p, const float (&x)[N]) {
  if constexpr (N == 2) {
    *reinterpret_cast<float2*>(p) = make_float2(x[0], x[1]);
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
  }
}
// One rounding, to nearest even, of values computed in fp32.
template <int N>
__device__ __forceinline__ void pg_store(__nv_bfloat16* __restrict__ p, const float (&x)[N]) {
  uint32_t w[N / 2];
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&t);
  }
  if constexpr (N == 2)
    *reinterpret_cast<uint32_t*>(p) = w[0];
  else if constexpr (N == 4)
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(w);
  else
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(w);
}

__device__ __forceinline__ float pg_f32(float x) { return x; }
__device__ __forceinline__ float pg_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

struct PgKvArgs {
  const int* batch;
  int n_tokens;  // of the launch: a replay must not find more tokens,
  int max_pos;   //   nor positions behind the rotary tables
  const void* q;
  const void* k;
  const void* v;
  void* q_out;
  long long q_stride, k_stride, v_stride, q_out_stride;
  void* storage;              // this layer's K block of page 0, head 0
  long long page_elems;       // values from one page to the next
  long long v_off;            // values from the K to the V block of a layer
  int page_size, shift, n_heads, n_kv;
  const float2* tab;          // [max_pos][rotary/2]
  const float* q_norm;        // this layer's weights, or null
  const float* k_norm;
  float eps;
  int rotary, interleaved;
  int rows_per_warp;          // head rows of one token that a warp takes
  int* err;
};

constexpr int kPgKvWarps = 8;

// Rotation and write of the new rows, for what the streamed form below does not take: tokens of which two do not fit its
// ring, and odd numbers of pairs.  One warp takes `rows_per_warp`
// consecutive head rows (query heads first, then K heads, then V heads) of one
// token; cosines and sines are read once for all of them.
//   x' = x * rsqrt(mean x^2 + eps) * w              (where norm weights are given)
//   (a, b) -> (a cos - b sin, a sin + b cos)        for the pairs of the first `rotary` values
// in fp32, rounded once on the way out.  Bound by memory: every row is read and
// written once.  A pair's partner sits in another lane in the half layout, at
// a distance that depends on `rotary`, so rows pass through shared memory there.
template <typename T, int HD>
__global__ void __launch_bounds__(kPgKvWarps * 32) paged_rope_kernel(const PgKvArgs a) {
  constexpr int N = HD / 32;
  constexpr int U = 4;  // rows that a warp turns at once
  __shared__ __align__(16) float row_s[kPgKvWarps][U][HD];
  const PgHeader* h = reinterpret_cast<const PgHeader*>(a.batch);
  const int n_tok = h->n_tokens;
  griddep_wait();  // the rows come from the kernel before this one
  griddep_launch();
  if (n_tok > a.n_tokens) {  // a replay on a larger batch than the captured one
    if (blockIdx.x == 0 && threadIdx.x == 0) *reinterpret_cast<volatile int*>(a.err) = kErrBadArg;
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n_rows = a.n_heads + 2 * a.n_kv;
  const int chunks = (n_rows + a.rows_per_warp - 1) / a.rows_per_warp;
  const long long item = (long long)blockIdx.x * kPgKvWarps + warp;
  const int tok = (int)(item / chunks);
  if (tok >= n_tok) return;
  const int r0 = (int)(item % chunks) * a.rows_per_warp, r1 = min(r0 + a.rows_per_warp, n_rows);
  const int2 tp = *reinterpret_cast<const int2*>(a.batch + h->tok + 2 * tok);
  if (tp.y >= a.max_pos) {
    if (lane == 0) *reinterpret_cast<volatile int*>(a.err) = kErrBadArg;
    return;
  }
  const int d0 = lane * N;  // this lane's values of a row
  float cs[N], sn[N];
  const int half = a.rotary / 2;
  if (r0 < a.n_heads + a.n_kv) {
    const float2* t = a.tab + (long long)tp.y * half;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int d = d0 + i;
      cs[i] = 1.f, sn[i] = 0.f;
      if (d < a.rotary) {
        const float2 c = t[a.interleaved ? d / 2 : d < half ? d : d - half];
        // x' = x cos + partner * s, s negative for the first of a pair
        const bool first = a.interleaved ? (d & 1) == 0 : d < half;
        cs[i] = c.x;
        sn[i] = first ? -c.y : c.y;
      }
    }
  }
  const int page = tp.x >> a.shift, slot = tp.x & (a.page_size - 1);
  T* page_k = static_cast<T*>(a.storage) + (long long)page * a.page_elems + (long long)slot * HD + d0;
  const T* qt = static_cast<const T*>(a.q) + tok * a.q_stride + d0;
  const T* kt = static_cast<const T*>(a.k) + tok * a.k_stride + d0;
  const T* vt = static_cast<const T*>(a.v) + tok * a.v_stride + d0;
  T* qo = static_cast<T*>(a.q_out) + tok * a.q_out_stride + d0;
  const long long head_elems = (long long)a.page_size * HD;
  float wq[N], wk[N];
  if (a.q_norm != nullptr && r0 < a.n_heads + a.n_kv) {
    pg_load<N>(a.q_norm + d0, wq);
    pg_load<N>(a.k_norm + d0, wk);
  }
  for (int r = r0; r < r1; r += U) {
    float x[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int rr = min(r + u, r1 - 1);
      const T* src = rr < a.n_heads ? qt + rr * HD
                     : rr < a.n_heads + a.n_kv ? kt + (rr - a.n_heads) * HD
                                               : vt + (rr - a.n_heads - a.n_kv) * HD;
      pg_load<N>(src, x[u]);
    }
    // the U rows together, so that their reductions and exchanges overlap; V rows are only copied
    const bool turns = r < a.n_heads + a.n_kv;
    if (turns && a.q_norm != nullptr) {
      float ss[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        ss[u] = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) ss[u] += x[u][i] * x[u][i];
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int u = 0; u < U; ++u) ss[u] += __shfl_xor_sync(0xffffffffu, ss[u], o);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float f = 1.0f / sqrtf(ss[u] * (1.0f / HD) + a.eps);
        if (r + u < a.n_heads + a.n_kv) {
#pragma unroll
          for (int i = 0; i < N; ++i) x[u][i] = x[u][i] * f * (r + u < a.n_heads ? wq[i] : wk[i]);
        }
      }
    }
    if (turns && a.interleaved) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (r + u < a.n_heads + a.n_kv) {
#pragma unroll
          for (int i = 0; i < N; i += 2) {
            const float p = x[u][i], q = x[u][i + 1];
            if (d0 + i < a.rotary) {
              x[u][i] = p * cs[i] + q * sn[i];
              x[u][i + 1] = q * cs[i + 1] + p * sn[i + 1];
            }
          }
        }
    } else if (turns) {
      __syncwarp();  // the rows before have been read
#pragma unroll
      for (int u = 0; u < U; ++u) pg_store<N>(row_s[warp][u] + d0, x[u]);
      __syncwarp();
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (r + u < a.n_heads + a.n_kv) {
          float y[N];  // the partners
          if (half % N == 0) {
            pg_load<N>(row_s[warp][u] + (d0 < half ? d0 + half : d0 < a.rotary ? d0 - half : d0), y);
          } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
              const int d = d0 + i;
              y[i] = row_s[warp][u][d < half ? d + half : d < a.rotary ? d - half : d];
            }
          }
#pragma unroll
          for (int i = 0; i < N; ++i)
            if (d0 + i < a.rotary) x[u][i] = x[u][i] * cs[i] + y[i] * sn[i];
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int rr = r + u;
      if (rr >= r1) break;
      if (rr < a.n_heads)
        pg_store<N>(qo + rr * HD, x[u]);
      else if (rr < a.n_heads + a.n_kv)
        pg_store<N>(page_k + (rr - a.n_heads) * head_elems, x[u]);
      else
        pg_store<N>(page_k + a.v_off + (rr - a.n_heads - a.n_kv) * head_elems, x[u]);
    }
  }
}

// The same, streamed: one producer warp brings whole tokens (q, k, v rows and the token's row of the table) into a ring in
// shared memory with bulk copies, eight warps turn a head row each from there; partners are read where they lie.  Norm
// weights are folded into the cosines and sines once a token, so a row costs ~80 instructions (8191 tokens, 8B heads, fp32,
// 403 MB with norms: 77 us = 5.2 TB/s, 81 % of a copy; half of the issue slots).
constexpr int kPgRingThreads = (kPgKvWarps + 1) * 32;
constexpr int kPgRingStages = 4;  // at most
struct PgRingArgs {
  int stages, stage_bytes;            // of the ring; a stage: q rows, k rows, v rows, table row
  int q_bytes, kv_bytes, tab_bytes;
};

template <typename T, int HD>
__global__ void __launch_bounds__(kPgRingThreads) paged_rope_ring_kernel(const PgKvArgs a, const PgRingArgs g) {
  constexpr int N = HD / 32;
  extern __shared__ __align__(128) unsigned char rope_ring[];
  __shared__ __align__(8) uint64_t full[kPgRingStages], empty[kPgRingStages];
  __shared__ int2 s_tok[kPgRingStages];
  const PgHeader* h = reinterpret_cast<const PgHeader*>(a.batch);
  const int n_tok = h->n_tokens;
  if (threadIdx.x == 0) {
    for (int s = 0; s < g.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], kPgKvWarps);
    }
    fence_mbar_init();
  }
  __syncthreads();
  griddep_wait();  // the rows come from the kernel before this one
  griddep_launch();  // not earlier: the next kernel's CTAs would only wait (64 tokens, 8B heads, call after call: 2.7 us, 2.9)
  if (n_tok > a.n_tokens) {
    if (blockIdx.x == 0 && threadIdx.x == 0) *reinterpret_cast<volatile int*>(a.err) = kErrBadArg;
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int half = a.rotary / 2;
  if (warp == kPgKvWarps) {
    if (lane == 0) {
      int i = 0;
      for (int tok = blockIdx.x; tok < n_tok; tok += gridDim.x, ++i) {
        const int s = i % g.stages, use = i / g.stages;
        const int2 tp = *reinterpret_cast<const int2*>(a.batch + h->tok + 2 * tok);
        if (use > 0 && !mbar_wait_bounded(&empty[s], (uint32_t)((use - 1) & 1), a.err)) break;
        const bool ok = tp.y < a.max_pos;  // else the warps report it
        s_tok[s] = tp;
        unsigned char* st = rope_ring + s * g.stage_bytes;
        mbar_arrive_expect_tx(&full[s], (uint32_t)(g.q_bytes + 2 * g.kv_bytes + (ok ? g.tab_bytes : 0)));
        auto copy = [&](unsigned char* dst, const void* src, int bytes) {
          asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_addr(dst)),
                       "l"(src), "r"(bytes), "r"(smem_addr(&full[s]))
                       : "memory");
        };
        copy(st, static_cast<const T*>(a.q) + tok * a.q_stride, g.q_bytes);
        copy(st + g.q_bytes, static_cast<const T*>(a.k) + tok * a.k_stride, g.kv_bytes);
        copy(st + g.q_bytes + g.kv_bytes, static_cast<const T*>(a.v) + tok * a.v_stride, g.kv_bytes);
        if (ok) copy(st + g.q_bytes + 2 * g.kv_bytes, a.tab + (long long)tp.y * half, g.tab_bytes);
      }
      for (int x = i > g.stages ? i - g.stages : 0; x < i; ++x)  // no copy may still be landing when the CTA ends
        mbar_wait_bounded(&full[x % g.stages], (uint32_t)((x / g.stages) & 1), a.err);
    }
    return;
  }
  const int d0 = lane * N;
  const long long head_elems = (long long)a.page_size * HD;
  // the partner of this lane's value e
  auto partner = [&](int e) {
    const int d = d0 + e;
    return a.interleaved ? d ^ 1 : d < half ? d + half : d < a.rotary ? d - half : d;
  };
  const bool norm = a.q_norm != nullptr;
  float wq[N], wqp[N], wk[N], wkp[N];  // norm weights of the values and of their partners
#pragma unroll
  for (int e = 0; e < N; ++e) {
    wq[e] = norm ? a.q_norm[d0 + e] : 1.f;
    wk[e] = norm ? a.k_norm[d0 + e] : 1.f;
    wqp[e] = norm ? a.q_norm[partner(e)] : 1.f;
    wkp[e] = norm ? a.k_norm[partner(e)] : 1.f;
  }
  // x' = f (x c + partner s) with c = cos w, s = +-sin w of the partner, and f of the row's norm
  auto turn = [&](const T* row, T* dst, const float (&c)[N], const float (&sn)[N]) {
    float x[N], y[N], f = 1.f;
    pg_load<N>(row + d0, x);
    if (a.interleaved) {
#pragma unroll
      for (int e = 0; e < N; ++e) y[e] = x[e ^ 1];
    } else if (half % N == 0) {
      pg_load<N>(row + partner(0), y);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) y[e] = pg_f32(row[partner(e)]);
    }
    if (norm) {
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < N; ++e) ss += x[e] * x[e];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      f = rsqrtf(ss * (1.0f / HD) + a.eps);  // within 2 units of the last place
    }
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float z = x[e] * c[e];
      x[e] = (d0 + e < a.rotary ? z + y[e] * sn[e] : z) * f;
    }
    pg_store<N>(dst, x);
  };
  int i = 0;
  for (int tok = blockIdx.x; tok < n_tok; tok += gridDim.x, ++i) {
    const int s = i % g.stages;
    if (!__all_sync(0xffffffffu, mbar_wait_bounded(&full[s], (uint32_t)((i / g.stages) & 1), a.err))) return;
    const unsigned char* st = rope_ring + s * g.stage_bytes;
    const int2 tp = s_tok[s];
    if (tp.y >= a.max_pos) {
      if (lane == 0) *reinterpret_cast<volatile int*>(a.err) = kErrBadArg;
    } else {
      const float2* tab = reinterpret_cast<const float2*>(st + g.q_bytes + 2 * g.kv_bytes);
      float cq[N], sq[N], ck[N], sk[N];
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int d = d0 + e;
        float2 t = make_float2(1.f, 0.f);
        if (d < a.rotary) {
          t = tab[a.interleaved ? d / 2 : d < half ? d : d - half];
          if (a.interleaved ? (d & 1) == 0 : d < half) t.y = -t.y;  // the first of a pair
        }
        cq[e] = t.x * wq[e], sq[e] = t.y * wqp[e];
        ck[e] = t.x * wk[e], sk[e] = t.y * wkp[e];
      }
      const int page = tp.x >> a.shift, slot = tp.x & (a.page_size - 1);
      T* page_k = static_cast<T*>(a.storage) + (long long)page * a.page_elems + (long long)slot * HD + d0;
      T* qo = static_cast<T*>(a.q_out) + tok * a.q_out_stride + d0;
      const T* rows = reinterpret_cast<const T*>(st);  // q, k and v rows, one after the other
      int r = warp;
#pragma unroll 4
      for (; r < a.n_heads; r += kPgKvWarps) turn(rows + r * HD, qo + r * HD, cq, sq);
      r -= a.n_heads;
      rows += a.n_heads * HD;
      for (; r < a.n_kv; r += kPgKvWarps) turn(rows + r * HD, page_k + r * head_elems, ck, sk);
      r -= a.n_kv;
      rows += a.n_kv * HD;
      for (; r < a.n_kv; r += kPgKvWarps) {
        float x[N];
        pg_load<N>(rows + r * HD + d0, x);
        pg_store<N>(page_k + a.v_off + r * head_elems, x);
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[s]);
  }
}

// The new rows as they are: K and V of a token, 16 bytes a thread.
__global__ void paged_append_kernel(const PgKvArgs a, int vecs, int es) {
  const PgHeader* h = reinterpret_cast<const PgHeader*>(a.batch);
  const int n_tok = h->n_tokens;
  griddep_wait();
  griddep_launch();
  if (n_tok > a.n_tokens) {
    if (blockIdx.x == 0 && threadIdx.x == 0) *reinterpret_cast<volatile int*>(a.err) = kErrBadArg;
    return;
  }
  const int per_tok = 2 * a.n_kv * vecs;  // vecs: 16-byte pieces of a head row
  const long long n = (long long)n_tok * per_tok;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
    const int tok = (int)(i / per_tok), r = (int)(i % per_tok);
    const int head = r / vecs, c = r % vecs;
    const bool is_v = head >= a.n_kv;
    const int kvh = is_v ? head - a.n_kv : head;
    const int slot_row = a.batch[h->tok + 2 * tok];
    const int page = slot_row >> a.shift, slot = slot_row & (a.page_size - 1);
    const char* src = static_cast<const char*>(is_v ? a.v : a.k) + (tok * (is_v ? a.v_stride : a.k_stride)) * es +
                      ((long long)kvh * vecs + c) * 16;
    char* dst = static_cast<char*>(a.storage) + (page * a.page_elems + (is_v ? a.v_off : 0)) * es +
                (((long long)kvh * a.page_size + slot) * vecs + c) * 16;
    *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
  }
}

// Copies the first `rows` rows of every (layer, K/V, head) block of a page to
// another page.  Destinations are free pages, so no job reads what another
// writes.  One warp per block, four 16-byte loads a lane in flight; bound by
// memory.  grid (CTAs, jobs).
__global__ void __launch_bounds__(256) paged_copy_kernel(const int4* __restrict__ jobs, char* storage, long long page_bytes,
                                                         int blocks, int block_bytes, int row_bytes) {
  const int4 j = jobs[blockIdx.y];
  const int lane = threadIdx.x & 31;
  const int n = j.z * row_bytes / 16;  // 16-byte pieces of a block's rows
  for (int b = blockIdx.x * 8 + (threadIdx.x >> 5); b < blocks; b += gridDim.x * 8) {
    const uint4* src = reinterpret_cast<const uint4*>(storage + j.x * page_bytes + (long long)b * block_bytes);
    uint4* dst = reinterpret_cast<uint4*>(storage + j.y * page_bytes + (long long)b * block_bytes);
    int i = lane;
    for (; i + 96 < n; i += 128) {
      const uint4 t0 = src[i], t1 = src[i + 32], t2 = src[i + 64], t3 = src[i + 96];
      dst[i] = t0, dst[i + 32] = t1, dst[i + 64] = t2, dst[i + 96] = t3;
    }
    for (; i < n; i += 32) dst[i] = src[i];
  }
}

// (cos, sin) * factor of pos * freq[i], the angle and both functions in double precision.
__global__ void paged_rope_table_kernel(float2* tab, const double* __restrict__ freq, int half, int n_pos, double factor) {
  const long long n = (long long)n_pos * half;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
    double s, c;
    sincos((double)(i / half) * freq[i % half], &s, &c);
    tab[i] = make_float2((float)(c * factor), (float)(s * factor));
  }
}

}  // namespace l3p

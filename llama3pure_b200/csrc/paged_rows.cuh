// paged_rows.cuh -- attention of few query rows per KV head over paged keys
// and values (sm_100a): decoding sequences, drafts, short chunk tails.
//
// Mathematics.  For the rows r of one sequence and KV head
//   s_rj = scale q_r . k_j,  o_r = sum_j 2^(s_rj log2e - m_r) v_j / l_r
// over the keys j in [max(0, t_r - w + 1), t_r], in one pass over K and V with
// the running maximum m and sum l of each row in fp32.
//
// What bounds it: the K/V bytes.  A KV head's rows serve the whole group of
// query heads, so every byte is read once for up to 8*NT rows.
//
// Split.  The host lays the 16-key tiles of all (sequence, KV head, row block)
// units end to end and cuts them into one equal run per CTA (plan_rows), so
// every SM streams the same number of bytes whatever the lengths are.  Inside
// a run the CTA's warps take tiles in turn, each through its own ring of
// cp.async places; a warp prefetches across the end of a segment, so the merge
// of one sequence overlaps the loads of the next.  A unit cut by a run boundary
// is merged by the part that ends last, in the order of the parts.
//
// Products.  The keys are the M side of the matrix instructions and the query
// rows the N side (S^T = K Q^T, O^T = V^T P^T): a block of 8 rows wastes
// nothing, where rows on the M side would pad them to 16.  mma.sync, not
// tcgen05: at 8 rows per KV head an SM has ~350 cycles per 8 KB of K/V from
// HBM and needs ~50 of them for the products, so operands go from the ring to
// registers with ldmatrix and nothing waits for tensor memory.
//   bf16: m16n8k16, fp32 accumulators; P is rounded to bf16 for the second
//         product (at most 2^-8 of each weight), l sums the unrounded P.
//   fp32: 3xTF32 m16n8k8 (x = hi + lo; hi*hi + hi*lo + lo*hi).  The matrix
//         instruction cuts its sums off instead of rounding them, a bias that
//         grows with every instruction in a chain (1.4e-5 of the output at
//         128K keys), so at most six instructions share an accumulator and
//         what they leave is added to the running fp32 sums by ordinary adds.
#pragma once
#include <cuda_bf16.h>

#include "paged.h"
#include "ptx.cuh"

namespace l3p {

struct PgRowArgs {
  const int* batch;
  const void* q;
  void* out;
  long long q_stride, out_stride;
  const void* storage;  // the layer's K block of page 0, head 0
  long long page_elems, v_off;
  int shift, G, win, window;
  PgLimits lim;
  int late;          // the kernel before is a tensor-core kernel of the same call: wait for it at the end only
  float scale_log2;
  float* ws_o;       // [slot][8*NT][HD]
  float* ws_ml;      // [slot][8*NT][2]
  unsigned* tickets;
  int* err;
};

template <typename T, int HD>
struct PgRowCfg {
  static constexpr int kEs = (int)sizeof(T);
  static constexpr int kRow = HD * kEs;               // bytes of a K or V row
  static constexpr int kTileBytes = kPgTile * kRow;  // a tile's K or V
  // 192 KB of rings per CTA, at least three places per warp: the one that it computes on and those in flight.  A place
  // holds K and V of a tile; for fp32, whose split products keep a warp on a tile for 2.5K cycles, K or V, which makes room
  // for twice the warps (one token on 128K keys, 8B heads, the same 1.07 GB call after call, of which L2 keeps a tenth: 181 ->
  // 163 us; on caches in turn 182 us = 5.9 TB/s.  64 sequences of 4095, Gemma heads: 250 -> 142 us.  bf16 loses 5 % to the
  // second wait a tile).  Four warps for head_dim 256, whose merge buffer is twice as large.
  static constexpr bool kPair = kEs == 2;
  static constexpr int kPlaceBytes = kPair ? 2 * kTileBytes : kTileBytes;
  static constexpr int kWarps = HD == 256 ? 4 : 8;
  static constexpr int kPlaces = 196608 / (kWarps * kPlaceBytes);
  static constexpr int kRing = kWarps * kPlaces * kPlaceBytes;
  // one block of 8 rows per warp; at least the weights of kPgMaxCtas parts for 32 rows
  static constexpr int kMerge = kWarps * 8 * HD * 4 > 32 * kPgMaxCtas * 4 ? kWarps * 8 * HD * 4 : 32 * kPgMaxCtas * 4;
  static constexpr int kSmem = kRing + kMerge + kWarps * 32 * 2 * 4;
  static_assert(kPlaces >= 3 && kSmem <= 232448 - 64, "shared memory of the row kernel");
};

__device__ __forceinline__ void pg_cp16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void pg_ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void pg_ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t pg_transpose(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ void pg_mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void pg_mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = hi + lo: hi is x rounded to tf32's 11 significant bits, lo = x - hi is
// exact in fp32.  Rounding hi to nearest leaves lo 12 bits of either sign, so
// the bit that tf32 drops of it has no bias.
__device__ __forceinline__ void pg_split(float x, uint32_t& hi, uint32_t& lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xFFFFE000u;
  lo = __float_as_uint(x - __uint_as_float(hi));
}
__device__ __forceinline__ uint32_t pg_pack_bf16(float lo, float hi) {
  const __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&t);
}
__device__ __forceinline__ float pg_f32(float x) { return x; }
__device__ __forceinline__ float pg_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ bool pg_finite(float x) { return (__float_as_uint(x) & 0x7F800000u) != 0x7F800000u; }

// Byte offset of 16-byte piece c of row r in a K or V tile.  bf16: ldmatrix
// reads one piece of 8 rows.  fp32: a quarter warp reads 4 pieces of 2 rows
// (K: rows 2j, 2j+1) or 2 pieces of 4 rows (V): bits 2 and 1 of the piece are
// flipped by bits 0 and 1 of the row, so either hits 8 different pieces.
template <typename T, int HD>
__device__ __forceinline__ uint32_t pg_piece(int r, int c) {
  if constexpr (sizeof(T) == 2) return (uint32_t)(r * (HD * 2) + ((c ^ (r & 7)) << 4));
  return (uint32_t)(r * (HD * 4) + ((c ^ (((r & 1) << 2) | (r & 2))) << 4));
}

// Whether a 16-byte piece of a V tile holds a value that is not finite, and
// the piece with such values set to 0.
template <typename T>
__device__ __forceinline__ bool pg_clean(uint4& v) {
  uint32_t* w = reinterpret_cast<uint32_t*>(&v);
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 2) {
      if ((w[i] & 0x7F80u) == 0x7F80u) w[i] &= 0xFFFF0000u, bad = true;
      if ((w[i] & 0x7F800000u) == 0x7F800000u) w[i] &= 0x0000FFFFu, bad = true;
    } else {
      if ((w[i] & 0x7F800000u) == 0x7F800000u) w[i] = 0u, bad = true;
    }
  }
  return bad;
}

template <typename T, int HD, int NT>
__global__ void __launch_bounds__(PgRowCfg<T, HD>::kWarps * 32, 1) paged_rows_kernel(const PgRowArgs a) {
  using C = PgRowCfg<T, HD>;
  constexpr bool kB = sizeof(T) == 2;
  constexpr int NW = C::kWarps, NP = C::kPlaces;
  constexpr int MT = HD / 16;        // 16-value blocks of O^T
  constexpr int KS = HD / 16;        // bf16: k-steps of S; fp32: pairs of k-steps
  extern __shared__ __align__(128) unsigned char sm[];
  __shared__ int s_last;
  float* merge = reinterpret_cast<float*>(sm + C::kRing);
  float* s_ml = reinterpret_cast<float*>(sm + C::kRing + C::kMerge);  // [warp][8*NT][2]

  const PgHeader* h = reinterpret_cast<const PgHeader*>(a.batch);
  const PgLists l = h->lists[a.win];
  griddep_launch();
  // In a batch with chunks this kernel follows a tensor-core kernel, which lets it start once all of its CTAs have seen the
  // kernel before them complete.  The two read the same rows and write others, so they run side by side; this one's CTAs
  // wait at their end, so that what follows this kernel follows both.
  const bool fits = pg_fits(h, l, a.lim);
  if (!fits || (int)blockIdx.x >= l.row_ctas) {
    griddep_wait();
    if (!fits && blockIdx.x == 0 && threadIdx.x == 0) *reinterpret_cast<volatile int*>(a.err) = kErrBadArg;
    return;
  }
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const int seg_end = a.batch[l.row_first + blockIdx.x + 1];
  const PgSeg* segs = reinterpret_cast<const PgSeg*>(a.batch + l.row_segs);
  const int* tables = a.batch + h->tbl;
  const uint32_t ring = smem_addr(sm) + warp * NP * C::kPlaceBytes;
  const T* kbase = static_cast<const T*>(a.storage);
  const long long head_elems = (long long)HD << a.shift;

  // ---- loads: tiles in the order they are used, across segments ----------------
  int is = a.batch[l.row_first + blockIdx.x];  // segment of the next tile to load
  const int seg0 = is;
  int it = 0, ie = 0, ilo = 0, ihi = 0, itbl = 0, ikvh = 0, ipage = 0;
  auto load_seg = [&]() {
    const PgSeg& s = segs[is];
    it = s.tile0 + warp, ie = s.tile1, ilo = s.key_lo, ihi = s.key_hi, itbl = s.tbl, ikvh = s.kvh;
  };
  auto settle = [&]() {  // to the next tile of this warp, and its page
    while (is < seg_end && it >= ie)
      if (++is < seg_end) load_seg();
    if (is < seg_end) ipage = tables[itbl + ((it * kPgTile) >> a.shift)];
  };
  int iplace = 0;
  bool iv = false;  // V of the tile is next, not K (places that hold one of the two)
  auto issue = [&]() {
    if (is < seg_end) {
      const uint32_t dst = ring + iplace * C::kPlaceBytes;
      const int key0 = it * kPgTile;
      const T* src = kbase + (iv ? a.v_off : 0) + (long long)ipage * a.page_elems + ikvh * head_elems +
                     (long long)(key0 & ((1 << a.shift) - 1)) * HD;
#pragma unroll
      for (int i = 0; i < C::kTileBytes / 512; ++i) {
        const int p = i * 32 + lane, r = p / (C::kRow / 16), c = p % (C::kRow / 16);
        // rows that nobody attends to read as zero, whatever the page holds
        const int bytes = key0 + r >= ilo && key0 + r < ihi ? 16 : 0;
        const uint32_t off = pg_piece<T, HD>(r, c);
        pg_cp16(dst + off, src + p * (16 / C::kEs), bytes);
        if (C::kPair) pg_cp16(dst + C::kTileBytes + off, src + a.v_off + p * (16 / C::kEs), bytes);
      }
      if (C::kPair || iv) {
        it += NW;
        settle();
      }
      if (!C::kPair) iv = !iv;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    iplace = iplace + 1 == NP ? 0 : iplace + 1;
  };
  if (is < seg_end) load_seg();
  settle();
  // q and the new tokens' rows come from the kernel before this one, and older rows may: begin copies shared pages, callers
  // write the storage with kernels of their own, and none of that is visible before the wait (tiles of older rows loaded
  // ahead of it saved 0.2 to 1.2 us a layer: one token on 8K keys, 8B heads, with its rotation 14.0 us, now 15.2).
  if (!a.late) griddep_wait();
#pragma unroll
  for (int i = 0; i < NP - 1; ++i) issue();

  // the next place in the order of use, once it is there; the place used before it goes to the load after the last
  int cplace = 0;
  auto next_place = [&]() {
    asm volatile("cp.async.wait_group %0;" ::"n"(NP - 2) : "memory");
    __syncwarp();
    issue();
    const uint32_t at = ring + cplace * C::kPlaceBytes;
    cplace = cplace + 1 == NP ? 0 : cplace + 1;
    return at;
  };
  for (int si = seg0; si < seg_end; ++si) {
    const PgSeg& sg = segs[si];
    const int n_rows = sg.n_rows, r0 = sg.r0, pos0 = sg.pos0, q_row0 = sg.q_row0, kvh = sg.kvh, key_lo = sg.key_lo,
              key_hi = sg.key_hi, tbl = sg.tbl, tile0 = sg.tile0, tile1 = sg.tile1;
    // positions of this thread's rows (rows beyond n_rows follow the last one)
    int qp[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) qp[n][j] = pos0 + (r0 + min(n * 8 + 2 * t4 + j, n_rows - 1)) / a.G;
    const int full_hi = pos0 + r0 / a.G + 1;  // keys below: every row attends to them
    const int last_pos = pos0 + (r0 + n_rows - 1) / a.G;
    const int full_lo = a.win ? max(0, last_pos - a.window + 1) : 0;

    // ---- Q fragments: this thread holds row g of each block ----------------------
    uint32_t qa[NT][KS][kB ? 2 : 4], qb[NT][kB ? 1 : KS][4];  // bf16: qa; fp32: qa hi, qb lo
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = r0 + n * 8 + g;
      const bool ok = n * 8 + g < n_rows;
      const T* qr = static_cast<const T*>(a.q) + (long long)(q_row0 + r / a.G) * a.q_stride +
                    (long long)(kvh * a.G + r % a.G) * HD;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        if constexpr (kB) {
          qa[n][k][0] = ok ? *reinterpret_cast<const uint32_t*>(qr + 16 * k + 2 * t4) : 0u;
          qa[n][k][1] = ok ? *reinterpret_cast<const uint32_t*>(qr + 16 * k + 8 + 2 * t4) : 0u;
        } else {
          const float4 x = ok ? *reinterpret_cast<const float4*>(qr + 16 * k + 4 * t4) : make_float4(0.f, 0.f, 0.f, 0.f);
          pg_split(x.x, qa[n][k][0], qb[n][k][0]);
          pg_split(x.y, qa[n][k][1], qb[n][k][1]);
          pg_split(x.z, qa[n][k][2], qb[n][k][2]);
          pg_split(x.w, qa[n][k][3], qb[n][k][3]);
        }
      }
    }
    float o[NT][MT][4], m[NT][2], lsum[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      lsum[n][0] = lsum[n][1] = 0.f;
#pragma unroll
      for (int i = 0; i < MT; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
    }

    for (int t = tile0 + warp; t < tile1; t += NW) {
      const uint32_t ks = next_place();
      const int key0 = t * kPgTile;
      // ---- S^T = K Q^T --------------------------------------------------------------
      float sc[NT][4], sd[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[n][i] = sd[n][i] = 0.f;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        if constexpr (kB) {
          uint32_t ka[4];
          pg_ldsm4(ka, ks + pg_piece<T, HD>((lane & 7) + (lane & 8), 2 * k + (lane >> 4)));
#pragma unroll
          for (int n = 0; n < NT; ++n) pg_mma_bf16(k & 1 ? sd[n] : sc[n], ka, qa[n][k][0], qa[n][k][1]);
        } else {
          float4 x, y;
          const uint32_t ax = ks + pg_piece<T, HD>(g, 4 * k + t4), ay = ks + pg_piece<T, HD>(g + 8, 4 * k + t4);
          asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(ax));
          asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(y.x), "=f"(y.y), "=f"(y.z), "=f"(y.w) : "r"(ay));
          uint32_t hi[4], lo[4];
          pg_split(x.x, hi[0], lo[0]);
          pg_split(y.x, hi[1], lo[1]);
          pg_split(x.y, hi[2], lo[2]);
          pg_split(y.y, hi[3], lo[3]);
          float c0[NT][4], c1[NT][4];
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            c0[n][0] = c0[n][1] = c0[n][2] = c0[n][3] = 0.f;
            pg_mma_tf32(c0[n], lo, qa[n][k][0], qa[n][k][1]);
            pg_mma_tf32(c0[n], hi, qb[n][k][0], qb[n][k][1]);
            pg_mma_tf32(c0[n], hi, qa[n][k][0], qa[n][k][1]);
          }
          pg_split(x.z, hi[0], lo[0]);
          pg_split(y.z, hi[1], lo[1]);
          pg_split(x.w, hi[2], lo[2]);
          pg_split(y.w, hi[3], lo[3]);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            c1[n][0] = c1[n][1] = c1[n][2] = c1[n][3] = 0.f;
            pg_mma_tf32(c1[n], lo, qa[n][k][2], qa[n][k][3]);
            pg_mma_tf32(c1[n], hi, qb[n][k][2], qb[n][k][3]);
            pg_mma_tf32(c1[n], hi, qa[n][k][2], qa[n][k][3]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              sc[n][i] += c0[n][i];
              sd[n][i] += c1[n][i];
            }
          }
        }
      }
      // ---- softmax: this thread has keys key0 + g, key0 + g + 8 of rows 2*t4, 2*t4 + 1 ---
      const bool full = key0 >= full_lo && key0 + kPgTile <= full_hi;
      bool grew = false;
      float alpha[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sc[n][i] = (sc[n][i] + sd[n][i]) * a.scale_log2;
          if (!full) {
            const int key = key0 + g + (i >> 1) * 8, p = qp[n][i & 1];
            if (key > p || (a.win && key <= p - a.window)) sc[n][i] = -INFINITY;
          }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float mt = fmaxf(sc[n][j], sc[n][2 + j]);
          mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 4));
          mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 8));
          mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 16));
          const float m_new = fmaxf(m[n][j], mt);
          const float base = m_new == -INFINITY ? 0.f : m_new;
          alpha[n][j] = fast_exp2(m[n][j] - base);
          grew |= m_new != m[n][j];
          m[n][j] = m_new;
          sc[n][j] = fast_exp2(sc[n][j] - base);
          sc[n][2 + j] = fast_exp2(sc[n][2 + j] - base);
          lsum[n][j] = lsum[n][j] * alpha[n][j] + (sc[n][j] + sc[n][2 + j]);
        }
      }
      if (kB && __any_sync(0xffffffffu, grew)) {  // fp32 scales where it adds
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            o[n][i][0] *= alpha[n][0];
            o[n][i][1] *= alpha[n][1];
            o[n][i][2] *= alpha[n][0];
            o[n][i][3] *= alpha[n][1];
          }
      }
      const uint32_t vs = C::kPair ? ks + C::kTileBytes : next_place();
      // A tile that some rows attend to and others do not: a weight of 0 times a
      // value that is not finite would reach the others, so such values are
      // taken out and added below to the rows that attend to them.
      bool patch = false;
      if (!full) {
#pragma unroll 1
        for (int i = 0; i < C::kTileBytes / 512; ++i) {
          uint4 v;
          const uint32_t at = vs + (i * 32 + lane) * 16;
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
          if (pg_clean<T>(v)) {
            patch = true;
            asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
          }
        }
        patch = __any_sync(0xffffffffu, patch);
        __syncwarp();
      }
      // ---- O^T += V^T P^T --------------------------------------------------------------
      if constexpr (kB) {
        uint32_t pb[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          pb[n][0] = pg_transpose(pg_pack_bf16(sc[n][0], sc[n][1]));
          pb[n][1] = pg_transpose(pg_pack_bf16(sc[n][2], sc[n][3]));
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          uint32_t va[4];
          pg_ldsm4t(va, vs + pg_piece<T, HD>((lane & 7) + ((lane >> 4) << 3), 2 * i + ((lane >> 3) & 1)));
#pragma unroll
          for (int n = 0; n < NT; ++n) pg_mma_bf16(o[n][i], va, pb[n][0], pb[n][1]);
        }
      } else {
        uint32_t bh[2][NT][2], bl[2][NT][2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              // P[key 8 kb + 4 j + t4][row g] sits in lane 4 * (4 j + t4) + g / 2
              const int src = 4 * (4 * j + t4) + (g >> 1);
              const float p0 = __shfl_sync(0xffffffffu, sc[n][2 * kb], src);
              const float p1 = __shfl_sync(0xffffffffu, sc[n][2 * kb + 1], src);
              pg_split(g & 1 ? p1 : p0, bh[kb][n][j], bl[kb][n][j]);
            }
#pragma unroll
        for (int i = 0; i < MT; i += 2) {
          float c0[NT][4], c1[NT][4];
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) c0[n][e] = c1[n][e] = 0.f;
#pragma unroll
          for (int kb = 0; kb < 2; ++kb) {
            float4 x, y;  // values 16 i + 4 g .. + 3 of keys 8 kb + t4 and 8 kb + 4 + t4
            const uint32_t ax = vs + pg_piece<T, HD>(8 * kb + t4, 4 * i + g), ay = vs + pg_piece<T, HD>(8 * kb + 4 + t4, 4 * i + g);
            asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(ax));
            asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(y.x), "=f"(y.y), "=f"(y.z), "=f"(y.w) : "r"(ay));
            uint32_t hi[4], lo[4];
            pg_split(x.x, hi[0], lo[0]);
            pg_split(x.y, hi[1], lo[1]);
            pg_split(y.x, hi[2], lo[2]);
            pg_split(y.y, hi[3], lo[3]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              pg_mma_tf32(c0[n], lo, bh[kb][n][0], bh[kb][n][1]);
              pg_mma_tf32(c0[n], hi, bl[kb][n][0], bl[kb][n][1]);
              pg_mma_tf32(c0[n], hi, bh[kb][n][0], bh[kb][n][1]);
            }
            pg_split(x.z, hi[0], lo[0]);
            pg_split(x.w, hi[1], lo[1]);
            pg_split(y.z, hi[2], lo[2]);
            pg_split(y.w, hi[3], lo[3]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              pg_mma_tf32(c1[n], lo, bh[kb][n][0], bh[kb][n][1]);
              pg_mma_tf32(c1[n], hi, bl[kb][n][0], bl[kb][n][1]);
              pg_mma_tf32(c1[n], hi, bh[kb][n][0], bh[kb][n][1]);
            }
          }
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              o[n][i][e] = o[n][i][e] * alpha[n][e & 1] + c0[n][e];
              o[n][i + 1][e] = o[n][i + 1][e] * alpha[n][e & 1] + c1[n][e];
            }
        }
      }
      if (patch) {
#pragma unroll 1
        for (int key = max(key0, key_lo); key < min(key0 + kPgTile, key_hi); ++key) {
          const T* vr = kbase + a.v_off + (long long)tables[tbl + (key >> a.shift)] * a.page_elems + kvh * head_elems +
                        (long long)(key & ((1 << a.shift) - 1)) * HD;
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float v = pg_f32(vr[kB ? 16 * i + 8 * e + g : 32 * (i / 2) + 4 * g + 2 * (i & 1) + e]);
              if (!pg_finite(v))
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                  for (int j = 0; j < 2; ++j)
                    if (key <= qp[n][j] && !(a.win && key <= qp[n][j] - a.window)) o[n][i][2 * e + j] += v;
            }
        }
      }
    }

    // ---- merge of the CTA's warps -----------------------------------------------------
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float x = lsum[n][j];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        if (g == 0) {
          float* d = s_ml + ((warp * NT + n) * 8 + 2 * t4 + j) * 2;
          d[0] = m[n][j];
          d[1] = x;
        }
      }
    __syncthreads();
    const bool split = sg.n_parts > 1;
    const int part = sg.part, n_parts = sg.n_parts, cta0 = sg.cta0;
    const long long slot = part == 0 ? 2 * cta0 + 1 : 2 * (cta0 + part);
    T* out = static_cast<T*>(a.out);
    auto out_row = [&](int row) {  // output address of row `row` of the segment
      const int r = r0 + row;
      return out + (long long)(q_row0 + r / a.G) * a.out_stride + (long long)(kvh * a.G + r % a.G) * HD;
    };
    auto store4 = [&](int row, int d, float4 v) {
      if constexpr (kB)
        *reinterpret_cast<uint2*>(out_row(row) + d) = make_uint2(pg_pack_bf16(v.x, v.y), pg_pack_bf16(v.z, v.w));
      else
        *reinterpret_cast<float4*>(out_row(row) + d) = v;
    };
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (n * 8 < n_rows) {
        float f[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float M = -INFINITY;
#pragma unroll
          for (int w = 0; w < NW; ++w) M = fmaxf(M, s_ml[((w * NT + n) * 8 + 2 * t4 + j) * 2]);
          f[j] = m[n][j] == -INFINITY ? 0.f : fast_exp2(m[n][j] - M);
        }
        // row r of this warp's block at r * HD, 8-value groups of it flipped by r / 2: no two lanes of a store share a bank
        float* mb = merge + warp * 8 * HD;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int d = (kB ? 16 * i + 8 * e + g : 32 * (i / 2) + 4 * g + 2 * (i & 1) + e) ^ (t4 << 3);
            mb[(2 * t4) * HD + d] = o[n][i][2 * e] * f[0];
            mb[(2 * t4 + 1) * HD + d] = o[n][i][2 * e + 1] * f[1];
          }
      }
      __syncthreads();
      for (int x = tid; x < 8 * (HD / 4); x += NW * 32) {
        const int r = x / (HD / 4), d = (x % (HD / 4)) * 4, row = n * 8 + r;
        if (row >= n_rows) break;
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) M = fmaxf(M, s_ml[((w * NT + n) * 8 + r) * 2]);
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          const float mw = s_ml[((w * NT + n) * 8 + r) * 2];
          L += s_ml[((w * NT + n) * 8 + r) * 2 + 1] * (mw == -INFINITY ? 0.f : fast_exp2(mw - M));
          const float4 v = lds128(merge + w * 8 * HD + r * HD + (d ^ ((r >> 1) << 3)));
          s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
        }
        if (split) {
          *reinterpret_cast<float4*>(a.ws_o + (slot * 8 * NT + row) * HD + d) = s;
          if (d == 0) *reinterpret_cast<float2*>(a.ws_ml + (slot * 8 * NT + row) * 2) = make_float2(M, L);
        } else {
          const float inv = 1.f / L;
          store4(row, d, make_float4(s.x * inv, s.y * inv, s.z * inv, s.w * inv));
        }
      }
      __syncthreads();
    }
    if (split) {
      __syncthreads();
      if (tid == 0) {
        __threadfence();  // the CTA's partial rows, ahead of its ticket
        s_last = atomicAdd(a.tickets + cta0, 1u) == (unsigned)n_parts - 1;
        __threadfence();
      }
      __syncthreads();
      if (s_last) {
        if (tid == 0) a.tickets[cta0] = 0;
        auto part_slot = [&](int p) -> long long { return p == 0 ? 2 * cta0 + 1 : 2 * (cta0 + p); };
        // weights of the parts for every row, 1/L folded in: [row][part].  A warp's rows together, so that their loads overlap.
        constexpr int RW = 8 * NT / NW;
        float M[RW], L[RW];
#pragma unroll
        for (int i = 0; i < RW; ++i) M[i] = -INFINITY, L[i] = 0.f;
        for (int p = lane; p < n_parts; p += 32) {
          float2 ml[RW];
#pragma unroll
          for (int i = 0; i < RW; ++i)
            ml[i] = __ldcg(reinterpret_cast<const float2*>(a.ws_ml + (part_slot(p) * 8 * NT + min(warp + i * NW, n_rows - 1)) * 2));
#pragma unroll
          for (int i = 0; i < RW; ++i) {
            const float m1 = fmaxf(M[i], ml[i].x), base = m1 == -INFINITY ? 0.f : m1;
            L[i] = L[i] * fast_exp2(M[i] - base) + ml[i].y * fast_exp2(ml[i].x - base);
            M[i] = m1;
            if (warp + i * NW < n_rows) merge[(warp + i * NW) * n_parts + p] = ml[i].x;
          }
        }
#pragma unroll
        for (int i = 0; i < RW; ++i) {
#pragma unroll
          for (int x = 16; x > 0; x >>= 1) {
            const float m2 = __shfl_xor_sync(0xffffffffu, M[i], x), l2 = __shfl_xor_sync(0xffffffffu, L[i], x);
            const float m1 = fmaxf(M[i], m2), base = m1 == -INFINITY ? 0.f : m1;
            L[i] = L[i] * fast_exp2(M[i] - base) + l2 * fast_exp2(m2 - base);
            M[i] = m1;
          }
          const float inv = 1.f / L[i], base = M[i] == -INFINITY ? 0.f : M[i];
          if (warp + i * NW < n_rows)
            for (int p = lane; p < n_parts; p += 32) {
              float* w = merge + (warp + i * NW) * n_parts + p;
              *w = fast_exp2(*w - base) * inv;
            }
        }
        __syncthreads();
        constexpr int U = 4;  // pieces of a thread in flight
        const int pieces = n_rows * (HD / 4);
        for (int x0 = tid; x0 < pieces; x0 += U * NW * 32) {
          float4 s[U];
          int row[U], d[U];
#pragma unroll
          for (int i = 0; i < U; ++i) {
            const int x = min(x0 + i * NW * 32, pieces - 1);
            row[i] = x / (HD / 4), d[i] = (x % (HD / 4)) * 4;
            s[i] = make_float4(0.f, 0.f, 0.f, 0.f);
          }
#pragma unroll 4
          for (int p = 0; p < n_parts; ++p) {
            const float* base = a.ws_o + part_slot(p) * 8 * NT * HD;
            float4 v[U];
#pragma unroll
            for (int i = 0; i < U; ++i) v[i] = __ldcg(reinterpret_cast<const float4*>(base + row[i] * HD + d[i]));
#pragma unroll
            for (int i = 0; i < U; ++i) {
              const float w = merge[row[i] * n_parts + p];
              s[i].x += w * v[i].x, s[i].y += w * v[i].y, s[i].z += w * v[i].z, s[i].w += w * v[i].w;
            }
          }
#pragma unroll
          for (int i = 0; i < U; ++i)
            if (x0 + i * NW * 32 < pieces) store4(row[i], d[i], s[i]);
        }
      }
      __syncthreads();  // the merge buffer is free again
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (a.late) griddep_wait();
}

}  // namespace l3p

// paged_f32.cuh -- attention of many query rows per KV head over paged fp32
// keys and values on the tcgen05 tensor cores in 3xTF32 (sm_100a), head_dim 64
// or 128: chunks of prompts.
//
// Rows are (token, head of the group) pairs of one KV head as in paged_tc.cuh.
// The key tiles that the batch reads are first gathered from the pages and split
// into tf32 hi and lo images in the tensor cores' shared-memory layout
// (paged_prep_kernel; the layout is that of prefill_tc.cuh), once for all rows.
//
// Precision.  x = hi + lo with hi = x rounded to tf32; products are hi*hi +
// hi*lo + lo*hi (2^-22 of a product is dropped).  The tensor core cuts its
// accumulations off instead of rounding them: a chain of n MMAs loses about
// n/2 * 2^-24 of the sum, always towards zero (1.6e-5 of the last rows of a 2K
// prompt when O stays in one accumulator for all keys).  Therefore
//   * the small products (hi*lo, lo*hi) of S go in before the hi*hi ones, so
//     that only the latter meet a large accumulator;
//   * O is accumulated in registers: the MMAs of 64 keys form a partial sum in
//     tensor memory that an own warpgroup adds, in fp32 and rounded, to its row.
// That warpgroup also applies the running maximum's factors, so O is never
// rescaled in tensor memory.
//
// What bounds it: 6144 tensor-core cycles per 128 rows x 128 keys.
//
// CG = 2 (head_dim 128): the CTAs of a pair take 128 rows each of the same KV
// head; every MMA is cta_group::2 with M = 256, and each CTA stages half of
// every chunk.  CG = 1 for head_dim 64.
// Roles (512 threads per CTA): warps 0, 2 load chunks in turn (1-D bulk copies);
// warp 1 issues S (the odd CTA's relays landed chunks), warp 3 issues P V; warps
// 4-7 and 8-11 are the softmax of a tile's first and last 64 keys, thread = row
// (one warpgroup for all 128 took 11K cycles a tile); warps 12-15 hold O, thread = row.
#pragma once
#include "paged_tc.cuh"
#include "prefill_tc.cuh"

namespace l3p {

// Ring of the chunk kernel: one stage less than PfCfg has, for the statically
// allocated shared memory.  At least one tile's K chunks are held at once.
template <int CG, int HD>
struct PgF32Cfg {
  static constexpr int kStages = PfCfg<CG, HD>::kStages - 1;
  static constexpr int kSmem = PfGeom<HD>::kQloBytes + kStages * PfCfg<CG, HD>::kStageBytes + 1024;
  static_assert(kStages >= PfGeom<HD>::kKChunks + 1 && kSmem <= 232448 - 6144, "shared memory");
};

struct PgF32Args {
  const int* batch;
  const float* q;
  float* out;
  long long q_stride, out_stride;
  const float* storage;   // the layer's K block of page 0, head 0
  long long page_elems, v_off;
  float* img;             // [head of the group of heads][n_prep] tile images
  int* flags;             // [head][n_prep][4]: 32 keys' V hold values that are not finite (0 in the image)
  int kvh0, n_kvh, n_kv;  // group of KV heads of this launch, of all
  int shift, G, win, window;
  PgLimits lim;
  float scale_log2;
  float* ws_o;            // [slot][CG * 128][HD]
  float* ws_ml;
  int* err;
};

__device__ __forceinline__ float pg_tf32(float x) { return __uint_as_float((__float_as_uint(x) + 0x1000u) & 0xFFFFE000u); }

// Tile images of the keys that the batch's chunks attend to.  grid (tiles, KV heads of the group, 4: 32 keys each), 256 threads.
template <int CG, int HD>
__global__ void paged_prep_kernel(const PgF32Args a) {
  using C = PfCfg<CG, HD>;
  using Gm = PfGeom<HD>;
  const PgHeader* h = reinterpret_cast<const PgHeader*>(a.batch);
  const PgLists l = h->lists[a.win];
  griddep_launch();
  griddep_wait();  // the new rows come from the kernel before this one; the images are still read by it
  if (!pg_fits(h, l, a.lim) || (int)blockIdx.x >= l.n_prep) return;
  const PgPrep p = reinterpret_cast<const PgPrep*>(a.batch + l.prep)[blockIdx.x];
  const int* table = a.batch + h->tbl + p.tbl;
  const long long slot = (long long)blockIdx.y * a.lim.n_prep + p.img;
  unsigned char* base = reinterpret_cast<unsigned char*>(a.img) + slot * Gm::kTileBytes;
  const long long head = (long long)(a.kvh0 + blockIdx.y) * ((long long)HD << a.shift);
  constexpr int kVRows = HD / CG;
  constexpr int kVBase = Gm::kKChunks * C::kKBytes;
  int bad = 0;
#pragma unroll 4
  for (int idx = threadIdx.x; idx < 32 * HD / 4; idx += 256) {
    const int key = blockIdx.z * 32 + idx / (HD / 4), c16 = idx % (HD / 4);
    const int pos = p.key0 + key;
    float4 k = make_float4(0.f, 0.f, 0.f, 0.f), v = k;
    if (pos < p.key_hi) {
      const float* src = a.storage + (long long)table[pos >> a.shift] * a.page_elems + head +
                         (long long)(pos & ((1 << a.shift) - 1)) * HD + 4 * c16;
      k = *reinterpret_cast<const float4*>(src);
      v = *reinterpret_cast<const float4*>(src + a.v_off);
      uint4 w = *reinterpret_cast<const uint4*>(&v);
      if (pg_clean<float>(w)) {
        bad = 1;
        v = *reinterpret_cast<const float4*>(&w);
      }
    }
    const float4 kh = make_float4(pg_tf32(k.x), pg_tf32(k.y), pg_tf32(k.z), pg_tf32(k.w));
    const float4 kl = make_float4(k.x - kh.x, k.y - kh.y, k.z - kh.z, k.w - kh.w);
    const float4 vh = make_float4(pg_tf32(v.x), pg_tf32(v.y), pg_tf32(v.z), pg_tf32(v.w));
    const float4 vl = make_float4(v.x - vh.x, v.y - vh.y, v.z - vh.z, v.w - vh.w);
    const int part = c16 & 7;
    const int kr = key / C::kRows, kk = key % C::kRows;
    const int kb = kr * C::kHalfTile + (c16 >> 3) * C::kKBytes + kk * 128 + ((part ^ (kk & 7)) << 4);
    *reinterpret_cast<float4*>(base + kb) = kh;
    *reinterpret_cast<float4*>(base + kb + C::kKBytes / 2) = kl;
    const int dim = 4 * c16, vr = dim / kVRows, atom = (dim % kVRows) >> 5;
    const int kv = key & 31, byte = part * 16;
    const int vb = vr * C::kHalfTile + kVBase + (key >> 5) * C::kVBytes + atom * 4096 + (kv >> 2) * 512 + (kv & 3) * 128 +
                   ((((byte >> 5) ^ (kv & 3)) << 5) | (byte & 31));
    *reinterpret_cast<float4*>(base + vb) = vh;
    *reinterpret_cast<float4*>(base + vb + C::kVBytes / 2) = vl;
  }
  bad = __syncthreads_or(bad);
  if (threadIdx.x == 0) a.flags[4 * slot + blockIdx.z] = bad;
}

// MMAs and commits as in tc.cuh, issued by the lane for which `leader` is set in code that the whole warp runs (see
// mma_bf16_ss).
template <int CG>
__device__ __forceinline__ void pg_tf32_ts(uint32_t leader, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
  if constexpr (CG == 2)
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::tf32 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc),
        "r"(leader)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::tf32 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc),
        "r"(leader)
        : "memory");
}
template <int CG>
__device__ __forceinline__ void pg_tf32_ss(uint32_t leader, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
  if constexpr (CG == 2)
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::tf32 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc),
        "r"(leader)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::tf32 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc),
        "r"(leader)
        : "memory");
}
template <int CG>
__device__ __forceinline__ void pg_commit_g(uint32_t leader, uint32_t bar_cluster_addr) {
  if constexpr (CG == 2)
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar_cluster_addr), "r"(leader)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar_cluster_addr), "r"(leader)
        : "memory");
}

// The two softmax warpgroups meet: whether `ok` holds in all of their threads.  A warp whose bounded wait gave up must not
// leave a loop in which the others meet it at a barrier, which has no bound: all of them leave on the same tile.
__device__ __forceinline__ bool pg_meet(bool ok) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbar.red.and.pred q, 2, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"((uint32_t)ok)
      : "memory");
  return all != 0;
}

template <int CG, int HD>
__global__ void __launch_bounds__(512, 1) paged_f32_kernel(const PgF32Args a) {
  using C = PfCfg<CG, HD>;
  using Gm = PfGeom<HD>;
  constexpr int S = PgF32Cfg<CG, HD>::kStages;
  extern __shared__ unsigned char f32_smem_raw[];
  __shared__ uint32_t s_tmem;
  __shared__ float s_alpha[2][128], s_m[128], s_l[2][128], s_max[2][2][128];
  // Chunks in a CTA (full) and in the pair's other one (peer), by tile number modulo 3, not by stage: S and O have waiters
  // of their own, which have not seen the other's chunk land in a stage before theirs, and a wait tells a phase from its
  // neighbours only.  A chunk of tile t + 3 is loaded after a release that follows both waiters' use of tile t.
  __shared__ __align__(8) uint64_t bar_kv_full[3 * Gm::kChunks], bar_kv_peer[3 * Gm::kChunks], bar_kv_empty[S];
  auto k_bar = [](int t, int ch) { return t % 3 * Gm::kKChunks + ch; };
  auto v_bar = [](int t, int ch) { return 3 * Gm::kKChunks + t % 3 * Gm::kVChunks + ch; };
  static_assert(S < 3 * Gm::kChunks / 2, "the reach of the ring");
  __shared__ __align__(8) uint64_t bar_s_full, bar_s_free, bar_p_full[2], bar_p_free[2][2];
  __shared__ __align__(8) uint64_t bar_o_full, bar_o_free, bar_q_ready, bar_sm_done, bar_alpha[2], bar_mma_idle[2];

  const PgHeader* hd = reinterpret_cast<const PgHeader*>(a.batch);
  const PgLists l = hd->lists[a.win];
  const bool rows_next = a.lim.with_rows && a.kvh0 + a.n_kvh == a.n_kv;
  if (!rows_next) griddep_launch();
  const bool fits = pg_fits(hd, l, a.lim);
  if (!fits || (int)blockIdx.x / CG >= l.n_tc) {
    griddep_wait();
    griddep_launch();
    if (!fits && blockIdx.x == 0 && threadIdx.x == 0) *reinterpret_cast<volatile int*>(a.err) = kErrBadArg;
    return;
  }
  const PgPart u = reinterpret_cast<const PgPart*>(a.batch + l.tc_parts)[blockIdx.x / CG];
  if (u.kvh < a.kvh0 || u.kvh >= a.kvh0 + a.n_kvh) {  // both CTAs of a pair
    griddep_wait();
    griddep_launch();
    return;
  }
  const int* table = a.batch + hd->tbl + u.tbl;
  unsigned char* qlo = (unsigned char*)(((uintptr_t)f32_smem_raw + 1023) & ~(uintptr_t)1023);
  unsigned char* ring = qlo + Gm::kQloBytes;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = CG == 2 ? cluster_ctarank() : 0;
  const int nt = u.tile1 - u.tile0;
  const long long img_slot = (long long)(u.kvh - a.kvh0) * a.lim.n_prep + u.img + u.tile0;

  if (warp == 0) {
    tc::tmem_alloc_g<CG>(&s_tmem, 512);
    tc::tmem_relinquish_g<CG>();
  }
  if (tid == 32) {
    for (int s = 0; s < 3 * Gm::kChunks; ++s) {
      mbar_init(&bar_kv_full[s], 1);
      mbar_init(&bar_kv_peer[s], 1);
    }
    for (int s = 0; s < S; ++s) mbar_init(&bar_kv_empty[s], 1);
    mbar_init(&bar_s_full, 1);
    mbar_init(&bar_s_free, 8 * CG);
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bar_p_full[b], 4 * CG);
      mbar_init(&bar_p_free[0][b], 1);
      mbar_init(&bar_p_free[1][b], 1);
      mbar_init(&bar_mma_idle[b], 1);
      mbar_init(&bar_alpha[b], 4);
    }
    mbar_init(&bar_o_full, 1);
    mbar_init(&bar_o_free, 4 * CG);
    mbar_init(&bar_q_ready, 8 * CG);
    mbar_init(&bar_sm_done, 8);
    fence_mbar_init();
  }
  tc::fence_before_sync();
  if constexpr (CG == 2)
    cluster_sync_all();
  else
    __syncthreads();
  tc::fence_after_sync();
  const uint32_t tm = s_tmem;
  griddep_wait();  // the images and q come from the kernels before this one
  if (rows_next) griddep_launch();  // the row kernel relies on that wait
  const uint32_t T_QHI = tm + 0, T_O = tm + HD, T_S = tm + 2 * HD, T_P = tm + 2 * HD + kPfBN;

  // Barriers that carry tensor memory, copies that have landed or room (not ordinary stores) between the CTAs of a pair are
  // used at their default scope: with .release.cluster / .acquire.cluster every arrive and poll is a memory barrier of
  // 300 to 1000 cycles, of which a tile has 40.
  auto wait = [&](uint64_t* bar, uint32_t parity) -> bool { return pg_wait(bar, parity, a.err); };
  auto arrive_issuer = [&](uint64_t* bar) {
    if constexpr (CG == 2)
      asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(mapa_shared(smem_addr(bar), 0)) : "memory");
    else
      mbar_arrive(bar);
  };
  auto commit_all = [&](uint32_t leader, uint64_t* bar) {
    pg_commit_g<CG>(leader, smem_addr(bar));
    if constexpr (CG == 2) pg_commit_g<CG>(leader, mapa_shared(smem_addr(bar), 1));
  };
  // row of this thread (softmax and O warpgroups); rows behind the last one compute what it computes
  const int row = (warp & 3) * 32 + lane;
  const int rr = (int)rank * 128 + row;
  const bool valid = rr < u.n_rows;
  const int r = u.r0 + min(rr, u.n_rows - 1);
  const int tok = r / a.G, head = u.kvh * a.G + r % a.G;
  const long long q_off = (long long)(u.q_row0 + tok) * a.q_stride + (long long)head * HD;
  const long long o_off = (long long)(u.q_row0 + tok) * a.out_stride + (long long)head * HD;
  const int qpos = u.pos0 + tok;
  const int kmin = a.win ? max(0, qpos - a.window + 1) : 0;
  const uint32_t lb = (uint32_t)((warp & 3) * 32) << 16;
  const bool any_row = (int)rank * 128 + (warp & 3) * 32 < u.n_rows;

  // registers: 512 x 128 at launch >= 128 x 56 + 256 x 120 + 128 x 208
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 0 || warp == 2) {
      // ---------------- producers: every second stage each ----------------
      if (lane == 0) {
        const int me = warp >> 1;
        const unsigned char* img = reinterpret_cast<const unsigned char*>(a.img) + img_slot * Gm::kTileBytes + rank * C::kHalfTile;
        int c = 0;
        bool ok = true;
        for (int n = 0; ok && n <= nt; ++n) {
          for (int part = 0; ok && part < 2; ++part) {
            const int t = n - part;
            if (t < 0 || t >= nt) continue;
            const int n_ch = part == 0 ? Gm::kKChunks : Gm::kVChunks;
            for (int ch = 0; ch < n_ch; ++ch, ++c) {
              const int s = c % S, use = c / S;
              if (s % kProducers != me) continue;  // a stage is always the same warp's, which has seen its last release
              if (use >= 1 && !wait(&bar_kv_empty[s], (uint32_t)((use - 1) & 1))) {
                ok = false;
                break;
              }
              const uint32_t bytes = part == 0 ? C::kKBytes : C::kVBytes;
              const long long off = part == 0 ? (long long)ch * C::kKBytes
                                              : (long long)Gm::kKChunks * C::kKBytes + (long long)ch * C::kVBytes;
              uint64_t* full = &bar_kv_full[part == 0 ? k_bar(t, ch) : v_bar(t, ch)];
              mbar_arrive_expect_tx(full, bytes);
              asm volatile(
                  "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                      smem_addr(ring + s * C::kStageBytes)),
                  "l"(img + (long long)t * Gm::kTileBytes + off), "r"(bytes), "r"(smem_addr(full))
                  : "memory");
            }
          }
        }
        // no copy of this thread may still be landing when the CTA ends
        const int n0 = max(0, c - S) / Gm::kChunks;  // K of tile n0 and V of the tile before are not later than the last S loads
        for (int n = n0, i = n0 == 0 ? 0 : n0 * Gm::kChunks - Gm::kVChunks; n <= nt && i < c; ++n)
          for (int part = 0; part < 2; ++part) {
            const int t = n - part, n_ch = part == 0 ? Gm::kKChunks : Gm::kVChunks;
            if (t < 0 || t >= nt) continue;
            for (int ch = 0; ch < n_ch; ++ch, ++i)
              if (i >= c - S && i < c && i % S % kProducers == me)
                wait(&bar_kv_full[part == 0 ? k_bar(t, ch) : v_bar(t, ch)], (uint32_t)((t / 3) & 1));
          }
      }
    } else if (warp == 1 && rank == 1) {
      if (lane == 0)  // relay: chunk landed here -> issuers
        for (int n = 0; n < 2 * nt; ++n) {  // K0 K1 V0 K2 V1 ...
          const bool v = n == 2 * nt - 1 || (n > 0 && (n & 1) == 0);
          const int t = !v ? (n + 1) / 2 : n == 2 * nt - 1 ? nt - 1 : n / 2 - 1, n_ch = v ? Gm::kVChunks : Gm::kKChunks;
          bool ok = true;
          for (int ch = 0; ok && ch < n_ch; ++ch) {
            const int b = v ? v_bar(t, ch) : k_bar(t, ch);
            ok = wait(&bar_kv_full[b], (uint32_t)((t / 3) & 1));
            if (ok) asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(mapa_shared(smem_addr(&bar_kv_peer[b]), 0)) : "memory");
          }
          if (!ok) break;
        }
    } else if (rank == 0) {
      // ---------------- MMA issuers: warp 1 S, warp 3 O ----------------
      constexpr int nK = Gm::kKChunks, nKV = Gm::kChunks;
      uint32_t leader;
      asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(leader));
      auto wait_all = [&](uint64_t* bar, uint32_t parity) { return (bool)__all_sync(0xffffffffu, wait(bar, parity)); };
      auto k_chunk0 = [&](int t) { return t == 0 ? 0 : nK + (t - 1) * nKV; };
      auto v_chunk0 = [&](int t) { return t + 1 < nt ? 2 * nK + t * nKV : nK + t * nKV; };
      auto chunk_ready = [&](int b, int t) -> bool {
        if (!wait_all(&bar_kv_full[b], (uint32_t)((t / 3) & 1))) return false;
        if (CG == 2 && !wait_all(&bar_kv_peer[b], (uint32_t)((t / 3) & 1))) return false;
        tc::fence_after_sync();
        return true;
      };
      auto stage = [&](int c) { return (uint32_t)((c % S) * C::kStageBytes); };
      bool ok = true;
      if (warp == 1) {
        constexpr uint32_t id_s = tc::idesc_tf32(kPfBM * CG, kPfBN, false);
        const uint64_t qlo_d = tc::sdesc_sw128(smem_addr(qlo), 16, 1024);
        const uint64_t k_d = tc::sdesc_sw128(smem_addr(ring), 16, 1024);
        ok = __all_sync(0xffffffffu, mbar_wait_bounded_cluster(&bar_q_ready, 0, a.err));
        tc::fence_after_sync();
        for (int t = 0; ok && t < nt; ++t) {
          if (t >= 1) {
            if (!(ok = wait_all(&bar_s_free, (uint32_t)((t - 1) & 1)))) break;
            tc::fence_after_sync();
          }
#pragma unroll 1
          for (int ch = 0; ch < nK; ++ch) {  // the small products
            if (!(ok = chunk_ready(k_bar(t, ch), t))) break;
            const uint64_t kh = desc_add(k_d, stage(k_chunk0(t) + ch)), kl = desc_add(kh, C::kStageBytes / 2);
            const uint64_t ql = desc_add(qlo_d, ch * 16384);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
              pg_tf32_ts<CG>(leader, T_S, T_QHI + ch * 32 + kk * 8, desc_add(kl, kk * 32), id_s, ch > 0 || kk > 0);
              pg_tf32_ss<CG>(leader, T_S, desc_add(ql, kk * 32), desc_add(kh, kk * 32), id_s, true);
            }
          }
          if (!ok) break;
#pragma unroll 1
          for (int ch = 0; ch < nK; ++ch) {  // hi * hi
            const uint64_t kh = desc_add(k_d, stage(k_chunk0(t) + ch));
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) pg_tf32_ts<CG>(leader, T_S, T_QHI + ch * 32 + kk * 8, desc_add(kh, kk * 32), id_s, true);
            commit_all(leader, &bar_kv_empty[(k_chunk0(t) + ch) % S]);
          }
          commit_all(leader, &bar_s_full);
        }
        pg_commit_g<CG>(leader, smem_addr(&bar_mma_idle[0]));
        wait(&bar_mma_idle[0], 0);
      } else {
        constexpr uint32_t id_o = tc::idesc_tf32(kPfBM * CG, HD, true);
        const uint64_t v_d = sdesc_mn_sw128_32b(smem_addr(ring));
        for (int t = 0; ok && t < nt; ++t) {
#pragma unroll 1
          for (int qq = 0; ok && qq < Gm::kVChunks; ++qq) {
            const int c = v_chunk0(t) + qq, slot = qq & 1;
            if (!(ok = chunk_ready(v_bar(t, qq), t))) break;
            // a new partial sum every 64 keys: the one before has been taken
            const int half = 2 * t + (qq >> 1);
            if (slot == 0 && half >= 1 && !(ok = wait_all(&bar_o_free, (uint32_t)((half - 1) & 1)))) break;
            if (!(ok = wait_all(&bar_p_full[slot], (uint32_t)((qq >> 1) & 1)))) break;
            tc::fence_after_sync();
            const uint64_t vh = desc_add(v_d, stage(c)), vl = desc_add(vh, C::kVBytes / 2);
            const uint32_t p_hi = T_P + slot * 64, p_lo = p_hi + 32;
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
              pg_tf32_ts<CG>(leader, T_O, p_hi + ks * 8, desc_add(vl, ks * 1024), id_o, slot > 0 || ks > 0);
              pg_tf32_ts<CG>(leader, T_O, p_lo + ks * 8, desc_add(vh, ks * 1024), id_o, true);
            }
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) pg_tf32_ts<CG>(leader, T_O, p_hi + ks * 8, desc_add(vh, ks * 1024), id_o, true);
            commit_all(leader, &bar_kv_empty[c % S]);
            commit_all(leader, &bar_p_free[qq >> 1][slot]);
            if (slot == 1) commit_all(leader, &bar_o_full);
          }
        }
        pg_commit_g<CG>(leader, smem_addr(&bar_mma_idle[1]));
        wait(&bar_mma_idle[1], 0);
      }
    }
  } else if (warp < 12) {
    // ---------------- softmax: thread = row and half of the tile's keys ----------------
    asm volatile("setmaxnreg.dec.sync.aligned.u32 120;");
    const int half = (warp - 4) >> 2;
    {
      // This half's 32-column chunks of the warp's 32 rows: whole 128-byte lines into the place of the Q lo image, then every
      // thread its row from there.
      float4 t[HD / 64][8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float* src = a.q + __shfl_sync(0xffffffffu, q_off, i * 4 + (lane >> 3)) + (lane & 7) * 4;
#pragma unroll
        for (int c = 0; c < HD / 64; ++c) t[c][i] = *reinterpret_cast<const float4*>(src + (2 * c + half) * 32);
      }
#pragma unroll
      for (int c = 0; c < HD / 64; ++c) {
        unsigned char* img = qlo + (2 * c + half) * 16384;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int x = (warp & 3) * 32 + i * 4 + (lane >> 3);
          *reinterpret_cast<float4*>(img + x * 128 + (((lane & 7) ^ (x & 7)) << 4)) = t[c][i];
        }
        __syncwarp();
        unsigned char* rp = img + row * 128;
        float hi[32], lo[32];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float4 y = *reinterpret_cast<const float4*>(rp + ((i ^ (row & 7)) << 4));
          hi[4 * i] = pg_tf32(y.x), lo[4 * i] = y.x - hi[4 * i];
          hi[4 * i + 1] = pg_tf32(y.y), lo[4 * i + 1] = y.y - hi[4 * i + 1];
          hi[4 * i + 2] = pg_tf32(y.z), lo[4 * i + 2] = y.z - hi[4 * i + 2];
          hi[4 * i + 3] = pg_tf32(y.w), lo[4 * i + 3] = y.w - hi[4 * i + 3];
        }
        tc::st32(T_QHI + lb + (2 * c + half) * 32, hi);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          *reinterpret_cast<float4*>(rp + ((i ^ (row & 7)) << 4)) = make_float4(lo[4 * i], lo[4 * i + 1], lo[4 * i + 2], lo[4 * i + 3]);
      }
      tc::wait_st();
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CG == 2)
          mbar_arrive_cluster(mapa_shared(smem_addr(&bar_q_ready), 0));  // ordinary stores: the image of Q lo
        else
          mbar_arrive(&bar_q_ready);
      }
    }
    float m = -INFINITY, lsum = 0.f;
    bool ok = true;
    for (int j = 0; j < nt; ++j) {
      ok = ok && __all_sync(0xffffffffu, wait(&bar_s_full, (uint32_t)(j & 1)));
      tc::fence_after_sync();
      if (!any_row) {  // lanes without a row: S, P and O as they come (MMA rows are independent)
        if (lane == 0 && ok) arrive_issuer(&bar_s_free);
        if (!(ok = pg_meet(ok))) break;
        if (half == 0 && lane == 0) mbar_arrive(&bar_alpha[j & 1]);
        for (int qq = 0; qq < 2; ++qq) {
          if (j >= 1 || half > 0) ok = ok && __all_sync(0xffffffffu, wait(&bar_p_free[half ^ 1][qq], (uint32_t)((half ? j : j - 1) & 1)));
          if (lane == 0 && ok) arrive_issuer(&bar_p_full[qq]);
        }
        continue;
      }
      float sv[64];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float t[32];
        tc::ld32(T_S + lb + half * 64 + c * 32, t);
#pragma unroll
        for (int i = 0; i < 32; ++i) sv[c * 32 + i] = t[i];
      }
      tc::wait_ld();
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0 && ok) arrive_issuer(&bar_s_free);
      const int key0 = (u.tile0 + j) * kPfBN + half * 64;
      if (!__all_sync(0xffffffffu, key0 >= kmin && key0 + 63 <= qpos)) {
        const int last = qpos - key0, from = kmin - key0;
#pragma unroll
        for (int c = 0; c < 64; ++c)
          if (c > last || c < from) sv[c] = -INFINITY;
      }
      float mx[4] = {sv[0], sv[1], sv[2], sv[3]};
#pragma unroll
      for (int c = 4; c < 60; c += 8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) mx[i] = max3(mx[i], sv[c + 2 * i], sv[c + 2 * i + 1]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) mx[i] = fmaxf(mx[i], sv[60 + i]);
      s_max[j & 1][half][row] = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      // both halves of a row meet here once a tile, whether their waits succeeded or not
      if (!(ok = pg_meet(ok))) break;
      const float m_new = fmaxf(m, fmaxf(s_max[j & 1][0][row], s_max[j & 1][1][row]) * a.scale_log2);
      const float base = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = fast_exp2(m - base);
      m = m_new;
      if (half == 0) {
        s_alpha[j & 1][row] = alpha;
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar_alpha[j & 1]);
      }
      lsum *= alpha;
#pragma unroll
      for (int qq = 0; qq < 2; ++qq) {
        float ph[32], pl[32], ls[2] = {0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          const float p = fast_exp2(fmaf(sv[qq * 32 + c], a.scale_log2, -base));
          ls[c & 1] += p;
          ph[c] = pg_tf32(p);
          pl[c] = p - ph[c];
        }
        lsum += ls[0] + ls[1];
        if (j >= 1 || half > 0) {
          // the slot's quarter before, the other half's, has been multiplied (a barrier for each half: of one that both
          // halves' quarters complete, a warpgroup could be two phases behind)
          ok = ok && __all_sync(0xffffffffu, wait(&bar_p_free[half ^ 1][qq], (uint32_t)((half ? j : j - 1) & 1)));
          tc::fence_after_sync();
        }
        tc::st32(T_P + lb + qq * 64, ph);
        tc::st32(T_P + lb + qq * 64 + 32, pl);
        tc::wait_st();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0 && ok) arrive_issuer(&bar_p_full[qq]);
      }
    }
    if (half == 0) s_m[row] = m;
    s_l[half][row] = lsum;
    __syncwarp();
    if (lane == 0) mbar_arrive(&bar_sm_done);
  } else {
    // ---------------- O: thread = row ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    float acc[HD];
#pragma unroll
    for (int i = 0; i < HD; ++i) acc[i] = 0.f;
    bool ok = true;
    for (int x = 0; ok && x < 2 * nt; ++x) {
      ok = __all_sync(0xffffffffu, wait(&bar_o_full, (uint32_t)(x & 1)));
      if (ok && !(x & 1)) ok = __all_sync(0xffffffffu, wait(&bar_alpha[(x >> 1) & 1], (uint32_t)((x >> 2) & 1)));
      if (!ok) break;
      tc::fence_after_sync();
      if (!any_row) {
        if (lane == 0) arrive_issuer(&bar_o_free);
        continue;
      }
      const float f = x & 1 ? 1.f : s_alpha[(x >> 1) & 1][row];
#pragma unroll
      for (int c = 0; c < HD / 32; ++c) {
        float ov[32];
        tc::ld32(T_O + lb + c * 32, ov);
        tc::wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) acc[c * 32 + i] = fmaf(acc[c * 32 + i], f, ov[i]);
      }
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) arrive_issuer(&bar_o_free);
    }
    if (ok) ok = __all_sync(0xffffffffu, wait(&bar_sm_done, 0));
    if (ok && any_row) {
      // values of V that are not finite, to the rows that attend to them
      const int* flags = a.flags + 4 * img_slot;
      for (int t = 0; t < nt; ++t) {
        const int4 f4 = reinterpret_cast<const int4*>(flags)[t];
        if ((f4.x | f4.y | f4.z | f4.w) == 0) continue;
        const int key0 = (u.tile0 + t) * kPfBN;
        for (int key = max(kmin, key0); key <= min(qpos, key0 + kPfBN - 1); ++key) {
          const float* v = a.storage + a.v_off + (long long)table[key >> a.shift] * a.page_elems +
                           ((long long)u.kvh << a.shift) * HD + (long long)(key & ((1 << a.shift) - 1)) * HD;
#pragma unroll
          for (int i = 0; i < HD; ++i) {
            const float y = v[i];
            if (!pg_finite(y)) acc[i] += y;
          }
        }
      }
      const float lsum = s_l[0][row] + s_l[1][row];
      // rows through the ring, which no MMA reads any more, so that the warp stores whole rows
      const bool split = u.n_parts > 1;
      const float inv = split ? 1.f : 1.f / lsum;
      unsigned char* buf = ring + (warp & 3) * (32 * HD * 4);
#pragma unroll
      for (int i = 0; i < HD / 4; ++i)
        *reinterpret_cast<float4*>(buf + lane * (HD * 4) + ((i ^ (lane & 7)) << 4)) =
            make_float4(acc[4 * i] * inv, acc[4 * i + 1] * inv, acc[4 * i + 2] * inv, acc[4 * i + 3] * inv);
      __syncwarp();
      const long long ws_row0 = (long long)(u.slot + u.part) * (CG * 128);
      if (split && valid) *reinterpret_cast<float2*>(a.ws_ml + (ws_row0 + rr) * 2) = make_float2(s_m[row], lsum);
      constexpr int kPieces = HD / 4, kRows = 32 / kPieces > 0 ? 32 / kPieces : 1;  // rows a warp stores at once
#pragma unroll 4
      for (int x = 0; x < 32 / kRows; ++x) {
        const int y = x * kRows + lane / kPieces, pc = lane % kPieces;
        const int yr = (int)rank * 128 + (warp & 3) * 32 + y;
        const long long off = __shfl_sync(0xffffffffu, o_off, y);
        float* dst = split ? a.ws_o + (ws_row0 + yr) * HD : a.out + off;
        if (yr < u.n_rows)
          *reinterpret_cast<float4*>(dst + 4 * pc) = *reinterpret_cast<const float4*>(buf + y * (HD * 4) + ((pc ^ (y & 7)) << 4));
      }
    }
  }
  tc::fence_before_sync();
  if constexpr (CG == 2)
    cluster_sync_all();
  else
    __syncthreads();
  if (warp == 0) {
    tc::fence_after_sync();
    tc::tmem_dealloc_g<CG>(tm, 512);
  }
}

}  // namespace l3p

// paged_tc.cuh -- attention of many query rows per KV head over paged bf16
// keys and values on the tcgen05 tensor cores (sm_100a): chunks of prompts.
//
// Rows.  The query heads of a KV head's group and the chunk's tokens are one
// axis of rows (row r: token r / G, head r % G of the group), so a 128-row MMA
// is full for any group size, and every K/V tile serves the whole group.  One
// CTA takes 256 rows (two Q tiles; one of 128 for head_dim 256) and a run of
// key tiles of 128 (64) keys.
//
// S = Q K^T and O += P V accumulate in tensor memory in fp32.  Softmax is
// online, in fp32, thread = row; P is rounded to bf16 for the second product
// (at most 2^-8 of each weight; l sums the unrounded P) and takes the place of
// the S it came from.  O is rescaled only when a row's maximum grew by more
// than 2^8 since its reference was set; the reference is exact, so this
// changes no result but by rounding.
//
// What bounds it: for head_dim 128 the MMAs of a key tile and both Q tiles take
// 2048 cycles, and so do its 32K exponentials at 16 a cycle; with the rest of
// softmax and its hand-over to the tensor core it is 3.8K cycles (four chunks of
// 2K tokens on up to 8K keys: 960 TFLOP/s).  Two Q tiles in turn keep the tensor core
// on one while the other's softmax runs.  Up to 128 rows: the loads, 4.8 TB/s.
//
// Tiles come from the pages by TMA, one box per page (or 128-key tile) and 64
// columns, into a ring in consumption order K0 V0 K1 V1 ..., 128-byte swizzled:
// K is the K-major B operand of S, V the MN-major B operand of O.
//
// Roles: warps 0 and 3 load K and V; warp 1 issues MMAs; warp 2, of the last tiles with
// warp 3, checks V tiles that some row does not attend to entirely (masked weights are 0, and 0 times a value that
// is not finite is NaN: rows outside every window become 0, such values are
// taken out and added in the epilogue to the rows that attend to them); warps
// 4-7 and 8-11 are the softmax of Q tile 0 and 1.
//
// Long key ranges with few rows are cut into parts (plan_tc), which
// paged_merge_kernel joins.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>

#include "paged_rows.cuh"
#include "tc.cuh"

namespace l3p {

template <int HD>
struct PgTcCfg {
  static constexpr int kNQ = HD == 256 ? 1 : 2;     // Q tiles of 128 rows
  static constexpr int kTN = HD == 256 ? 64 : 128;  // keys of a tile
  static constexpr int kQBytes = kNQ * 128 * HD * 2;
  static constexpr int kStage = kTN * HD * 2;
  static constexpr int kStages = HD == 64 ? 8 : 5;
  static constexpr int kSmem = kQBytes + kStages * kStage + 1024;
  static constexpr int kThreads = 128 + kNQ * 128;
  // tensor memory columns: S (and P in its place), then O
  static constexpr int kS = HD == 256 ? 64 : 128;
  static constexpr int kO = 256;
  static constexpr int kHands = HD == 256 ? 1 : 2;  // parts in which a tile's P is handed to the second product
  static_assert(kSmem <= 232448 - 1536, "shared memory");
};

struct PgTcArgs {
  const int* batch;
  const void* q;
  void* out;
  long long q_stride, out_stride;
  const __nv_bfloat16* storage;  // page 0
  long long page_elems;
  int row_k;       // storage row of (page 0, layer, K, head 0, slot 0)
  int page_rows;   // storage rows of a page
  int n_kv, shift, G, win, window;
  PgLimits lim;
  float scale_log2;
  float* ws_o;     // [slot][kNQ * 128][HD]
  float* ws_ml;    // [slot][kNQ * 128][2]
  int* err;
};

// mbar_wait_bounded with a limit of about a second: no wait inside one GPU
// takes longer than the kernel's own milliseconds.
__device__ __forceinline__ bool pg_wait(uint64_t* bar, uint32_t parity, int* err) {
  for (uint32_t i = 0; i < (1u << 18); ++i)
    if (mbar_try_wait(bar, parity)) return true;
  *reinterpret_cast<volatile int*>(err) = kErrTimeout;
  return false;
}

__host__ __device__ constexpr uint32_t idesc_bf16(int M, int N, bool b_mn_major) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
// Issued by the lane for which `leader` is set, in code that the whole warp runs:
// outside divergent code the descriptors stay in uniform registers (an issue
// costs a lone thread ~85 cycles, 16 of which a tile has no time for).
__device__ __forceinline__ void mma_bf16_ss(uint32_t leader, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc),
      "r"(leader)
      : "memory");
}
__device__ __forceinline__ void mma_bf16_ts(uint32_t leader, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc),
      "r"(leader)
      : "memory");
}
__device__ __forceinline__ void pg_commit(uint32_t leader, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_addr(bar)), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void pg_tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(smem_addr(bar))
      : "memory");
}
__device__ __forceinline__ void tmem_st32u(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]),
      "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]),
      "r"(v[31])
      : "memory");
}

// ---- two fp32 values in one 64-bit register: half the issue slots
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pk2(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void un2(f32x2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Joins the parts of split units: row = sum_p w_p o_p / sum_p w_p l_p with
// w_p = 2^(m_p - max m), in part order.  One warp per row, a lane holds HD/32
// values; a kernel of its own because the last of the parts' CTAs, alone on its SM,
// took 50 us for what all SMs do in 3.  grid (units, rows / 8).
template <typename T, int HD>
__global__ void __launch_bounds__(256) paged_merge_kernel(const int* batch, int win, PgLimits lim, int rows, const float* __restrict__ ws_o,
                                                          const float* __restrict__ ws_ml, T* out, long long out_stride, int G) {
  constexpr int N = HD / 32;
  const PgHeader* h = reinterpret_cast<const PgHeader*>(batch);
  const PgLists& l = h->lists[win];
  const int lane = threadIdx.x & 31, row = blockIdx.y * 8 + (threadIdx.x >> 5);
  griddep_launch();
  griddep_wait();
  if (!pg_fits(h, l, lim) || (int)blockIdx.x >= l.n_merge) return;
  const PgPart u = reinterpret_cast<const PgPart*>(batch + l.merges)[blockIdx.x];
  if (row >= u.n_rows) return;
  const float2* ml = reinterpret_cast<const float2*>(ws_ml) + (long long)u.slot * rows + row;
  const float* o = ws_o + ((long long)u.slot * rows + row) * HD + lane * N;
  float M = -INFINITY;
  for (int p = lane; p < u.n_parts; p += 32) M = fmaxf(M, __ldcg(ml + (long long)p * rows).x);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
  const float base = M == -INFINITY ? 0.f : M;
  float acc[N], L = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.f;
#pragma unroll 8
  for (int p = 0; p < u.n_parts; ++p) {
    const float2 t = __ldcg(ml + (long long)p * rows);
    const float* src = o + (long long)p * rows * HD;
    float v[N];
    if constexpr (N == 2) {
      const float2 y = __ldcg(reinterpret_cast<const float2*>(src));
      v[0] = y.x, v[1] = y.y;
    } else {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const float4 y = __ldcg(reinterpret_cast<const float4*>(src + i));
        v[i] = y.x, v[i + 1] = y.y, v[i + 2] = y.z, v[i + 3] = y.w;
      }
    }
    const float w = fast_exp2(t.x - base);
    L += w * t.y;
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] += w * v[i];
  }
  const float inv = 1.f / L;
  const int r = u.r0 + row;
  T* dst = out + (long long)(u.q_row0 + r / G) * out_stride + (long long)(u.kvh * G + r % G) * HD + lane * N;
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    if constexpr (sizeof(T) == 2)
      *reinterpret_cast<uint32_t*>(dst + i) = pg_pack_bf16(acc[i] * inv, acc[i + 1] * inv);
    else
      *reinterpret_cast<float2*>(dst + i) = make_float2(acc[i] * inv, acc[i + 1] * inv);
  }
}

template <int HD>
__global__ void __launch_bounds__(PgTcCfg<HD>::kThreads, 1)
    paged_tc_kernel(const PgTcArgs a, const __grid_constant__ CUtensorMap tmap) {
  using C = PgTcCfg<HD>;
  constexpr int S = C::kStages, TN = C::kTN, NQ = C::kNQ;
  extern __shared__ unsigned char tc_smem_raw[];
  __shared__ uint32_t s_tmem;
  __shared__ int s_bad;
  __shared__ float s_m1[128], s_l1[128];
  __shared__ __align__(8) uint64_t k_full[S], v_full[S], v_ok[S], kv_empty[S + 2];
  __shared__ __align__(8) uint64_t s_full[2], p_full[2][2], o_done[2], q_ready[2], mma_idle;

  const PgHeader* h = reinterpret_cast<const PgHeader*>(a.batch);
  const PgLists l = h->lists[a.win];
  if (!a.lim.with_rows) griddep_launch();
  if (!pg_fits(h, l, a.lim) || (int)blockIdx.x >= l.n_tc) {
    griddep_wait();
    griddep_launch();
    if (!pg_fits(h, l, a.lim) && blockIdx.x == 0 && threadIdx.x == 0) *reinterpret_cast<volatile int*>(a.err) = kErrBadArg;
    return;
  }
  const PgPart u = reinterpret_cast<const PgPart*>(a.batch + l.tc_parts)[blockIdx.x];
  const int* table = a.batch + h->tbl + u.tbl;
  unsigned char* sq = (unsigned char*)(((uintptr_t)tc_smem_raw + 1023) & ~(uintptr_t)1023);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int nt = u.tile1 - u.tile0;
  // Two streams of key tiles: one per Q tile, each over all key tiles; or, for up to 128 rows, both for the one Q tile,
  // over the even and the odd key tiles, joined at the end.
  const bool dual = NQ == 2 && u.n_rows <= 128;
  const int nq = NQ == 2 && (!dual || nt > 1) ? 2 : 1;
  // The ring, in the order of use: K0 V0 K1 V1 ... or, with two streams of tiles, K0 K1 V0 K2 V1 K3 ...; then the second Q
  // tile's place is part of it.  Nearly all of it is in flight at any time, which is what HBM needs: ~19 MB over the GPU
  // for its full rate.
  constexpr int kMore = NQ == 2 ? 128 * HD * 2 / C::kStage : 0;  // stages in a Q tile's place
  static_assert(kMore <= 2, "barriers");
  unsigned char* ring = sq + C::kQBytes - (dual ? kMore * C::kStage : 0);
  auto stage_of = [&](int t) { return dual ? t % (S + kMore) : t % S; };
  auto k_at = [&](int j) { return dual ? (j < 2 ? j : 2 * j - 1) : 2 * j; };             // position of K tile j in the ring's order
  auto v_at = [&](int j) { return dual ? min(2 * j + 2, 2 * nt - 1) : 2 * j + 1; };      // and of V tile j
  const int first_pos = u.pos0 + u.r0 / a.G, last_pos = u.pos0 + (u.r0 + u.n_rows - 1) / a.G;
  const int lo_first = a.win ? max(0, first_pos - a.window + 1) : 0;  // keys below: no row attends to them
  const int lo_last = a.win ? max(0, last_pos - a.window + 1) : 0;    // keys from here to first_pos: every row does

  // Barriers.  A wait tells one phase from its neighbours only, so a barrier's phases follow what its waiter has seen:
  // k_full, v_full and v_ok are by the tile's number (the stage alternates between K and V in most rings, and the
  // waiter for one has not seen the other land), kv_empty by stage, in about whose order stages are released.
  if (warp == 0) {
    tc::tmem_alloc(&s_tmem, 512);
    tc::tmem_relinquish();
  }
  if (tid == 32) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_ok[s], 2);
    }
    for (int s = 0; s < S + 2; ++s) mbar_init(&kv_empty[s], 1);
    for (int b = 0; b < 2; ++b) {
      mbar_init(&s_full[b], 1);
      mbar_init(&p_full[b][0], 4);
      mbar_init(&p_full[b][1], 4);
      mbar_init(&o_done[b], 1);
      mbar_init(&q_ready[b], 4);
    }
    mbar_init(&mma_idle, 1);
    s_bad = 0;
    fence_mbar_init();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tm = s_tmem;
  griddep_wait();  // q and the new rows come from the kernel before this one
  if (a.lim.with_rows) griddep_launch();  // the row kernel relies on that wait

  // Registers: 384 x 168 at launch = 128 x 88 + 256 x 208.  Inside the branches: behind their join the compiler would
  // count with the smaller number.
  if (warp < 4) {
  bool loaded = true;
  if (NQ == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
  if (warp == 0 || warp == 3) {
    // ---------------- loads: warp 0 K, warp 3 V ----------------
    // Few instructions a load: the softmax warps want the issue slots, and at 16 or 32 positions a page these loads bound
    // the kernel (16 sequences x 9 tokens x 3000 keys, 8B heads, pages of 16: 49.5 us with stages and tiles found by
    // division from the load's number, 44.0 us with running counters and a page looked up a tile ahead, 41.1 us with a warp
    // for K and one for V, 42.5 us since barriers go by the tile's number).  A load waits for the release one ring earlier, and the warp's load before it has waited for a
    // later release than the one two rings earlier: one phase.
    const bool is_v = warp == 3;
    const int box = min(1 << a.shift, TN), n_box = TN / box;  // keys of a box, boxes down a tile
    const int i = lane % n_box, c = lane / n_box;             // this lane's box and column block
    const int n_stage = dual ? S + kMore : S, in_page = (1 << a.shift) - 1;
    const int base = a.row_k + ((u.kvh + (is_v ? a.n_kv : 0)) << a.shift);
    const uint32_t to = smem_addr(ring) + c * (TN * 128) + i * (box * 128);
    const int key_end = c < HD / 64 ? u.key_hi : 0;
    auto at = [&](int j) { return is_v ? v_at(j) : k_at(j); };
    int key = u.tile0 * TN + i * box;  // this lane's first key of tile j
    int page = key < key_end ? table[key >> a.shift] : 0;
    uint64_t* fulls = is_v ? v_full : k_full;
    int s = at(0), n_used = 0, fb = 0;
    uint32_t free_parity = 1;  // of a stage's last release; at first no stage has to be waited for
    while (n_used < nt) {
      const bool mine = key < key_end;
      const int row = page * a.page_rows + base + (key & in_page);
      key += TN;
      page = key < key_end ? table[key >> a.shift] : 0;
      if (!__all_sync(0xffffffffu, pg_wait(&kv_empty[s], free_parity, a.err))) break;
      const int n = __popc(__ballot_sync(0xffffffffu, mine));
      uint64_t* full = fulls + fb;
      if (lane == 0) mbar_arrive_expect_tx(full, (uint32_t)(n * box * 128));
      __syncwarp();
      if (mine) pg_tma_2d(to + s * C::kStage, &tmap, c * 64, row, full);
      ++n_used;
      if (++fb == S) fb = 0;
      s += dual && n_used == (is_v ? nt - 1 : 1) ? 1 : 2;  // the next one's place in the order of use
      if (s >= n_stage) s -= n_stage, free_parity ^= 1;
    }
    loaded = n_used == nt;
    // no copy may still be landing when the CTA ends (of V, warp 3 waits for the last three tiles below; the ones before had
    // landed when it could load the last)
    if (!is_v || !loaded)
      for (int j = max(0, n_used - S); j < n_used; ++j) pg_wait(&fulls[j % S], (uint32_t)(j / S & 1), a.err);
  } else if (warp == 1) {
    // ---------------- MMA issue ----------------
    constexpr uint32_t id_s = idesc_bf16(128, TN, false), id_o = idesc_bf16(128, HD, true);
    uint32_t leader;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(leader));
    const uint64_t q_d = tc::sdesc_sw128(smem_addr(sq), 16, 1024);
    const uint64_t k_d = tc::sdesc_sw128(smem_addr(ring), 16, 1024);
    const uint64_t v_d = tc::sdesc_sw128(smem_addr(ring), TN * 128, 1024);
    auto qk = [&](int b, int slot, int stage) {  // S[slot] = Q[b] K^T
      const uint64_t kd = k_d + (uint64_t)((stage * C::kStage) >> 4), qd = q_d + (uint64_t)(b * (128 * HD * 2) >> 4);
#pragma unroll
      for (int k = 0; k < HD / 16; ++k)
        mma_bf16_ss(leader, tm + slot * C::kS, qd + (((k / 4) * 16384 + (k % 4) * 32) >> 4),
                    kd + (((k / 4) * (TN * 128) + (k % 4) * 32) >> 4), id_s, k > 0);
    };
    auto pv = [&](int b, int slot, int stage, int hf, bool acc) {  // O[b] += P[slot] V, the part's keys
      const uint64_t vd = v_d + (uint64_t)((stage * C::kStage) >> 4);
#pragma unroll
      for (int k = hf * (TN / 16 / C::kHands); k < (hf + 1) * (TN / 16 / C::kHands); ++k)
        mma_bf16_ts(leader, tm + C::kO + b * HD, tm + slot * C::kS + k * 8, vd + (k * 2048 >> 4), id_o, acc || k > 0);
    };
    auto wait = [&](uint64_t* bar, int phase) {
      const bool r = __all_sync(0xffffffffu, pg_wait(bar, (uint32_t)(phase & 1), a.err));
      tc::fence_after_sync();
      return r;
    };
    bool ok = true;
    // running numbers instead of divisions (16 sequences x 9 tokens x 3000 keys, head_dim 64: 29.3 -> 26.8 us; now 27.9): V tile j's and
    // the next K tile's barriers, phases and stages
    int vb = 0, vp = 0, kb = 0, kp = 0;
    auto next_v = [&] { if (++vb == S) vb = 0, vp ^= 1; };
    auto next_k = [&] { if (++kb == S) kb = 0, kp ^= 1; };
    auto step = [&](int x, int by, int n) { return x + by >= n ? x + by - n : x + by; };
    if (dual) {
      // stream b = j & 1: O += P V of key tile j, then S of key tile j + 2
      constexpr int n = S + kMore;
      int sv = stage_of(v_at(0)), sk = 0;
      ok = wait(&q_ready[0], 0);
      for (int j = -2; ok && j < nt; ++j) {
        const int b = j & 1;
        const bool next = j + 2 < nt;
        if (j >= 0) {
          if (!(ok = wait(&v_ok[vb], vp))) break;
          next_v();
#pragma unroll
          for (int hf = 0; hf < C::kHands; ++hf) {
            if (!(ok = ok && wait(&p_full[b][hf], j >> 1))) break;
            pv(b, b, sv, hf, j > 1);
          }
          if (!ok) break;
          pg_commit(leader, &kv_empty[sv]);
          pg_commit(leader, &o_done[b]);
          sv = step(sv, j + 2 == nt ? 1 : 2, n);
        }
        if (next) {
          if (!(ok = wait(&k_full[kb], kp))) break;
          next_k();
          qk(0, b, sk);
          pg_commit(leader, &s_full[b]);
          pg_commit(leader, &kv_empty[sk]);
          sk = step(sk, j == -2 ? 1 : 2, n);
        }
      }
    } else {
      ok = wait(&k_full[0], 0);
      for (int b = 0; ok && b < nq; ++b) {
        if (!(ok = wait(&q_ready[b], 0))) break;
        qk(b, NQ == 2 ? b : 0, 0);
        pg_commit(leader, &s_full[b]);
      }
      pg_commit(leader, &kv_empty[0]);
      next_k();
    }
    int sv = 1, sk = 2;
    for (int j = 0; ok && !dual && j < nt; ++j) {
      if constexpr (NQ == 2) {
        // per Q tile: O += P V, then S of the next key tile.  MMAs run in the order of issue, so S may overwrite the P
        // that the product before it reads
        if (!(ok = wait(&v_ok[vb], vp) && (j + 1 == nt || wait(&k_full[kb], kp)))) break;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          if (b >= nq || !ok) break;
#pragma unroll
          for (int hf = 0; hf < C::kHands; ++hf) {
            if (!(ok = ok && wait(&p_full[b][hf], j))) break;
            pv(b, b, sv, hf, j > 0);
          }
          if (!ok) break;
          if (j + 1 < nt) {
            qk(b, b, sk);
            pg_commit(leader, &s_full[b]);
          }
          pg_commit(leader, &o_done[b]);
          if (b == nq - 1) {
            pg_commit(leader, &kv_empty[sv]);
            if (j + 1 < nt) pg_commit(leader, &kv_empty[sk]);
          }
        }
      } else {
        // one Q tile, S in two places: S of the next key tile is issued ahead of this tile's O += P V
        if (j + 1 < nt) {
          if (!(ok = wait(&k_full[kb], kp))) break;
          qk(0, (j + 1) & 1, sk);
          pg_commit(leader, &s_full[(j + 1) & 1]);
          pg_commit(leader, &kv_empty[sk]);
        }
        if (!(ok = wait(&v_ok[vb], vp) && wait(&p_full[j & 1][0], j >> 1))) break;
        pv(0, j & 1, sv, 0, j > 0);
        pg_commit(leader, &kv_empty[sv]);
        pg_commit(leader, &o_done[j & 1]);
      }
      next_v(), next_k();
      sv = step(sv, 2, S), sk = step(sk, 2, S);
    }
    // every MMA has ended before tensor memory is released
    pg_commit(leader, &mma_idle);
    pg_wait(&mma_idle, 0, a.err);
  }
  if (warp >= 2) {
    // ---------------- V tiles that are not attended to entirely ----------------
    // Warp 2; the last three tiles, where most of them are, with warp 3, whose loads do not wait for those (four chunks of
    // 2K tokens, 8B heads: 214.7 us with warp 2 alone, 210.6 with both).
    const int both = max(0, nt - 3), j0 = warp == 2 ? 0 : both;
    int vb = j0 % S, vp = j0 / S & 1;
    bool ok = loaded;
    for (int j = j0; ok && j < nt; ++j) {
      ok = __all_sync(0xffffffffu, pg_wait(&v_full[vb], (uint32_t)vp, a.err));
      if (!ok) break;
      const int key0 = (u.tile0 + j) * TN, n_warps = j < both ? 1 : 2;
      if (key0 + TN - 1 > first_pos || key0 < lo_last) {
        bool bad = false;
        const int s = stage_of(v_at(j));
        // keys [a, b) of the tile
        auto check = [&](int ka, int kb) {
          const int n = (kb - ka) * 8;  // 16-byte pieces of a 64-column block
#pragma unroll 1
          for (int c = 0; c < HD / 64; ++c) {
            unsigned char* v = ring + s * C::kStage + c * (TN * 128) + (ka - key0) * 128;
#pragma unroll 4
            for (int x = (j < both ? 0 : (warp - 2) * 32) + lane; x < n; x += 32 * n_warps) {
              const int key = ka + x / 8;
              uint4* p = reinterpret_cast<uint4*>(v + x * 16);
              uint4 w = *p;
              if (key >= u.key_hi || key < lo_first) {
                *p = make_uint4(0u, 0u, 0u, 0u);
              } else if (pg_clean<__nv_bfloat16>(w)) {
                *p = w;
                bad = true;
              }
            }
          }
        };
        const int k1 = key0 + TN;
        if (lo_last > key0) check(key0, min(k1, lo_last));                                           // some window starts behind them
        if (first_pos + 1 < k1) check(max(max(key0, lo_last > key0 ? min(k1, lo_last) : key0), first_pos + 1), k1);  // some rows are before them
        if (bad) *reinterpret_cast<volatile int*>(&s_bad) = 1;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
      }
      if (lane < 3 - n_warps) mbar_arrive(&v_ok[vb]);
      if (++vb == S) vb = 0, vp ^= 1;
    }
  }
  } else {
  if (NQ == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
  if ((warp - 4) / 4 < nq) {
    // ---------------- softmax: thread = row ----------------
    const int b = (warp - 4) / 4;
    const int row = (warp & 3) * 32 + lane;  // of this Q tile
    const uint32_t lb = (uint32_t)((warp & 3) * 32) << 16;
    const int rr = dual ? row : b * 128 + row;  // of the part
    const bool valid = rr < u.n_rows;
    const int r = u.r0 + min(rr, u.n_rows - 1);
    const int tok = r / a.G, head = u.kvh * a.G + r % a.G;
    const int qpos = u.pos0 + tok;
    const int kmin = a.win ? max(0, qpos - a.window + 1) : 0;
    if (!dual || b == 0) {
      const uint4* src = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.q) +
                                                        (long long)(u.q_row0 + tok) * a.q_stride + (long long)head * HD);
      unsigned char* dst = sq + b * (128 * HD * 2) + row * 128;
#pragma unroll 8
      for (int i = 0; i < HD / 8; ++i)
        *reinterpret_cast<uint4*>(dst + (i / 8) * 16384 + (((i % 8) ^ (row & 7)) << 4)) = valid ? src[i] : make_uint4(0u, 0u, 0u, 0u);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_ready[b]);
    }
    float m = -INFINITY, lsum = 0.f;  // m: largest score before scaling
    bool ok = true;
    const float sl = a.scale_log2;
    const uint32_t T_O = tm + C::kO + b * HD + lb;
    // this stream's key tiles: tile0 + step * j + first
    const int step = dual ? 2 : 1, first = dual ? b : 0, n_mine = (nt - first + step - 1) / step;
    for (int j = 0; j < n_mine; ++j) {
      const int slot = NQ == 2 ? b : j & 1;
      ok = __all_sync(0xffffffffu, pg_wait(&s_full[slot], (uint32_t)((NQ == 2 ? j : j >> 1) & 1), a.err));
      if (!ok) break;
      tc::fence_after_sync();
      const uint32_t T_S = tm + slot * C::kS + lb;
      float sv[TN];
#pragma unroll
      for (int c = 0; c < TN / 32; ++c) {
        float t[32];
        tc::ld32(T_S + c * 32, t);
#pragma unroll
        for (int i = 0; i < 32; ++i) sv[c * 32 + i] = t[i];
      }
      tc::wait_ld();
      const int key0 = (u.tile0 + step * j + first) * TN;
      if (!__all_sync(0xffffffffu, key0 >= kmin && key0 + TN - 1 <= qpos)) {
        const int last = qpos - key0;
#pragma unroll
        for (int c = 0; c < TN; ++c)
          if (c > last) sv[c] = -INFINITY;
        if (a.win) {
          const int from = kmin - key0;
#pragma unroll
          for (int c = 0; c < TN; ++c)
            if (c < from) sv[c] = -INFINITY;
        }
      }
      // p = 2^(s scale log2e - m scale log2e)
      constexpr int N2 = TN / 2 / C::kHands;  // pairs of a part
      const f32x2 sl2 = pk2(sl, sl);
      f32x2 ls[2], neg2;
      uint32_t pk[N2];
      auto weights = [&](int hf) {
#pragma unroll
        for (int c = 0; c < N2; ++c) {
          const int e = 2 * (hf * N2 + c);
          const f32x2 x = fma2(pk2(sv[e], sv[e + 1]), sl2, neg2);
          float p0, p1;
          un2(x, p0, p1);
          p0 = fast_exp2(p0);
          p1 = fast_exp2(p1);
          ls[c & 1] = add2(ls[c & 1], pk2(p0, p1));
          pk[c] = pg_pack_bf16(p0, p1);
        }
      };
      // The first part is computed with the reference of the tiles before while the maximum is found; the reference
      // changes only when a row's maximum grew by more than 2^8, and then the part is computed again.
      float neg = m == -INFINITY ? 0.f : -m * sl;
      neg2 = pk2(neg, neg);
      ls[0] = ls[1] = 0ull;
      float mx[4] = {sv[0], sv[1], sv[2], sv[3]};
#pragma unroll
      for (int c = 4; c < TN - 4; c += 8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) mx[i] = max3(mx[i], sv[c + 2 * i], sv[c + 2 * i + 1]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) mx[i] = fmaxf(mx[i], sv[TN - 4 + i]);
      const float m_new = fmaxf(m, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
      const bool grow = m == -INFINITY ? m_new != -INFINITY : (m_new - m) * sl > 8.f;
      if (j > 0) weights(0);
      if (__any_sync(0xffffffffu, grow || j == 0)) {
        float alpha = 1.f;
        if (grow) {
          alpha = m == -INFINITY ? 0.f : fast_exp2((m - m_new) * sl);
          lsum *= alpha;
          m = m_new;
        }
        if (j > 0) {
          ok = __all_sync(0xffffffffu, pg_wait(&o_done[NQ == 2 ? b : (j - 1) & 1], (uint32_t)((NQ == 2 ? j - 1 : (j - 1) >> 1) & 1), a.err));
          if (!ok) break;
          tc::fence_after_sync();
#pragma unroll 1
          for (int c = 0; c < HD / 32; ++c) {
            float ov[32];
            tc::ld32(T_O + c * 32, ov);
            tc::wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) ov[i] *= alpha;
            tc::st32(T_O + c * 32, ov);
          }
        }
        neg = m == -INFINITY ? 0.f : -m * sl;
        neg2 = pk2(neg, neg);
        ls[0] = ls[1] = 0ull;
        weights(0);
      }
#pragma unroll
      for (int hf = 0; hf < C::kHands; ++hf) {
        if (hf > 0) weights(hf);
        tmem_st32u(T_S + hf * N2, pk);
        tc::wait_st();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[slot][hf]);
      }
      float l0, l1, l2, l3;
      un2(ls[0], l0, l1);
      un2(ls[1], l2, l3);
      lsum += (l0 + l1) + (l2 + l3);
    }
    // With S in two places softmax may be two tiles ahead of O, two phases that one barrier's parity would not tell apart:
    // o_done is a barrier per place then.
    if (ok)
      ok = __all_sync(0xffffffffu, pg_wait(&o_done[NQ == 2 ? b : (n_mine - 1) & 1], (uint32_t)((NQ == 2 ? n_mine - 1 : (n_mine - 1) >> 1) & 1), a.err));
    float f0 = 1.f, f1 = 0.f;  // factors of this stream's sums and the other's
    float* xo = reinterpret_cast<float*>(ring);  // the odd stream's O, [column][row], where the tiles were
    if constexpr (NQ == 2) {
      if (dual && nq == 2) {
        // Neither stream's MMAs read the tiles any more once both are done.
        if (b == 1) {
          if (ok) ok = __all_sync(0xffffffffu, pg_wait(&o_done[0], (uint32_t)(((nt + 1) / 2 - 1) & 1), a.err));
          tc::fence_after_sync();
          s_m1[row] = m;
          s_l1[row] = lsum;
#pragma unroll 1
          for (int c = 0; c < HD / 32; ++c) {
            float ov[32];
            tc::ld32(T_O + c * 32, ov);
            tc::wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) xo[(c * 32 + i) * 128 + row] = ov[i];
          }
        }
        asm volatile("bar.sync 3, 256;" ::: "memory");
        if (b == 1) ok = false;  // the even stream's warps write the rows
        const float m1 = s_m1[row], mm = fmaxf(m, m1), base = mm == -INFINITY ? 0.f : mm;
        f0 = fast_exp2((m - base) * sl);
        f1 = fast_exp2((m1 - base) * sl);
        lsum = lsum * f0 + s_l1[row] * f1;
        m = mm;
      }
    }
    if (ok) {
      tc::fence_after_sync();
      const bool split = u.n_parts > 1;
      const float inv = split ? 1.f : 1.f / lsum;
      const bool bad = *reinterpret_cast<volatile int*>(&s_bad) != 0;
      const long long ws_row = (long long)(u.slot + u.part) * (NQ * 128) + rr;
      __nv_bfloat16* orow = static_cast<__nv_bfloat16*>(a.out) + (long long)(u.q_row0 + tok) * a.out_stride + (long long)head * HD;
      const __nv_bfloat16* vbase = a.storage + ((long long)a.row_k + ((long long)(a.n_kv + u.kvh) << a.shift)) * HD;
#pragma unroll 1
      for (int c = 0; c < HD / 32; ++c) {
        float ov[32];
        tc::ld32(T_O + c * 32, ov);
        tc::wait_ld();
        if (NQ == 2 && dual && nq == 2) {
#pragma unroll
          for (int i = 0; i < 32; ++i) ov[i] = ov[i] * f0 + xo[(c * 32 + i) * 128 + row] * f1;
        }
        if (bad && valid) {
          for (int key = max(kmin, u.tile0 * TN); key <= min(qpos, u.tile1 * TN - 1); ++key) {
            const int key0 = key / TN * TN;
            if (!(key0 + TN - 1 > first_pos || key0 < lo_last)) continue;  // not taken out of this tile
            const __nv_bfloat16* v = vbase + (long long)table[key >> a.shift] * a.page_elems + (long long)(key & ((1 << a.shift) - 1)) * HD + c * 32;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const float x = __bfloat162float(v[i]);
              if (!pg_finite(x)) ov[i] += x;
            }
          }
        }
        if (valid) {
          if (split) {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              *reinterpret_cast<float4*>(a.ws_o + ws_row * HD + c * 32 + i) = make_float4(ov[i], ov[i + 1], ov[i + 2], ov[i + 3]);
          } else {
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              uint4 w;
              w.x = pg_pack_bf16(ov[i] * inv, ov[i + 1] * inv);
              w.y = pg_pack_bf16(ov[i + 2] * inv, ov[i + 3] * inv);
              w.z = pg_pack_bf16(ov[i + 4] * inv, ov[i + 5] * inv);
              w.w = pg_pack_bf16(ov[i + 6] * inv, ov[i + 7] * inv);
              *reinterpret_cast<uint4*>(orow + c * 32 + i) = w;
            }
          }
        }
      }
      if (split && valid) *reinterpret_cast<float2*>(a.ws_ml + ws_row * 2) = make_float2(m * sl, lsum);
    }
  }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 0) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tm, 512);
  }
}

}  // namespace l3p

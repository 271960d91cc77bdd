// Packed causal attention backward on the tensor cores (sm_100a, bf16 / f16,
// Dk = Dv = HD of 64 or 128), in two passes that each recompute S and dP:
//
//   dQ pass   CTA = 128 queries of one head over their 128-key tiles:
//             S = Q K^T, dP = dO V^T, dQ += dX K.
//   dKV pass  CTA = 128 keys of one key head over the 128-query tiles that see
//             them, head by head of the group: S^T = K Q^T, dP^T = V dO^T,
//             dV += P^T dO, dK += dX^T Q.
//   P = exp2(logit2 - lse2),  dX = P softcap' (dP - Delta).
//
// Seven products instead of the five of a single pass, and nothing is summed by
// atomics: the results do not depend on the order in which CTAs run.
//
// Delta comes from the forward's out, whose weights were rounded: its error is that of
// one more rounding of dX where few keys share a row.  Where a query tile has one key
// tile only, the dQ pass forms it from P and dP instead, before dX, and leaves it for
// the dKV pass (rows of 2 to 128 keys: dK 1.40 of its own rounding's error for 1.46).
//
// -lse and -Delta: in the dQ pass a row's two numbers sit in its thread.  In the
// dKV pass they belong to columns, and reading them from shared memory for every
// element took half of the compute warps' time (128 words a warp and tile);
// there they ride on the products instead: one more 16-dim step of ones times
// three bf16 terms per query (24 bits) leaves s - lse / scale and dP - Delta in
// the accumulators.  (With the softcap lse comes after the tanh: from shared
// memory.)
//
// Both passes: warp 0 TMA producer, warp 1 MMA issuer, warps 4-11 compute: a
// thread owns one TMEM lane (query, or key) and 64 of the tile's 128 columns.
// P and dX leave as 16-bit pairs in tensor memory and are the A operands of the
// accumulating products: they never pass through shared memory.  Where it is full
// (dQ pass; dKV pass with HD 128) they take the first half of the thread's own
// columns of S or dP.  MMAs are ordered only where they share an accumulator and a
// shape, so there a next tile's S (dP) waits until the product that reads P (dX)
// out of its columns has completed.
//
// dKV pass, TMEM: S^T, dP^T, dV, dK.  Per tile the compute warps work in two
// halves, exp of S then dX of dP, and the tensor core does the other half's
// products meanwhile (dK of the last tile and dP during exp; dV and the next S
// during dX).  dQ pass, TMEM: S, two dP, dQ.  S of the next tile is issued as soon
// as this one's is in registers and dP a tile ahead, so the compute warps wait
// for no product that depends on them.
//
// Measured, 8 / 2 heads of 128, 16384 tokens, bf16: dQ 573-598 us (1380-1440 TFLOP/s of
// its three products), dK/dV 925-980 us (1120-1190 of its four and their extra step),
// the tensor pipe busy 71 and 68 %.  Softcap, 2 x 4096, 16 heads, five examples: 156 and
// 222 us, bound by the exp2 unit: exp2 and a quotient for the tanh and exp2 for P are
// three results an element, 16 a clock, twice (the softcap dK/dV kernels also spill 44
// to 68 bytes).  The dK/dV pass with the products in the order dV, dK, S, dP: 5 %
// slower; without its waits for the reading products it took 900-920 us, with 8 compute
// warps of 64 columns then 1.00 ms for 0.96 with 16 of 32, and with lse and Delta from
// shared memory 0.96 for 0.90.
#include "causal_tc.cuh"

namespace tc {
namespace {

using namespace ctc;

// Columns of a tile per compute thread, and the CTA's sizes that follow.
template <int COLS> struct Shape {
  static constexpr int kParts = 128 / COLS;             // threads per TMEM lane
  static constexpr int kWarps = 4 * kParts;             // compute warps
  static constexpr int kThreads = 128 + 32 * kWarps;
  static constexpr int kSteps = COLS / 16;              // 16-column steps of an A operand per thread
};
constexpr int kDqCols = 64, kDkvCols = 32;
constexpr int BLK = 128 * 128;  // one 64-column block of a 128-row tile

struct BwdParams {
  CausalParams c;
  GridOrder order;
  float kq, kc;  // logit2 = kq s, or kc tanh(kq s)
};

template <int HD> struct BwdSmem {
  static constexpr int kTile = 128 * HD * 2;
  static constexpr int kNK = 3, kNV = 2, kNQ = 2;
  static constexpr int kAug = (2 + kNQ) * kAugTile;
  static constexpr int kDq = (2 + kNK + kNV) * kTile + 2 * 128 * 4 + 256 + 1024;
  static constexpr int kDkv = (2 + 2 * kNQ) * kTile + kAug + kNQ * 128 * 4 + 256 + 1024;
  static_assert(kDq <= 227 * 1024 && kDkv <= 227 * 1024, "backward shared memory exceeds the per-CTA limit");
};

// 1 - 2 / (e^2x + 1): tanh to a few 1e-7
__device__ __forceinline__ float tanh_exp(float x) {
  return 1.f - __fdividef(2.f, exp2_fast(x * (2.f * kLog2e)) + 1.f);
}

// p = exp2(logit2(s) + nl2) and pg = p softcap' of two columns.
template <bool CAP>
__device__ __forceinline__ void p_pair(float2 s, float2 nl2, float kq, float kc, float2* p, float2* pg) {
  if constexpr (CAP) {
    const float2 y = fmul2(s, make_float2(kq, kq));
    const float2 t = make_float2(tanh_exp(y.x), tanh_exp(y.y));
    const float2 a = ffma2(t, make_float2(kc, kc), nl2);
    *p = make_float2(exp2_fast(a.x), exp2_fast(a.y));
    *pg = fmul2(*p, ffma2(make_float2(-t.x, -t.y), t, make_float2(1.f, 1.f)));
  } else {
    const float2 a = ffma2(s, make_float2(kq, kq), nl2);
    *p = make_float2(exp2_fast(a.x), exp2_fast(a.y));
    *pg = *p;
  }
}

// Tile column base + i inside [jlo, jhi)?
__device__ __forceinline__ bool inside(int i, int jlo, int jhi) { return i >= jlo && i < jhi; }

// dX = pg (dP + nd), or pg dP unless DELTA, of a thread's COLS columns of dP at
// d_addr, as 16-bit pairs at x_addr (which may be d_addr: each 32 are read before
// they are overwritten).
template <typename T, int COLS, bool MASK, bool DELTA>
__device__ __forceinline__ void dx_columns(uint32_t d_addr, uint32_t x_addr, const float* pg, float2 nd, int jlo,
                                           int jhi) {
#pragma unroll
  for (int h = 0; h < COLS / 32; ++h) {
    float dp[32];
    uint32_t w[16];
    tmem_ld32(d_addr + 32 * h, dp);
    tmem_wait_ld();
#pragma unroll
    for (int k = 0; k < 32; k += 2) {
      float2 v = make_float2(dp[k], dp[k + 1]);
      if constexpr (DELTA) v = fadd2(v, nd);
      v = fmul2(make_float2(pg[32 * h + k], pg[32 * h + k + 1]), v);
      if constexpr (MASK) {
        v.x = inside(32 * h + k, jlo, jhi) ? v.x : 0.f;
        v.y = inside(32 * h + k + 1, jlo, jhi) ? v.y : 0.f;
      }
      w[k >> 1] = Pack2<T>::pack(v.x, v.y);
    }
    tmem_st16u(x_addr + 16 * h, w);
  }
}

// Sum of P dP over a thread's COLS columns inside [jlo, jhi), dP at d_addr and scores
// in pg, which become P softcap'.
template <int COLS, bool CAP>
__device__ __forceinline__ float p_sum(uint32_t d_addr, float* pg, float2 nl2, float kq, float kc, int jlo, int jhi) {
  float sum = 0.f;
#pragma unroll
  for (int h = 0; h < COLS / 32; ++h) {
    float dp[32];
    tmem_ld32(d_addr + 32 * h, dp);
    tmem_wait_ld();
#pragma unroll
    for (int k = 0; k < 32; k += 2) {
      float* x = pg + 32 * h + k;
      float2 pr, g;
      p_pair<CAP>(make_float2(x[0], x[1]), nl2, kq, kc, &pr, &g);
      if (inside(32 * h + k, jlo, jhi)) sum += pr.x * dp[k];
      if (inside(32 * h + k + 1, jlo, jhi)) sum += pr.y * dp[k + 1];
      x[0] = g.x;
      x[1] = g.y;
    }
  }
  return sum;
}

// P of a thread's COLS columns (scores in pg), as 16-bit pairs at p_addr; pg
// becomes P softcap'.  With the softcap nl holds -lse2 per column; without it the
// scores come as s - lse / scale.
template <typename T, int COLS, bool CAP, bool MASK>
__device__ __forceinline__ void p_columns_t(uint32_t p_addr, float* pg, const float* nl, float kq, float kc, int jlo,
                                            int jhi) {
#pragma unroll
  for (int h = 0; h < COLS / 32; ++h) {
    uint32_t w[16];
#pragma unroll
    for (int k = 0; k < 32; k += 4) {
      float4 l = make_float4(0.f, 0.f, 0.f, 0.f);
      if constexpr (CAP) l = *reinterpret_cast<const float4*>(nl + 32 * h + k);
#pragma unroll
      for (int m = 0; m < 4; m += 2) {
        float* x = pg + 32 * h + k + m;
        float2 pr, g;
        if constexpr (CAP) {
          p_pair<true>(make_float2(x[0], x[1]), m ? make_float2(l.z, l.w) : make_float2(l.x, l.y), kq, kc, &pr, &g);
        } else {
          const float2 a = fmul2(make_float2(x[0], x[1]), make_float2(kq, kq));
          pr = g = make_float2(exp2_fast(a.x), exp2_fast(a.y));
        }
        if constexpr (MASK) {
          pr.x = inside(32 * h + k + m, jlo, jhi) ? pr.x : 0.f;
          pr.y = inside(32 * h + k + m + 1, jlo, jhi) ? pr.y : 0.f;
        }
        w[(k + m) >> 1] = Pack2<T>::pack(pr.x, pr.y);
        x[0] = g.x;
        x[1] = g.y;
      }
    }
    tmem_st16u(p_addr + 16 * h, w);
  }
}

// Row `r` of a 128-row fp32 accumulator in TMEM (zeros unless have) times mul, as T.
template <typename T, int HD>
__device__ __forceinline__ void store_row(uint32_t taddr, bool have, T* out, float mul, bool store) {
#pragma unroll 1
  for (int d = 0; d < HD; d += 32) {
    float v[32];
    if (have) {
      tmem_ld32(taddr + d, v);
      tmem_wait_ld();
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = 0.f;
    }
    if (store) {
#pragma unroll
      for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(out + d + i * 8) = pack8<T>(v + i * 8, mul);
    }
  }
}

// ---------------------------------------------------------------------------
// dQ
// ---------------------------------------------------------------------------
template <typename T, int HD, bool CAP>
__global__ void __launch_bounds__(Shape<kDqCols>::kThreads, 1)
    causal_dq_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmg,
                     const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv,
                     const __grid_constant__ BwdParams p) {
  using Z = BwdSmem<HD>;
  constexpr int TB = Z::kTile, NK = Z::kNK, NV = Z::kNV;
  constexpr uint32_t kColP = 128, kColQ = 384;  // S, dP [128, 384), dQ
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* q_s = sm;
  uint8_t* g_s = q_s + TB;
  uint8_t* k_s = g_s + TB;
  uint8_t* v_s = k_s + NK * TB;
  float* sum_s = reinterpret_cast<float*>(v_s + NV * TB);  // [2][128] sums of P dP of the rows' halves
  uint64_t* bars = reinterpret_cast<uint64_t*>(sum_s + 2 * 128);
  uint64_t* q_full = bars;           // Q
  uint64_t* g_full = bars + 1;       // dO
  uint64_t* k_full = g_full + 1;     // [NK]
  uint64_t* k_empty = k_full + NK;
  uint64_t* v_full = k_empty + NK;   // [NV]
  uint64_t* v_empty = v_full + NV;
  uint64_t* s_full = v_empty + NV;
  uint64_t* s_free = s_full + 1;     // S in registers
  uint64_t* p_full = s_free + 1;     // [2] dP computed
  uint64_t* x_full = p_full + 2;     // [2] dX written
  uint64_t* q_done = x_full + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(q_done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  static_assert((2 + 2 * NK + 2 * NV + 7) * 8 + 8 <= 256, "barrier area");

  const CausalParams& c = p.c;
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  int block, hq, b;
  grid_place(p.order, &block, &hq, &b);
  const int q0 = (grid_blocks(p.order) - 1 - block) * 128, hkv = hq / c.E;
  int32_t* status = c.status;
  const int first0 = first_key(c, b, q0), last = min(q0 + 128, c.N) - 1;
  const int j0 = first0 <= last ? first0 / 128 : 0, j1 = first0 <= last ? last / 128 + 1 : 0;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(g_full, 1);
    for (int i = 0; i < NK; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < NV; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    mbar_init(s_full, 1);
    mbar_init(s_free, Shape<kDqCols>::kWarps);
    mbar_init(&p_full[0], 1);
    mbar_init(&p_full[1], 1);
    // one per dP buffer: a warp may be done with a tile's dX before another is with
    // the last one's (not two tiles ahead: S of the next waits for s_free of all)
    mbar_init(&x_full[0], Shape<kDqCols>::kWarps);
    mbar_init(&x_full[1], Shape<kDqCols>::kWarps);
    mbar_init(q_done, 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_holder, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;

  if (warp == 0) {
    if (lane == 0 && j0 < j1) {
      mbar_expect_tx(q_full, TB);
      load_rows<HD, 128>(q_s, &tmq, hq, q0, b, q_full);
      bool ok = true;
      auto load_k = [&](int j) {
        const int i = j - j0, st = i % NK;
        if (i >= NK && !mbar_wait(&k_empty[st], ((i / NK) - 1) & 1, abort_flag, status)) return false;
        mbar_expect_tx(&k_full[st], TB);
        load_rows<HD, 128>(k_s + st * TB, &tmk, hkv, j * 128, b, &k_full[st]);
        return true;
      };
      ok = load_k(j0);
      mbar_expect_tx(g_full, TB);
      load_rows<HD, 128>(g_s, &tmg, hq, q0, b, g_full);
      for (int j = j0; ok && j < j1; ++j) {
        const int i = j - j0, st = i % NV;
        if (i >= NV && !mbar_wait(&v_empty[st], ((i / NV) - 1) & 1, abort_flag, status)) break;
        mbar_expect_tx(&v_full[st], TB);
        load_rows<HD, 128>(v_s + st * TB, &tmv, hkv, j * 128, b, &v_full[st]);
        if (j + 1 < j1) ok = load_k(j + 1);
      }
    }
  } else if (warp == 1 && j0 < j1) {
    constexpr uint32_t kIdS = idesc_f16(128, 128, Pack2<T>::kFmt, 0, 0);
    constexpr uint32_t kIdQ = idesc_f16(128, HD, Pack2<T>::kFmt, 0, 1);
    const uint32_t qd = desc_lo(q_s, 16), gd = desc_lo(g_s, 16), kd0 = desc_lo(k_s, 16), vd0 = desc_lo(v_s, 16),
                   kt0 = desc_lo(k_s, BLK);
    const uint32_t tm = uniform(tmem);
    const int n = uniform(j1 - j0);
    const bool leader = elect_one();
    auto issue_s = [&](int i) {
      if (!mbar_wait(&k_full[i % NK], (i / NK) & 1, abort_flag, status)) return false;
      tc_fence_after();
      if (leader) {
        mma_tile_ss<HD>(tm, qd, kd0 + (((i % NK) * TB) >> 4), kIdS);
        mma_commit(s_full);
      }
      return true;
    };
    auto issue_p = [&](int i) {
      if (!mbar_wait(&v_full[i % NV], (i / NV) & 1, abort_flag, status)) return false;
      tc_fence_after();
      if (leader) {
        mma_tile_ss<HD>(tm + kColP + (i & 1) * 128, gd, vd0 + (((i % NV) * TB) >> 4), kIdS);
        mma_commit(&p_full[i & 1]);
        mma_commit(&v_empty[i % NV]);
      }
      return true;
    };
    bool ok = mbar_wait(q_full, 0, abort_flag, status) && issue_s(0) && mbar_wait(g_full, 0, abort_flag, status) &&
              issue_p(0);
    for (int i = 0; ok && i < n; ++i) {
      if (i + 1 < n) {
        if (!mbar_wait(s_free, i & 1, abort_flag, status)) break;
        if (!issue_s(i + 1)) break;
        // dP of i + 1 replaces dX of i - 1: the product that reads it has completed
        if (i > 0 && !mbar_wait(&k_empty[(i - 1) % NK], ((i - 1) / NK) & 1, abort_flag, status)) break;
        if (!issue_p(i + 1)) break;
      }
      if (!mbar_wait(&x_full[i & 1], (i >> 1) & 1, abort_flag, status)) break;
      tc_fence_after();
      if (leader) {
        mma_tile_ts<Shape<kDqCols>::kSteps, kDqCols>(tm + kColQ, tm + kColP + (i & 1) * 128,
                                                     kt0 + (((i % NK) * TB) >> 4), kIdQ, i > 0 ? 1u : 0u);
        mma_commit(&k_empty[i % NK]);
        if (i + 1 == n) mma_commit(q_done);
      }
    }
  } else if (warp >= 4) {
    constexpr int COLS = kDqCols;
    const int part = (warp - 4) >> 2;  // columns [COLS part, COLS part + COLS)
    const int r = (threadIdx.x - 128) & 127, q = q0 + r;
    const bool row_ok = q < c.N;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const int64_t row = ((int64_t)b * c.N + q) * c.Hq + hq;
    const int first = row_ok ? first_key(c, b, q) : 1, end = row_ok ? q + 1 : 0;
    const float nl = row_ok ? -c.lse[row] * kLog2e : 0.f, nd = row_ok ? -c.delta[row] : 0.f;
    const float2 nl2 = make_float2(nl, nl), nd2 = make_float2(nd, nd);
    const uint32_t s_addr = tmem + lane_base + part * COLS;
    bool alive = true;
    int i = 0;
    if (j1 - j0 == 1) {  // the rows' only tile: Delta from it, for this pass and the next
      const int jlo = first - j0 * 128 - part * COLS, jhi = end - j0 * 128 - part * COLS;
      const uint32_t x_addr = s_addr + kColP;
      alive = __all_sync(0xffffffffu, mbar_wait(s_full, 0, abort_flag, status) && mbar_wait(&p_full[0], 0, abort_flag, status));
      float pg[COLS];
      if (alive) {
        tc_fence_after();
        tmem_ld<COLS>(s_addr, pg);
        tmem_wait_ld();
        sum_s[part * 128 + r] = p_sum<COLS, CAP>(x_addr, pg, nl2, p.kq, p.kc, jlo, jhi);
      }
      named_bar(1, 32 * Shape<COLS>::kWarps);
      if (alive) {
        const float delta = sum_s[r] + sum_s[128 + r] - (row_ok && c.dlse ? c.dlse[row] : 0.f);
        if (row_ok && part == 0) c.delta[row] = delta;
        dx_columns<T, COLS, true, true>(x_addr, x_addr, pg, make_float2(-delta, -delta), jlo, jhi);
        tmem_wait_st();
        tc_fence_before();
        warp_arrive(&x_full[0], lane);
        i = 1;
      }
    }
    for (int j = j0 + i; alive && j < j1; ++j, ++i) {
      alive = __all_sync(0xffffffffu, mbar_wait(s_full, i & 1, abort_flag, status));
      if (!alive) break;
      tc_fence_after();
      const uint32_t x_addr = s_addr + kColP + (i & 1) * 128;
      const int jlo = first - j * 128 - part * COLS, jhi = end - j * 128 - part * COLS;
      float pg[COLS];
      tmem_ld<COLS>(s_addr, pg);
      tmem_wait_ld();
      tc_fence_before();
      warp_arrive(s_free, lane);
#pragma unroll
      for (int k = 0; k < COLS; k += 2) {
        float2 pr, g;
        p_pair<CAP>(make_float2(pg[k], pg[k + 1]), nl2, p.kq, p.kc, &pr, &g);
        pg[k] = g.x;
        pg[k + 1] = g.y;
      }
      alive = __all_sync(0xffffffffu, mbar_wait(&p_full[i & 1], (i >> 1) & 1, abort_flag, status));
      if (!alive) break;
      tc_fence_after();
      if (__all_sync(0xffffffffu, jlo <= 0 && jhi >= COLS))
        dx_columns<T, COLS, false, true>(x_addr, x_addr, pg, nd2, jlo, jhi);
      else
        dx_columns<T, COLS, true, true>(x_addr, x_addr, pg, nd2, jlo, jhi);
      tmem_wait_st();
      tc_fence_before();
      warp_arrive(&x_full[i & 1], lane);
    }
    if (alive && i > 0) alive = __all_sync(0xffffffffu, mbar_wait(q_done, 0, abort_flag, status));
    if (alive) {
      tc_fence_after();
      if (part == 0)
        store_row<T, HD>(tmem + lane_base + kColQ, i > 0, static_cast<T*>(c.dq) + row * HD, c.scale, row_ok);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------------------
// dK, dV
// ---------------------------------------------------------------------------
template <typename T, int HD, bool CAP>
__global__ void __launch_bounds__(Shape<kDkvCols>::kThreads, 1)
    causal_dkv_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmg,
                      const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv,
                      const __grid_constant__ BwdParams p) {
  using Z = BwdSmem<HD>;
  using Z2 = Shape<kDkvCols>;
  constexpr int TB = Z::kTile, NQ = Z::kNQ;
  constexpr uint32_t kColD = 128, kColV = 256, kColK = 256 + HD;  // S^T, dP^T, dV, dK
  // P^T, dX^T: columns of their own, or the first halves of each thread's S^T, dP^T
  constexpr bool kOwnP = HD == 64;
  constexpr uint32_t kColP = kOwnP ? 256 + 2 * HD : 0, kColX = kOwnP ? kColP + 64 : kColD;
  constexpr int kStepP = kOwnP ? kDkvCols / 2 : kDkvCols;  // from one part's pairs to the next's
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* one_s = sm;                // [2] ones that pick -lse / scale (dims 0-2) and -Delta (3-5) out of aug_s
  uint8_t* aug_s = one_s + 2 * kAugTile;  // [NQ] per query: both, as three bf16 terms each
  uint8_t* k_s = aug_s + NQ * kAugTile;
  uint8_t* v_s = k_s + TB;
  uint8_t* q_s = v_s + TB;        // [NQ]
  uint8_t* g_s = q_s + NQ * TB;   // [NQ]
  float* nl_s = reinterpret_cast<float*>(g_s + NQ * TB);  // softcap: [NQ][128] -lse log2e of the tile's queries
  uint64_t* bars = reinterpret_cast<uint64_t*>(nl_s + NQ * 128);
  uint64_t* k_full = bars;
  uint64_t* v_full = bars + 1;
  uint64_t* q_full = bars + 2;      // [NQ] Q
  uint64_t* g_full = q_full + NQ;   // [NQ] dO
  uint64_t* i_full = g_full + NQ;   // [NQ] info
  uint64_t* q_empty = i_full + NQ;  // [NQ] Q, dO read by the last product
  uint64_t* i_empty = q_empty + NQ; // [NQ]
  uint64_t* s_full = i_empty + NQ;
  uint64_t* p_full = s_full + 1;    // P^T written
  uint64_t* d_full = p_full + 1;    // dP^T computed
  uint64_t* x_full = d_full + 1;    // dX^T written
  uint64_t* v_done = x_full + 1;    // P^T read by its product
  uint64_t* done = v_done + 1;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  static_assert((2 + 5 * NQ + 6) * 8 + 8 <= 256, "barrier area");

  const CausalParams& c = p.c;
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  int block, hkv, b;
  grid_place(p.order, &block, &hkv, &b);
  const int k0 = block * 128;  // the first keys are seen by the most queries
  int32_t* status = c.status;
  const int last = min(k0 + 128, c.N) - 1;
  const int t0 = k0 / 128, t1 = (query_end(c, b, last) + 127) / 128;  // query tiles
  const int nt = max(t1 - t0, 0);
  const int n = query_end(c, b, last) > k0 ? nt * c.E : 0;  // nobody sees a tile of padding

  if (threadIdx.x == 0) {
    mbar_init(k_full, 1);
    mbar_init(v_full, 1);
    for (int i = 0; i < NQ; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&g_full[i], 1);
      mbar_init(&i_full[i], 64);
      mbar_init(&q_empty[i], 1);
      mbar_init(&i_empty[i], Z2::kWarps);
    }
    mbar_init(s_full, 1);
    mbar_init(p_full, Z2::kWarps);
    mbar_init(d_full, 1);
    mbar_init(x_full, Z2::kWarps);
    mbar_init(v_done, 1);
    mbar_init(done, 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_holder, 512);
    tmem_relinquish();
  }
  if (threadIdx.x >= 128 && threadIdx.x < 256) {
    const int r = threadIdx.x - 128;
    const uint32_t one = 0x3f80u;  // bf16 1
    *reinterpret_cast<uint4*>(one_s + r * 16) = make_uint4(one | one << 16, one, 0u, 0u);
    *reinterpret_cast<uint4*>(one_s + kAugTile + r * 16) = make_uint4(0u, one << 16, one | one << 16, 0u);
    for (int i = 0; i < 2 + NQ; ++i)  // dims 8-15
      *reinterpret_cast<uint4*>(one_s + i * kAugTile + kAugHalf + r * 16) = make_uint4(0u, 0u, 0u, 0u);
    fence_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;

  if (warp == 0) {
    if (lane == 0 && n > 0) {
      mbar_expect_tx(k_full, TB);
      load_rows<HD, 128>(k_s, &tmk, hkv, k0, b, k_full);
      for (int i = 0; i < n; ++i) {
        const int st = i % NQ, hq = hkv * c.E + i / nt, qt = t0 + i % nt;
        if (i >= NQ && !mbar_wait(&q_empty[st], ((i / NQ) - 1) & 1, abort_flag, status)) break;
        mbar_expect_tx(&q_full[st], TB);
        load_rows<HD, 128>(q_s + st * TB, &tmq, hq, qt * 128, b, &q_full[st]);
        if (i == 0) {
          mbar_expect_tx(v_full, TB);
          load_rows<HD, 128>(v_s, &tmv, hkv, k0, b, v_full);
        }
        mbar_expect_tx(&g_full[st], TB);
        load_rows<HD, 128>(g_s + st * TB, &tmg, hq, qt * 128, b, &g_full[st]);
      }
    }
  } else if (warp == 1) {
    constexpr uint32_t kIdS = idesc_f16(128, 128, Pack2<T>::kFmt, 0, 0);
    constexpr uint32_t kIdA = idesc_f16(128, HD, Pack2<T>::kFmt, 0, 1);
    const uint32_t kd = desc_lo(k_s, 16), vd = desc_lo(v_s, 16), qd0 = desc_lo(q_s, 16), gd0 = desc_lo(g_s, 16),
                   qt0 = desc_lo(q_s, BLK), gt0 = desc_lo(g_s, BLK), one0 = aug_lo(one_s), aug0 = aug_lo(aug_s);
    const uint32_t tm = uniform(tmem);
    const int un = uniform(n);
    const bool leader = elect_one();
    auto issue_s = [&](int i) {
      if (!mbar_wait(&q_full[i % NQ], (i / NQ) & 1, abort_flag, status) ||
          !mbar_wait(&i_full[i % NQ], (i / NQ) & 1, abort_flag, status))
        return false;
      tc_fence_after();
      if (leader) {
        mma_tile_ss<HD>(tm, kd, qd0 + (((i % NQ) * TB) >> 4), kIdS);
        if constexpr (!CAP) mma_aug(tm, one0, aug0 + (((i % NQ) * kAugTile) >> 4));
        mma_commit(s_full);
      }
      return true;
    };
    auto issue_d = [&](int i) {
      if (!mbar_wait(&g_full[i % NQ], (i / NQ) & 1, abort_flag, status)) return false;
      tc_fence_after();
      if (leader) {
        mma_tile_ss<HD>(tm + kColD, vd, gd0 + (((i % NQ) * TB) >> 4), kIdS);
        mma_aug(tm + kColD, one0 + (kAugTile >> 4), aug0 + (((i % NQ) * kAugTile) >> 4));
        mma_commit(d_full);
      }
      return true;
    };
    bool ok = un > 0 && mbar_wait(k_full, 0, abort_flag, status) && issue_s(0) &&
              mbar_wait(v_full, 0, abort_flag, status) && issue_d(0);
    for (int i = 0; ok && i < un; ++i) {
      const int st = i % NQ;
      if (!mbar_wait(p_full, i & 1, abort_flag, status)) break;
      tc_fence_after();
      if (leader) {
        mma_tile_ts<Z2::kSteps, kStepP>(tm + kColV, tm + kColP, gt0 + ((st * TB) >> 4), kIdA, i > 0 ? 1u : 0u);
        if constexpr (!kOwnP) mma_commit(v_done);
      }
      // HD 128: S of i + 1 replaces P of i
      if (i + 1 < un && ((!kOwnP && !mbar_wait(v_done, i & 1, abort_flag, status)) || !issue_s(i + 1))) break;
      if (!mbar_wait(x_full, i & 1, abort_flag, status)) break;
      tc_fence_after();
      if (leader) {
        mma_tile_ts<Z2::kSteps, kStepP>(tm + kColK, tm + kColX, qt0 + ((st * TB) >> 4), kIdA, i > 0 ? 1u : 0u);
        mma_commit(&q_empty[st]);
        if (i + 1 == un) mma_commit(done);
      }
      // HD 128: dP of i + 1 replaces dX of i
      if (i + 1 < un) ok = (kOwnP || mbar_wait(&q_empty[st], (i / NQ) & 1, abort_flag, status)) && issue_d(i + 1);
    }
  } else if (warp < 4) {
    // the tile's per-query numbers, two queries a thread
    const int t = threadIdx.x - 64;
    for (int i = 0; i < n; ++i) {
      const int st = i % NQ, hq = hkv * c.E + i / nt, qt = t0 + i % nt;
      float lse[2], nd[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int q = qt * 128 + t + 64 * h;
        lse[h] = nd[h] = 0.f;
        if (q < c.N) {
          const int64_t row = ((int64_t)b * c.N + q) * c.Hq + hq;
          lse[h] = c.lse[row];
          nd[h] = -c.delta[row];
          if (lse[h] == -INFINITY) lse[h] = 0.f;  // sees nothing: masked everywhere
        }
      }
      // the products of step i - NQ have read the buffer (and the compute warps nl_s)
      if (i >= NQ && !(__all_sync(0xffffffffu, mbar_wait(&q_empty[st], ((i / NQ) - 1) & 1, abort_flag, status)) &&
                       (!CAP || __all_sync(0xffffffffu, mbar_wait(&i_empty[st], ((i / NQ) - 1) & 1, abort_flag, status)))))
        break;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = t + 64 * h;
        if constexpr (CAP) nl_s[st * 128 + r] = -lse[h] * kLog2e;
        const float x[2] = {-lse[h] / c.scale, nd[h]};
        float y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          y[3 * w] = round_to<__nv_bfloat16>(x[w]);
          y[3 * w + 1] = round_to<__nv_bfloat16>(x[w] - y[3 * w]);
          y[3 * w + 2] = x[w] - y[3 * w] - y[3 * w + 1];
        }
        *reinterpret_cast<uint4*>(aug_s + st * kAugTile + r * 16) = pack8<__nv_bfloat16>(y, 1.f);
      }
      fence_async_smem();
      mbar_arrive(&i_full[st]);
    }
  } else {
    constexpr int COLS = kDkvCols;
    const int part = (warp - 4) >> 2;
    const int r = (threadIdx.x - 128) & 127, k = k0 + r;
    const bool row_ok = k < c.N;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lane_base + part * COLS, d_addr = s_addr + kColD;
    const uint32_t p_addr = tmem + lane_base + kColP + part * kStepP, x_addr = tmem + lane_base + kColX + part * kStepP;
    const int qend = row_ok ? query_end(c, b, k) : 0;
    bool alive = true;
    int i = 0;
    for (; i < n; ++i) {
      const int st = i % NQ, qt = t0 + i % nt;
      const int jlo = k - qt * 128 - part * COLS, jhi = qend - qt * 128 - part * COLS;
      const bool interior = __all_sync(0xffffffffu, jlo <= 0 && jhi >= COLS);
      if constexpr (CAP) alive = __all_sync(0xffffffffu, mbar_wait(&i_full[st], (i / NQ) & 1, abort_flag, status));
      alive = alive && __all_sync(0xffffffffu, mbar_wait(s_full, i & 1, abort_flag, status));
      if (!alive) break;
      tc_fence_after();
      const float* nl = nl_s + st * 128 + part * COLS;
      float pg[COLS];
      tmem_ld<COLS>(s_addr, pg);
      tmem_wait_ld();
      if (interior) p_columns_t<T, COLS, CAP, false>(p_addr, pg, nl, p.kq, p.kc, jlo, jhi);
      else p_columns_t<T, COLS, CAP, true>(p_addr, pg, nl, p.kq, p.kc, jlo, jhi);
      tmem_wait_st();
      tc_fence_before();
      if constexpr (CAP) warp_arrive(&i_empty[st], lane);
      warp_arrive(p_full, lane);
      alive = __all_sync(0xffffffffu, mbar_wait(d_full, i & 1, abort_flag, status));
      if (!alive) break;
      tc_fence_after();
      if (interior) dx_columns<T, COLS, false, false>(d_addr, x_addr, pg, make_float2(0.f, 0.f), jlo, jhi);
      else dx_columns<T, COLS, true, false>(d_addr, x_addr, pg, make_float2(0.f, 0.f), jlo, jhi);
      tmem_wait_st();
      tc_fence_before();
      warp_arrive(x_full, lane);
    }
    if (alive && n > 0) alive = __all_sync(0xffffffffu, mbar_wait(done, 0, abort_flag, status));
    if (alive) {
      tc_fence_after();
      const int64_t row = ((int64_t)b * c.N + k) * c.Hkv + hkv;
      if (part == 0)
        store_row<T, HD>(tmem + lane_base + kColV, n > 0, static_cast<T*>(c.dv) + row * HD, 1.f, row_ok);
      else if (part == 1)
        store_row<T, HD>(tmem + lane_base + kColK, n > 0, static_cast<T*>(c.dk) + row * HD, c.scale, row_ok);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <typename T, int HD, bool CAP>
int launch_bwd(const CausalParams& a, int dtype, cudaStream_t st) {
  CUtensorMap mq, mg, mk, mv;
  const int64_t gh = HD, gn = (int64_t)a.Hq * HD, gb = gn * a.N;
  if (int rc = make_map_strided(&mq, a.q, dtype, a.B, a.N, a.Hq, HD, a.q_sb, a.q_sn, a.q_sh, 128)) return rc;
  if (int rc = make_map_strided(&mg, a.dout, dtype, a.B, a.N, a.Hq, HD, gb, gn, gh, 128)) return rc;
  if (int rc = make_map_strided(&mk, a.k, dtype, a.B, a.N, a.Hkv, HD, a.k_sb, a.k_sn, a.k_sh, 128)) return rc;
  if (int rc = make_map_strided(&mv, a.v, dtype, a.B, a.N, a.Hkv, HD, a.v_sb, a.v_sn, a.v_sh, 128)) return rc;
  BwdParams p;
  p.c = a;
  p.kq = a.has_cap ? a.scale / a.cap : a.scale * kLog2e;
  p.kc = a.cap * kLog2e;
  auto kq = causal_dq_kernel<T, HD, CAP>;
  auto kk = causal_dkv_kernel<T, HD, CAP>;
  if (cudaFuncSetAttribute(kq, cudaFuncAttributeMaxDynamicSharedMemorySize, BwdSmem<HD>::kDq) != cudaSuccess ||
      cudaFuncSetAttribute(kk, cudaFuncAttributeMaxDynamicSharedMemorySize, BwdSmem<HD>::kDkv) != cudaSuccess)
    return TC_ERR_CUDA;
  const int tiles = (a.N + 127) / 128;
  const int64_t rows = (int64_t)a.B * a.N * HD * 4;  // bytes of a head's K and V, or Q and dO
  dim3 grid = grid_order(tiles, a.Hq, a.B, rows * a.Hkv, &p.order);
  kq<<<grid, Shape<kDqCols>::kThreads, BwdSmem<HD>::kDq, st>>>(mq, mg, mk, mv, p);
  if (int rc = launch_status()) return rc;
  grid = grid_order(tiles, a.Hkv, a.B, rows * a.Hq, &p.order);
  kk<<<grid, Shape<kDkvCols>::kThreads, BwdSmem<HD>::kDkv, st>>>(mq, mg, mk, mv, p);
  return launch_status();
}

template <typename T>
int dispatch_bwd(const CausalParams& a, int dtype, cudaStream_t st) {
  if (a.Dk == 128)
    return a.has_cap ? launch_bwd<T, 128, true>(a, dtype, st) : launch_bwd<T, 128, false>(a, dtype, st);
  return a.has_cap ? launch_bwd<T, 64, true>(a, dtype, st) : launch_bwd<T, 64, false>(a, dtype, st);
}

}  // namespace

bool causal_bwd_tc_supported(const CausalParams& p, int dtype) {
  return ctc::tc_shape(p, dtype) &&
         ((uintptr_t)p.dout | (uintptr_t)p.dq | (uintptr_t)p.dk | (uintptr_t)p.dv) % 16 == 0;
}

int causal_bwd_tc(const CausalParams& p, int dtype, cudaStream_t st) {
  return dtype == TC_BF16 ? dispatch_bwd<__nv_bfloat16>(p, dtype, st) : dispatch_bwd<__half>(p, dtype, st);
}

}  // namespace tc

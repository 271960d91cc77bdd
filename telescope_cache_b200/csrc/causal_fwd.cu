// Packed causal attention forward on the tensor cores (sm_100a, bf16 / f16,
// Dk = Dv = HD of 64 or 128).
//
// CTA = 256 queries of one head as two 128-row tiles A and B that take turns on
// the tensor core: while one tile's scores are in its softmax, the other's
// products run.
//   warp 0      TMA producer: Q_A, Q_B once, then 128-key K and V tiles, each in
//               a ring of its own (K is free after S, V only after PV)
//   warp 1      MMA issuer: S_X = Q_X K^T into TMEM, O_X += P_X V with P_X read
//               from TMEM
//   warps 4-7   softmax of tile A, warps 8-11 of tile B: a thread owns a query
//               row and all 128 keys of a tile: mask, softcap, running maximum
//               and sums in fp32 (log2 units, O rescaled only when the maximum
//               grew by more than 2^8), P rounded to the operand type for the
//               second product, O over the sum of the rounded weights, lse from
//               that of the others.
// P in 16 bits leaves out 1.8e-3 to 2.0e-3 of its norm off (bf16; its own rounding
// alone: 1.6e-3); a second product for what the rounding left over would cost half of
// a tile's products again.  Weights that sum to one as they are used matter to the
// backward: Delta = sum w dP then errs by roundings of dX, not of P dP (values of mean
// 8, sharp rows: dQ 2.5e-3 off for 1.3e-2).  The second sum costs 4 %: 491 -> 511 us
// (pairs unpacked and added two at a time: 522).
// TMEM: S_A, S_B (128 columns each), O_A, O_B (HD each), P_A, P_B (64: 16-bit pairs).
// With HD 128 the first four fill it, and P_X takes the first half of S_X.  MMAs are
// ordered only where they share an accumulator and a shape, so there the next S_X
// waits for PV_X to complete before it overwrites P_X.  The commit of S_X covers the
// PV_X before it: when the softmax wakes O_X is current and the last P_X read.
//
// A query tile's keys run from the first key of its first row (starts do not
// descend) to the diagonal; tiles in between need no mask.  The heaviest blocks
// come first in the grid.
//
// Softcap: with y = x / c and a the largest |y| of the warp's rows in the tile,
// tanh comes from its odd Maclaurin series (through y^5 below 0.15, y^9 below
// 0.5: 1e-6 and 1e-5 of the value), else as 1 - 2 / (e^2y + 1).
//
// Measured, 8 / 2 heads of 128, 16384 tokens, bf16: 511-555 us (from box to box and
// with q, k, v as views of one projection), 990-1070 TFLOP/s of visible entries,
// 0.61-0.66 of a large GEMM's burst rate, tensor pipe 50 %.  Bound by each tile's chain
// (scores, maximum, exp2, product): of a warp's 3600 clocks a tile 1750 went to exp2 and
// rounding, which both tiles' warps share, 360 to the maximum.  Packed prompts (2 x
// 8192, 16 / 4 heads, seven examples): 230 us; with softcap (2 x 4096, 16 heads, five
// examples): 128 us.  Two threads a row, with a swap of their maxima, gained 2 % without
// softcap and lost 12 % with it.
//
// Every mbarrier wait is bounded (tc_ptx.cuh).
#include <cmath>
#include <type_traits>

#include "causal_tc.cuh"

namespace tc {
namespace {

using namespace ctc;

constexpr int kFwdThreads = 384;
constexpr float kLazy = 8.f;  // rescale threshold, log2 units
constexpr float kPoly5 = 0.15f, kPoly9 = 0.5f;
constexpr double kT3 = -1.0 / 3.0, kT5 = 2.0 / 15.0, kT7 = -17.0 / 315.0, kT9 = 62.0 / 2835.0;

template <int HD> struct FwdSmem {
  static constexpr int kTile = 128 * HD * 2;
  static constexpr int kStages = HD == 128 ? 2 : 4;  // of K, and of V
  static constexpr int kBytes = 2 * kTile + 2 * kStages * kTile + 256 + 1024;
  static_assert(kBytes <= 227 * 1024, "forward shared memory exceeds the per-CTA limit");
};

struct FwdParams {
  CausalParams c;
  GridOrder order;
  float kq, kc;              // logit2 = kq s, or kc tanh(kq s)
  float e1, e3, e5, e7, e9;  // its series in s
  float top5, top9;          // largest |y| of each; below 0 where fp32 does not hold its terms
};

enum { kPlain = 0, kS5 = 1, kS9 = 2, kTanh = 3 };

__device__ __forceinline__ float2 f2(float v) { return make_float2(v, v); }

template <int MODE>
__device__ __forceinline__ float logit2(float s, const FwdParams& p) {
  if constexpr (MODE == kPlain) return s * p.kq;
  const float w = s * s;
  if constexpr (MODE == kS5) return s * fmaf(w, fmaf(w, p.e5, p.e3), p.e1);
  if constexpr (MODE == kS9) return s * fmaf(w, fmaf(w, fmaf(w, fmaf(w, p.e9, p.e7), p.e5), p.e3), p.e1);
  return p.kc * (1.f - __fdividef(2.f, exp2_fast(s * p.kq * (2.f * kLog2e)) + 1.f));
}

// s += the two values of a packed pair (sums of a 16-bit and a 32-bit float).
template <typename T> __device__ __forceinline__ void add_pair(float2* s, uint32_t w) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
        "add.f32.bf16 %0, l, %0;\n\tadd.f32.bf16 %1, h, %1;\n\t}"
        : "+f"(s->x), "+f"(s->y)
        : "r"(w));
  else
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
        "add.f32.f16 %0, l, %0;\n\tadd.f32.f16 %1, h, %1;\n\t}"
        : "+f"(s->x), "+f"(s->y)
        : "r"(w));
}

// exp2(logit - m) of 32 scores as packed pairs, columns outside [jlo, jhi) zero;
// adds them up as they are (sum) and as the pairs hold them (held).
template <typename T, int MODE, bool MASK>
__device__ __forceinline__ void chunk_p(const float* sv, int c0, const FwdParams& p, float m, int jlo, int jhi,
                                        uint32_t* pw, float2* sum, float2* held) {
  const float2 negm = f2(-m);
#pragma unroll
  for (int c = 0; c < 32; c += 2) {
    const float2 u = make_float2(sv[c], sv[c + 1]);
    float2 a;
    if constexpr (MODE == kPlain) {
      a = ffma2(u, f2(p.kq), negm);
    } else if constexpr (MODE == kTanh) {
      a = fadd2(make_float2(logit2<kTanh>(u.x, p), logit2<kTanh>(u.y, p)), negm);
    } else {
      const float2 w = fmul2(u, u);
      float2 q;
      if constexpr (MODE == kS5) {
        q = ffma2(w, f2(p.e5), f2(p.e3));
      } else {
        q = ffma2(w, f2(p.e9), f2(p.e7));
        q = ffma2(w, q, f2(p.e5));
        q = ffma2(w, q, f2(p.e3));
      }
      a = ffma2(u, ffma2(w, q, f2(p.e1)), negm);
    }
    if constexpr (MASK) {
      a.x = (c0 + c >= jlo && c0 + c < jhi) ? a.x : -INFINITY;
      a.y = (c0 + c + 1 >= jlo && c0 + c + 1 < jhi) ? a.y : -INFINITY;
    }
    const float2 e = make_float2(exp2_fast(a.x), exp2_fast(a.y));
    *sum = fadd2(*sum, e);
    pw[c >> 1] = Pack2<T>::pack(e.x, e.y);
    add_pair<T>(held, pw[c >> 1]);
  }
}

template <typename T, int MODE>
__device__ __forceinline__ void half_p(bool interior, const float* sv, int c0, const FwdParams& p, float m, int jlo,
                                       int jhi, uint32_t* pw, float2* sum, float2* held) {
  if (interior) {
    chunk_p<T, MODE, false>(sv, c0, p, m, jlo, jhi, pw, sum, held);
    chunk_p<T, MODE, false>(sv + 32, c0 + 32, p, m, jlo, jhi, pw + 16, sum, held);
  } else {
    chunk_p<T, MODE, true>(sv, c0, p, m, jlo, jhi, pw, sum, held);
    chunk_p<T, MODE, true>(sv + 32, c0 + 32, p, m, jlo, jhi, pw + 16, sum, held);
  }
}

// The key tiles [lo, hi) of a 128-query tile that starts at q0 (none: 0, 0).
__device__ __forceinline__ void key_tiles(const CausalParams& p, int b, int q0, int* lo, int* hi) {
  *lo = *hi = 0;
  if (q0 >= p.N) return;
  const int last = min(q0 + 128, p.N) - 1, first = first_key(p, b, q0);
  if (first > last) return;  // padding alone
  *lo = first / KT;
  *hi = last / KT + 1;
}

template <typename T, int HD, bool CAP>
__global__ void __launch_bounds__(kFwdThreads, 1)
    causal_fwd_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
                      const __grid_constant__ CUtensorMap tmv, const __grid_constant__ FwdParams p) {
  using Z = FwdSmem<HD>;
  constexpr int TB = Z::kTile, NS = Z::kStages, BLK = 128 * 128;
  constexpr bool kOwnP = HD == 64;  // columns of P: its own, or S's
  constexpr uint32_t kColP = kOwnP ? 256 + 2 * HD : 0, kStepP = kOwnP ? 64 : 128;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* q_s = sm;             // [2] Q tiles
  uint8_t* k_s = q_s + 2 * TB;   // [NS]
  uint8_t* v_s = k_s + NS * TB;  // [NS]
  uint64_t* bars = reinterpret_cast<uint64_t*>(v_s + NS * TB);
  uint64_t* q_full = bars;           // [2]
  uint64_t* k_full = q_full + 2;     // [NS]
  uint64_t* k_empty = k_full + NS;   // [NS]
  uint64_t* v_full = k_empty + NS;   // [NS]
  uint64_t* v_empty = v_full + NS;   // [NS]
  uint64_t* s_full = v_empty + NS;   // [2]
  uint64_t* p_full = s_full + 2;     // [2]
  uint64_t* pv_done = p_full + 2;    // [2] P read: the next S may overwrite it
  uint64_t* o_done = pv_done + 2;    // [2]
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(o_done + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  static_assert((10 + 4 * NS) * 8 + 8 <= 256, "barrier area");

  const CausalParams& c = p.c;
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  int block, hq, b;
  grid_place(p.order, &block, &hq, &b);
  const int q0 = (grid_blocks(p.order) - 1 - block) * 256, hkv = hq / c.E;
  int32_t* status = c.status;
  int alo, ahi, blo, bhi;
  key_tiles(c, b, q0, &alo, &ahi);
  key_tiles(c, b, q0 + 128, &blo, &bhi);
  const bool has_a = alo < ahi, has_b = blo < bhi;
  // every tile that A or B waits for is issued, even if the caller's starts descend
  const int j0 = has_a && has_b ? min(alo, blo) : has_a ? alo : blo, j1 = has_b ? bhi : ahi;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&pv_done[i], 1);
      mbar_init(&o_done[i], 1);
    }
    for (int i = 0; i < NS; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_holder, 512);
    tmem_relinquish();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&tmq);
    prefetch_tmap(&tmk);
    prefetch_tmap(&tmv);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;

  if (warp == 0) {
    if (lane == 0) {
      if (has_a) {
        mbar_expect_tx(&q_full[0], TB);
        load_rows<HD, 128>(q_s, &tmq, hq, q0, b, &q_full[0]);
      }
      for (int j = j0, i = 0; j < j1; ++j, ++i) {
        const int st = i % NS;
        const uint32_t ph = ((i / NS) - 1) & 1;
        if (i >= NS && !mbar_wait(&k_empty[st], ph, abort_flag, status)) break;
        mbar_expect_tx(&k_full[st], TB);
        load_rows<HD, 128>(k_s + st * TB, &tmk, hkv, j * KT, b, &k_full[st]);
        if (i == 0 && has_b) {
          mbar_expect_tx(&q_full[1], TB);
          load_rows<HD, 128>(q_s + TB, &tmq, hq, q0 + 128, b, &q_full[1]);
        }
        if (i >= NS && !mbar_wait(&v_empty[st], ph, abort_flag, status)) break;
        mbar_expect_tx(&v_full[st], TB);
        load_rows<HD, 128>(v_s + st * TB, &tmv, hkv, j * KT, b, &v_full[st]);
      }
    }
  } else if (warp == 1) {
    constexpr uint32_t kIdS = idesc_f16(128, KT, Pack2<T>::kFmt, 0, 0);
    constexpr uint32_t kIdO = idesc_f16(128, HD, Pack2<T>::kFmt, 0, 1);
    const uint32_t qd0 = desc_lo(q_s, 16), kd0 = desc_lo(k_s, 16), vd0 = desc_lo(v_s, BLK);
    const uint32_t tm = uniform(tmem);
    const int ua0 = uniform(has_a ? alo : 0), ua1 = uniform(has_a ? ahi : 0), ub0 = uniform(has_b ? blo : 0),
              ub1 = uniform(has_b ? bhi : 0), u0 = uniform(j0), u1 = uniform(j1);
    const bool leader = elect_one();
    int np0 = 0, np1 = 0;
    auto issue_s = [&](int x, int np, int st) -> bool {  // behind the tile's np products with V
      if (!kOwnP && np > 0) {
        if (!mbar_wait(&pv_done[x], (np - 1) & 1, abort_flag, status)) return false;
        tc_fence_after();
      }
      if (leader) {
        mma_tile_ss<HD>(tm + x * 128, qd0 + ((x * TB) >> 4), kd0 + ((st * TB) >> 4), kIdS);
        mma_commit(&s_full[x]);
      }
      return true;
    };
    auto issue_pv = [&](int x, int& np, int st) -> bool {
      if (!mbar_wait(&p_full[x], np & 1, abort_flag, status)) return false;
      tc_fence_after();
      if (leader) {
        mma_tile_ts<8, 64>(tm + 256 + x * HD, tm + kColP + x * kStepP, vd0 + ((st * TB) >> 4), kIdO, np > 0 ? 1u : 0u);
        if constexpr (!kOwnP) mma_commit(&pv_done[x]);
      }
      ++np;
      return true;
    };
    auto commit = [&](uint64_t* bar) {
      if (leader) mma_commit(bar);
    };
    bool ok = u0 < u1;
    if (ok) ok = mbar_wait(&k_full[0], 0, abort_flag, status);
    if (ok && ua0 < ua1) ok = mbar_wait(&q_full[0], 0, abort_flag, status);
    if (ok && ub0 < ub1) ok = mbar_wait(&q_full[1], 0, abort_flag, status);
    tc_fence_after();
    if (ok) {
      if (u0 >= ua0 && u0 < ua1) issue_s(0, 0, 0);
      if (u0 >= ub0 && u0 < ub1) issue_s(1, 0, 0);
      commit(&k_empty[0]);
    }
    for (int j = u0, i = 0; ok && j < u1; ++j, ++i) {
      const int st = i % NS, st1 = (i + 1) % NS;
      if (j + 1 < u1 && !mbar_wait(&k_full[st1], ((i + 1) / NS) & 1, abort_flag, status)) break;
      if (!mbar_wait(&v_full[st], (i / NS) & 1, abort_flag, status)) break;
      if (j >= ua0 && j < ua1 && !issue_pv(0, np0, st)) break;
      if (j + 1 >= ua0 && j + 1 < ua1 && !issue_s(0, np0, st1)) break;
      if (ua0 < ua1 && j + 1 == ua1) commit(&o_done[0]);
      if (j >= ub0 && j < ub1 && !issue_pv(1, np1, st)) break;
      commit(&v_empty[st]);
      if (j + 1 >= ub0 && j + 1 < ub1 && !issue_s(1, np1, st1)) break;
      if (ub0 < ub1 && j + 1 == ub1) commit(&o_done[1]);
      if (j + 1 < u1) commit(&k_empty[st1]);
    }
  } else if (warp >= 4) {
    const int x = (warp - 4) >> 2;
    const int r = threadIdx.x - 128 - 128 * x;
    const int q = q0 + 128 * x + r;
    const bool row_ok = q < c.N;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lane_base + x * 128;
    const uint32_t o_addr = tmem + lane_base + 256 + x * HD;
    const uint32_t p_addr = tmem + lane_base + kColP + x * kStepP;
    const int first = row_ok ? first_key(c, b, q) : 1, end = row_ok ? q + 1 : 0;
    const int lo = x ? blo : alo, hi = x ? bhi : ahi;
    float m_used = -INFINITY, ell = 0.f, kept = 0.f;  // sums of the weights, and of the rounded ones
    bool alive = true;
    int n = 0;
    for (int j = lo; j < hi; ++j, ++n) {
      alive = __all_sync(0xffffffffu, mbar_wait(&s_full[x], n & 1, abort_flag, status));
      if (!alive) break;
      tc_fence_after();
      const int jlo = first - j * KT, jhi = end - j * KT;
      const bool interior = __all_sync(0xffffffffu, jlo <= 0 && jhi >= KT);
      float umax = -INFINITY, amax = 0.f;
#pragma unroll 1
      for (int c0 = 0; c0 < KT; c0 += 64) {
        float sv[64];
        tmem_ld32(s_addr + c0, sv);
        tmem_ld32(s_addr + c0 + 32, sv + 32);
        tmem_wait_ld();
        float m0 = -INFINITY, m1 = -INFINITY;
        if (interior) {
#pragma unroll
          for (int i = 0; i < 64; i += 4) {
            m0 = fmax3(m0, sv[i], sv[i + 1]);
            m1 = fmax3(m1, sv[i + 2], sv[i + 3]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 64; i += 2) {
            const float a0 = (c0 + i >= jlo && c0 + i < jhi) ? sv[i] : -INFINITY;
            const float a1 = (c0 + i + 1 >= jlo && c0 + i + 1 < jhi) ? sv[i + 1] : -INFINITY;
            if ((i >> 1) & 1) m1 = fmax3(m1, a0, a1);
            else m0 = fmax3(m0, a0, a1);
          }
        }
        umax = fmax3(umax, m0, m1);
        if constexpr (CAP) {
          float a0 = 0.f, a1 = 0.f;
#pragma unroll
          for (int i = 0; i < 64; i += 4) {
            a0 = fmax3(a0, fabsf(sv[i]), fabsf(sv[i + 1]));
            a1 = fmax3(a1, fabsf(sv[i + 2]), fabsf(sv[i + 3]));
          }
          amax = fmax3(amax, a0, a1);
        }
      }
      int mode = kPlain;
      if constexpr (CAP) {
        const float ay = amax * p.kq;
        mode = __all_sync(0xffffffffu, ay <= p.top5) ? kS5 : __all_sync(0xffffffffu, ay <= p.top9) ? kS9 : kTanh;
      }
      float mx = -INFINITY;
      if (umax > -INFINITY) {
        if constexpr (!CAP) mx = logit2<kPlain>(umax, p);
        else mx = mode == kS5 ? logit2<kS5>(umax, p) : mode == kS9 ? logit2<kS9>(umax, p) : logit2<kTanh>(umax, p);
      }
      bool rescale = false;
      float alpha = 1.f;
      if (mx > -INFINITY) {
        if (m_used == -INFINITY) {
          m_used = mx;
        } else if (mx > m_used + kLazy) {
          alpha = exp2_fast(m_used - mx);
          m_used = mx;
          rescale = true;
        }
      }
      if (__any_sync(0xffffffffu, rescale)) {
        ell *= alpha;
        kept *= alpha;
#pragma unroll 1
        for (int d = 0; d < HD; d += 32) {
          float ov[32];
          tmem_ld32(o_addr + d, ov);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) ov[i] *= alpha;
          tmem_st32(o_addr + d, ov);
        }
      }
      const float m_eff = m_used > -INFINITY ? m_used : 0.f;
      float2 sum = f2(0.f), held = f2(0.f);
#pragma unroll 1
      for (int c0 = 0; c0 < KT; c0 += 64) {
        float sv[64];
        uint32_t pw[32];
        tmem_ld32(s_addr + c0, sv);
        tmem_ld32(s_addr + c0 + 32, sv + 32);
        tmem_wait_ld();
        if constexpr (!CAP) {
          half_p<T, kPlain>(interior, sv, c0, p, m_eff, jlo, jhi, pw, &sum, &held);
        } else {
          if (mode == kS5) half_p<T, kS5>(interior, sv, c0, p, m_eff, jlo, jhi, pw, &sum, &held);
          else if (mode == kS9) half_p<T, kS9>(interior, sv, c0, p, m_eff, jlo, jhi, pw, &sum, &held);
          else half_p<T, kTanh>(interior, sv, c0, p, m_eff, jlo, jhi, pw, &sum, &held);
        }
        tmem_st16u(p_addr + c0 / 2, pw);
        tmem_st16u(p_addr + c0 / 2 + 16, pw + 16);
      }
      ell += sum.x + sum.y;
      kept += held.x + held.y;
      tmem_wait_st();
      tc_fence_before();
      warp_arrive(&p_full[x], lane);
    }
    if (alive && n > 0) alive = __all_sync(0xffffffffu, mbar_wait(&o_done[x], 0, abort_flag, status));
    if (alive) {
      tc_fence_after();
      const float inv = kept != 0.f ? 1.f / kept : 0.f;
      const int64_t at = (((int64_t)b * c.N + q) * c.Hq + hq) * HD;
      T* out = static_cast<T*>(c.out) + at;
      T* low = c.out_low ? static_cast<T*>(c.out_low) + at : nullptr;
#pragma unroll 1
      for (int d = 0; d < HD; d += 32) {
        float ov[32];
        if (n > 0) {
          tmem_ld32(o_addr + d, ov);
          tmem_wait_ld();
        }
        // a row without keys multiplied masked columns only: its zeros are written as such
        if (n == 0 || ell == 0.f) {
#pragma unroll
          for (int i = 0; i < 32; ++i) ov[i] = 0.f;
        }
        if (row_ok) {
#pragma unroll
          for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(out + d + i * 8) = pack8<T>(ov + i * 8, inv);
          if (low) {
#pragma unroll
            for (int i = 0; i < 32; ++i) ov[i] = ov[i] * inv - round_to<T>(ov[i] * inv);
#pragma unroll
            for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(low + d + i * 8) = pack8<T>(ov + i * 8, 1.f);
          }
        }
      }
      if (row_ok)
        c.lse[((int64_t)b * c.N + q) * c.Hq + hq] = ell != 0.f ? (m_used + log2f(ell)) * kLn2 : -INFINITY;
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
int launch_fwd(const CausalParams& a, int dtype, cudaStream_t st) {
  CUtensorMap mq, mk, mv;
  if (int rc = make_map_strided(&mq, a.q, dtype, a.B, a.N, a.Hq, HD, a.q_sb, a.q_sn, a.q_sh, 128)) return rc;
  if (int rc = make_map_strided(&mk, a.k, dtype, a.B, a.N, a.Hkv, HD, a.k_sb, a.k_sn, a.k_sh, KT)) return rc;
  if (int rc = make_map_strided(&mv, a.v, dtype, a.B, a.N, a.Hkv, HD, a.v_sb, a.v_sn, a.v_sh, KT)) return rc;
  FwdParams p;
  p.c = a;
  const double cap = a.has_cap ? (double)a.cap : 1.0;
  const double kq = a.has_cap ? (double)a.scale / cap : (double)a.scale * 1.4426950408889634;
  const double kc = cap * 1.4426950408889634;
  p.kq = (float)kq;
  p.kc = (float)kc;
  p.e1 = (float)(kc * kq);
  p.e3 = (float)(kc * kT3 * kq * kq * kq);
  p.e5 = (float)(kc * kT5 * kq * kq * kq * kq * kq);
  p.e7 = (float)(kc * kT7 * kq * kq * kq * kq * kq * kq * kq);
  p.e9 = (float)(kc * kT9 * kq * kq * kq * kq * kq * kq * kq * kq * kq);
  p.top5 = std::isnormal(p.e1) && std::isnormal(p.e3) && std::isnormal(p.e5) ? kPoly5 : -1.f;
  p.top9 = p.top5 > 0.f && std::isnormal(p.e7) && std::isnormal(p.e9) ? kPoly9 : -1.f;
  auto k = causal_fwd_kernel<T, HD, CAP>;
  constexpr int smem = FwdSmem<HD>::kBytes;
  if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return TC_ERR_CUDA;
  const dim3 grid = grid_order((a.N + 255) / 256, a.Hq, a.B, (int64_t)a.B * a.N * a.Hkv * HD * 4, &p.order);
  k<<<grid, kFwdThreads, smem, st>>>(mq, mk, mv, p);
  return launch_status();
}

template <typename T>
int dispatch_fwd(const CausalParams& a, int dtype, cudaStream_t st) {
  if (a.Dk == 128)
    return a.has_cap ? launch_fwd<T, 128, true>(a, dtype, st) : launch_fwd<T, 128, false>(a, dtype, st);
  return a.has_cap ? launch_fwd<T, 64, true>(a, dtype, st) : launch_fwd<T, 64, false>(a, dtype, st);
}

}  // namespace

// The results leave as 16-byte pieces (out_low may be null).
bool causal_tc_supported(const CausalParams& p, int dtype) {
  return ctc::tc_shape(p, dtype) && ((uintptr_t)p.out | (uintptr_t)p.out_low) % 16 == 0;
}

int causal_fwd_tc(const CausalParams& p, int dtype, cudaStream_t st) {
  return dtype == TC_BF16 ? dispatch_fwd<__nv_bfloat16>(p, dtype, st) : dispatch_fwd<__half>(p, dtype, st);
}

}  // namespace tc

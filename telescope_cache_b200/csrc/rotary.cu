// Rotary positions of a token's query and key heads in one pass (sm_100a).
//
// Each pair (x1, x2) of a head's first R dims turns by the angle of its
// position: y1 = x1 c - x2 s, y2 = x2 c + x1 s, with c, s rows of the caller's
// fp32 tables (which carry any scaling); dims from R on pass through.  The pair
// is (i, i + R / 2) in the half layout and (2 i, 2 i + 1) in the interleaved
// one.  Each product and sum is rounded on its own in fp32 and the result once
// to the element type, so the same definition gives the same bits in the cache
// write of kv_cache.cu.  The VJP is the same map with s negated.
//
// Bound by HBM: every element is read once and written once (the tables are a
// few MB and stay in L2).  A thread owns one 16-byte chunk of a head (the half
// layout: the two chunks of eight pairs) for kHeads heads of one token, so that
// the tables are loaded once for them and kHeads (half: 2 kHeads) loads are in
// flight per thread.  q and k are read in place through their strides (views
// of a fused projection need no copy) and written dense.  Measured: 0.67 GB (4 x
// 16384 tokens of 16 + 4 heads of 128, f16) in 109 us, 6.2 TB/s, 0.94 of a copy's
// rate; one token of 64 sequences 2.5 us, of which nearly all is latency.
#include "common.cuh"
#include "rotary.cuh"

using namespace tc;

namespace {

struct RotaryParams {
  int64_t tokens;  // B * N
  int N, Hq, Hk, D, R, interleaved, n_pos;
  float sgn;       // -1: inverse rotation
  const void* q;
  const void* k;
  int64_t q_sb, q_sn, q_sh, k_sb, k_sn, k_sh;
  void* qo;
  void* ko;
  const float* cos_t;
  const float* sin_t;
  const int32_t* pos;
  int64_t pos_sb;
  int units, groups;  // units per head, head groups per token
};

// 8 or 16 bytes of VE elements as floats.
template <typename T, int VE> struct Vec {
  using Raw = typename std::conditional<sizeof(T) * VE == 16, uint4, uint2>::type;
  Raw raw;
  __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const Raw*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Raw*>(p) = raw; }
  __device__ __forceinline__ float get(int i) const { return to_f(reinterpret_cast<const T*>(&raw)[i]); }
  __device__ __forceinline__ void set(int i, float v) { reinterpret_cast<T*>(&raw)[i] = from_f<T>(v); }
};

template <int N>
__device__ __forceinline__ void load_f(float* dst, const float* src) {
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    if constexpr (N >= 4) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(src + i));
      dst[i] = v.x, dst[i + 1] = v.y, dst[i + 2] = v.z, dst[i + 3] = v.w;
    } else {
      const float2 v = __ldg(reinterpret_cast<const float2*>(src + i));
      dst[i] = v.x, dst[i + 1] = v.y;
    }
  }
}

// Vector path.  IL: interleaved layout.  NH heads per thread.
template <typename T, int VE, bool IL, int NH>
__global__ void __launch_bounds__(256) rotary_vec(RotaryParams p) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t per = (int64_t)p.units * p.groups;
  const int64_t tok = i / per;
  if (tok >= p.tokens) return;
  const int rest = (int)(i - tok * per);
  const int u = rest % p.units, hg = rest / p.units;
  const int64_t b = tok / p.N;
  const int n = (int)(tok - b * p.N);
  const int half = p.R / 2, H = p.Hq + p.Hk;
  const int rot_units = IL ? p.R / VE : half / VE;  // units past them pass through
  const bool rot = u < rot_units;
  const int d0 = IL ? u * VE : (rot ? u * VE : p.R + (u - rot_units) * VE);
  constexpr bool kTwo = !IL;

  const T* src[NH];
  T* dst[NH];
  Vec<T, VE> a[NH], c[kTwo ? NH : 1];
#pragma unroll
  for (int j = 0; j < NH; ++j) {
    const int h = hg + j * p.groups;
    src[j] = nullptr;
    if (h >= H) continue;
    if (h < p.Hq) {
      src[j] = static_cast<const T*>(p.q) + b * p.q_sb + n * p.q_sn + h * p.q_sh + d0;
      dst[j] = static_cast<T*>(p.qo) + (tok * p.Hq + h) * p.D + d0;
    } else {
      src[j] = static_cast<const T*>(p.k) + b * p.k_sb + n * p.k_sn + (h - p.Hq) * p.k_sh + d0;
      dst[j] = static_cast<T*>(p.ko) + (tok * p.Hk + h - p.Hq) * p.D + d0;
    }
    a[j].load(src[j]);
    if constexpr (kTwo) {
      if (rot) c[j].load(src[j] + half);
    }
  }
  if (rot) {
    constexpr int NC = IL ? VE / 2 : VE;
    float cs[NC], sn[NC];
    const int pos = p.pos ? p.pos[b * p.pos_sb + n] : n;
    if (pos >= 0 && pos < p.n_pos) {
      const int64_t row = (int64_t)pos * half + (IL ? d0 / 2 : d0);
      load_f<NC>(cs, p.cos_t + row);
      load_f<NC>(sn, p.sin_t + row);
    } else {
#pragma unroll
      for (int x = 0; x < NC; ++x) cs[x] = sn[x] = NAN;  // a position outside the tables
    }
#pragma unroll
    for (int j = 0; j < NH; ++j) {
#pragma unroll
      for (int x = 0; x < NC; ++x) {
        const float s = p.sgn * sn[x];
        float y1, y2;
        if constexpr (IL) {
          rotate_pair(a[j].get(2 * x), a[j].get(2 * x + 1), cs[x], s, &y1, &y2);
          a[j].set(2 * x, y1);
          a[j].set(2 * x + 1, y2);
        } else {
          rotate_pair(a[j].get(x), c[j].get(x), cs[x], s, &y1, &y2);
          a[j].set(x, y1);
          c[j].set(x, y2);
        }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < NH; ++j) {
    if (!src[j]) continue;
    a[j].store(dst[j]);
    if constexpr (kTwo) {
      if (rot) c[j].store(dst[j] + half);
    }
  }
}

// Any sizes and strides: a thread per pair, or per passed-through element.
template <typename T>
__global__ void __launch_bounds__(256) rotary_scalar(RotaryParams p) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t per = (int64_t)p.units * (p.Hq + p.Hk);
  const int64_t tok = i / per;
  if (tok >= p.tokens) return;
  const int rest = (int)(i - tok * per);
  const int u = rest % p.units, h = rest / p.units;
  const int64_t b = tok / p.N;
  const int n = (int)(tok - b * p.N);
  const int half = p.R / 2;
  const T* src;
  T* dst;
  if (h < p.Hq) {
    src = static_cast<const T*>(p.q) + b * p.q_sb + n * p.q_sn + h * p.q_sh;
    dst = static_cast<T*>(p.qo) + (tok * p.Hq + h) * p.D;
  } else {
    src = static_cast<const T*>(p.k) + b * p.k_sb + n * p.k_sn + (h - p.Hq) * p.k_sh;
    dst = static_cast<T*>(p.ko) + (tok * p.Hk + h - p.Hq) * p.D;
  }
  if (u >= half) {
    dst[u + half] = src[u + half];
    return;
  }
  const int i1 = p.interleaved ? 2 * u : u, i2 = p.interleaved ? 2 * u + 1 : u + half;
  const int pos = p.pos ? p.pos[b * p.pos_sb + n] : n;
  float c = NAN, s = NAN, y1, y2;
  if (pos >= 0 && pos < p.n_pos) {
    c = p.cos_t[(int64_t)pos * half + u];
    s = p.sgn * p.sin_t[(int64_t)pos * half + u];
  }
  rotate_pair(to_f(src[i1]), to_f(src[i2]), c, s, &y1, &y2);
  dst[i1] = from_f<T>(y1);
  dst[i2] = from_f<T>(y2);
}

inline bool fits(int64_t v, int m) { return v % m == 0; }

// Whether every chunk of VE elements of T starts on its own size in bytes.
template <typename T, int VE>
bool vec_ok(const RotaryParams& p) {
  const int unit = p.interleaved ? p.R : p.R / 2;
  if (!fits(unit, VE) || !fits(p.D, VE) || !fits((int64_t)(uintptr_t)p.cos_t, 16) || !fits((int64_t)(uintptr_t)p.sin_t, 16) ||
      !fits(p.R / 2, 4))
    return false;
  const int bytes = VE * (int)sizeof(T);
  const bool q_ok = fits((int64_t)(uintptr_t)p.q, bytes) && fits((int64_t)(uintptr_t)p.qo, bytes) && fits(p.q_sb, VE) &&
                    fits(p.q_sn, VE) && fits(p.q_sh, VE);
  const bool k_ok = p.Hk == 0 || (fits((int64_t)(uintptr_t)p.k, bytes) && fits((int64_t)(uintptr_t)p.ko, bytes) &&
                                  fits(p.k_sb, VE) && fits(p.k_sn, VE) && fits(p.k_sh, VE));
  return q_ok && k_ok;
}

constexpr int kHeads = 4;

template <typename T, int VE, bool IL>
int launch_vec(RotaryParams p, cudaStream_t st) {
  const int H = p.Hq + p.Hk;
  p.units = IL ? p.D / VE : p.R / 2 / VE + (p.D - p.R) / VE;
  // one head per thread until that fills the card (148 SMs x 2048 threads):
  // with fewer threads than that a call is bound by its latency
  const bool wide = p.tokens * H * p.units >= 148 * 2048;
  p.groups = wide ? (H + kHeads - 1) / kHeads : H;
  const int64_t n = p.tokens * p.units * p.groups;
  const int block = wide ? 256 : 128;
  const int64_t grid = (n + block - 1) / block;
  if (grid > INT32_MAX) return TC_ERR_UNSUPPORTED;
  if (wide) rotary_vec<T, VE, IL, kHeads><<<(unsigned)grid, block, 0, st>>>(p);
  else rotary_vec<T, VE, IL, 1><<<(unsigned)grid, block, 0, st>>>(p);
  return launch_status();
}

template <typename T>
int launch_rotary(RotaryParams p, cudaStream_t st) {
  constexpr int V16 = 16 / sizeof(T);
  if (vec_ok<T, V16>(p))
    return p.interleaved ? launch_vec<T, V16, true>(p, st) : launch_vec<T, V16, false>(p, st);
  if constexpr (sizeof(T) == 2) {
    if (vec_ok<T, 4>(p)) return p.interleaved ? launch_vec<T, 4, true>(p, st) : launch_vec<T, 4, false>(p, st);
  }
  p.units = p.R / 2 + p.D - p.R;
  const int64_t n = p.tokens * p.units * (p.Hq + p.Hk);
  const int64_t grid = (n + 255) / 256;
  if (grid > INT32_MAX) return TC_ERR_UNSUPPORTED;
  rotary_scalar<T><<<(unsigned)grid, 256, 0, st>>>(p);
  return launch_status();
}

}  // namespace

extern "C" int tc_rotary(const tc_rotary_args* a, void* stream) {
  if (!a || a->B < 0 || a->N < 0 || a->Hq < 0 || a->Hk < 0 || a->D <= 0 || a->R < 0 || a->R > a->D || a->R % 2)
    return TC_ERR_ARG;
  if ((int64_t)a->B * a->N == 0 || a->Hq + a->Hk == 0) return TC_OK;
  if (a->R > 0 && (!a->cos_t || !a->sin_t || a->n_pos <= 0)) return TC_ERR_ARG;
  if ((a->Hq && (!a->q || !a->q_out)) || (a->Hk && (!a->k || !a->k_out))) return TC_ERR_ARG;
  RotaryParams p;
  p.tokens = (int64_t)a->B * a->N;
  p.N = a->N;
  p.Hq = a->Hq;
  p.Hk = a->Hk;
  p.D = a->D;
  p.R = a->R;
  p.interleaved = a->interleaved != 0;
  p.n_pos = a->n_pos;
  p.sgn = a->inverse ? -1.f : 1.f;
  p.q = a->q;
  p.k = a->k;
  p.q_sb = a->q_stride_b;
  p.q_sn = a->q_stride_n;
  p.q_sh = a->q_stride_h;
  p.k_sb = a->k_stride_b;
  p.k_sn = a->k_stride_n;
  p.k_sh = a->k_stride_h;
  p.qo = a->q_out;
  p.ko = a->k_out;
  p.cos_t = a->cos_t;
  p.sin_t = a->sin_t;
  p.pos = a->positions;
  p.pos_sb = a->pos_stride_b;
  p.units = p.groups = 0;
  TC_DISPATCH(a->dtype, T, return launch_rotary<T>(p, (cudaStream_t)stream));
}

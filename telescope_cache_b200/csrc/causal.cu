// Packed causal attention: the C entries, the example bounds, Delta, and the
// CUDA-core kernels (fp32, and the head dims that the tensor-core kernels of
// causal_fwd.cu and causal_bwd.cu do not cover).
//
//   X_ij = scale q_i . k_j,  S = c tanh(X / c) (or X),  i sees starts[i] <= j <= i
//   P = exp(S - lse),  out = P V
//   dS = P (dO V^T - Delta),  Delta = rowsum(dO * out) - dlse,  dX = dS (1 - tanh^2)
//   dQ = scale dX K,  dK = scale dX^T Q,  dV = P^T dO
#include <cmath>

#include "causal.cuh"

using namespace tc;

namespace {

// ---------------------------------------------------------------------------
// example bounds
// ---------------------------------------------------------------------------
// A CTA covers kBoundTok tokens of a row, four consecutive ones a thread.  The run
// that enters it (and the one that leaves it) may be long: the CTA looks for its
// start (end) 16 tokens a thread at a time.  A few us at 16384 tokens.  (One CTA
// per row: 31 us.)
constexpr int kBoundThreads = 512, kBoundTok = 4 * kBoundThreads, kReach = 16;
// Largest (FORWARD: smallest) run start over [lo, hi), -1 (N) where there is none;
// the same for every thread.
template <bool FORWARD, typename Id>
__device__ int edge(const Id* id, int lo, int hi, int N, int* box) {
  int best = FORWARD ? N : -1;
  Id v[kReach], w[kReach];
#pragma unroll
  for (int k = 0; k < kReach; ++k) {
    const int n = lo + threadIdx.x + k * kBoundThreads;
    const bool in = n < hi;
    v[k] = in ? id[n] : 0;
    w[k] = in && n > 0 ? id[n - 1] : 0;
  }
#pragma unroll
  for (int k = 0; k < kReach; ++k) {
    const int n = lo + threadIdx.x + k * kBoundThreads;
    if (n < hi && (n == 0 || v[k] != w[k])) best = FORWARD ? min(best, n) : max(best, n);
  }
  __syncthreads();
  if (threadIdx.x == 0) *box = FORWARD ? N : -1;
  __syncthreads();
  if (FORWARD ? best < N : best >= 0) {
    if (FORWARD) atomicMin(box, best);
    else atomicMax(box, best);
  }
  __syncthreads();
  return *box;
}

template <typename Id>
__global__ void __launch_bounds__(kBoundThreads) bounds_kernel(int N, const Id* seq, int32_t* starts, int32_t* ends) {
  __shared__ int last_w[kBoundThreads / 32], first_w[kBoundThreads / 32], box;
  const int64_t row = (int64_t)blockIdx.y * N;
  const Id* id = seq + row;
  const int c0 = blockIdx.x * kBoundTok, c1 = min(N, c0 + kBoundTok);
  const int n0 = c0 + 4 * threadIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Id v[5];  // id[n0 - 1 .. n0 + 3]
#pragma unroll
  for (int k = 0; k < 5; ++k) {
    const int n = n0 - 1 + k;
    v[k] = n >= 0 && n < N ? id[n] : 0;
  }
  int first = N, last = -1;  // run starts among the thread's tokens
#pragma unroll
  for (int k = 3; k >= 0; --k)
    if (n0 + k < c1 && (n0 + k == 0 || v[k + 1] != v[k])) first = n0 + k;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (n0 + k < c1 && (n0 + k == 0 || v[k + 1] != v[k])) last = n0 + k;
  // exclusive scans: the largest start before this thread, the smallest after it
  int before = last, after = first;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, before, o), y = __shfl_down_sync(0xffffffffu, after, o);
    if (lane >= o) before = max(before, x);
    if (lane + o < 32) after = min(after, y);
  }
  if (lane == 31) last_w[warp] = before;
  if (lane == 0) first_w[warp] = after;
  before = __shfl_up_sync(0xffffffffu, before, 1);
  after = __shfl_down_sync(0xffffffffu, after, 1);
  if (lane == 0) before = -1;
  if (lane == 31) after = N;
  __syncthreads();
  for (int w = 0; w < warp; ++w) before = max(before, last_w[w]);
  for (int w = warp + 1; w < kBoundThreads / 32; ++w) after = min(after, first_w[w]);
  int first_all = N;
  for (int w = 0; w < kBoundThreads / 32; ++w) first_all = min(first_all, first_w[w]);
  // the run that enters the CTA
  int enter = -1;
  if (first_all > c0)  // uniform
    for (int hi = c0; hi > 0 && enter < 0;) {
      const int lo = max(0, hi - kReach * kBoundThreads);
      enter = edge<false>(id, lo, hi, N, &box);
      hi = lo;
    }
  // and where the last one ends
  int leave = N;
  for (int lo = c1; lo < N && leave == N;) {
    const int hi = min(N, lo + kReach * kBoundThreads);
    leave = edge<true>(id, lo, hi, N, &box);
    lo = hi;
  }
  int start = before >= 0 ? before : enter;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int n = n0 + k;
    if (n >= c1) break;
    if (n == 0 || v[k + 1] != v[k]) start = n;
    starts[row + n] = v[k + 1] < 0 ? n + 1 : start;
  }
  int end = after < N ? after : leave;
#pragma unroll
  for (int k = 3; k >= 0; --k) {
    const int n = n0 + k;
    if (n >= c1) continue;
    ends[row + n] = v[k + 1] < 0 ? n : end;
    if (n == 0 || v[k + 1] != v[k]) end = n;
  }
}

template <typename Id>
int launch_bounds(int32_t B, int32_t N, const Id* seq_idx, int32_t* starts, int32_t* ends, cudaStream_t st) {
  if (B < 0 || N < 0) return TC_ERR_ARG;
  if ((int64_t)B * N == 0) return TC_OK;
  if (!seq_idx || !starts || !ends) return TC_ERR_ARG;
  if (B > 65535) return TC_ERR_UNSUPPORTED;
  bounds_kernel<<<dim3((N + kBoundTok - 1) / kBoundTok, B), kBoundThreads, 0, st>>>(N, seq_idx, starts, ends);
  return launch_status();
}

// ---------------------------------------------------------------------------
// Delta = rowsum(dO * out) - dlse, with out to twice its bits where its rounding's
// leftovers were kept: the rounding of out alone puts an error of 2^-9 of a row's
// |dO| |out| into every dX of the row (bf16, 1000 tokens: dQ off by 2.4e-3 of its norm
// with and without for normal data, by 2.4e-3 and 1.5e-2 for values of mean 8; 1.7e-3
// are its own rounding and as much dX's)
// ---------------------------------------------------------------------------
// LANES lanes per row, 16 bytes of dO and out each (LANES 0: a warp per row of
// any length).  Bound by HBM.
template <typename T, int LANES>
__global__ void __launch_bounds__(256) delta_rows(CausalParams p, int64_t rows) {
  constexpr int L = LANES ? LANES : 32, VE = 16 / sizeof(T);
  const int64_t r = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / L;
  const int lane = threadIdx.x % L;
  float s = 0.f;
  if (r < rows) {
    const T* o = static_cast<const T*>(p.o) + r * p.Dv;
    const T* g = static_cast<const T*>(p.dout) + r * p.Dv;
    const T* low = p.o_low ? static_cast<const T*>(p.o_low) + r * p.Dv : nullptr;
    if constexpr (LANES) {
      const uint4 a = *reinterpret_cast<const uint4*>(o + lane * VE), c = *reinterpret_cast<const uint4*>(g + lane * VE);
      uint4 r = make_uint4(0u, 0u, 0u, 0u);
      if (low) r = *reinterpret_cast<const uint4*>(low + lane * VE);
#pragma unroll
      for (int i = 0; i < VE; ++i)
        s += (to_f(reinterpret_cast<const T*>(&a)[i]) + to_f(reinterpret_cast<const T*>(&r)[i])) *
             to_f(reinterpret_cast<const T*>(&c)[i]);
    } else {
      for (int d = lane; d < p.Dv; d += 32) s += (to_f(o[d]) + (low ? to_f(low[d]) : 0.f)) * to_f(g[d]);
    }
  }
#pragma unroll
  for (int x = L / 2; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
  if (r < rows && lane == 0) p.delta[r] = s - (p.dlse ? p.dlse[r] : 0.f);
}

template <typename T>
int launch_delta(const CausalParams& p, cudaStream_t st) {
  const int64_t rows = (int64_t)p.B * p.N * p.Hq;
  const bool vec = (uintptr_t)p.o % 16 == 0 && (uintptr_t)p.dout % 16 == 0 && (uintptr_t)p.o_low % 16 == 0;
  const int lanes = vec ? p.Dv * (int)sizeof(T) / 16 : 0;
  const bool fit = vec && p.Dv * (int)sizeof(T) % 16 == 0 && (lanes == 8 || lanes == 16 || lanes == 32);
  const int64_t grid = (rows * (fit ? lanes : 32) + 255) / 256;
  if (grid > INT32_MAX) return TC_ERR_UNSUPPORTED;
  if (!fit) delta_rows<T, 0><<<(unsigned)grid, 256, 0, st>>>(p, rows);
  else if (lanes == 8) delta_rows<T, 8><<<(unsigned)grid, 256, 0, st>>>(p, rows);
  else if (lanes == 16) delta_rows<T, 16><<<(unsigned)grid, 256, 0, st>>>(p, rows);
  else delta_rows<T, 32><<<(unsigned)grid, 256, 0, st>>>(p, rows);
  return launch_status();
}

// ---------------------------------------------------------------------------
// CUDA-core tiles.  A group of GT threads (16 across) works a TM x TN score tile:
// thread (ty, tx) owns its rows ty + GT/16 i and columns tx + 16 j, and output rows
// ty + GT/16 i with the four-wide columns 4 tx + 64 j of a DM-wide row.  Shared
// rows are DM + 4 floats, so that 16 lanes reading float4s of 16 rows meet no bank
// twice.  fp32 throughout with the accurate expf / tanhf.
//
// A CTA's G groups take the tiles of its block in turn, each with operands, a
// barrier and sums of its own, and the first one joins them at the end in the order
// of the groups: one group's products run while another loads or waits.  Bound by
// FMA issue and shared memory reads: 12 wavefronts of float4 reads for a warp's 64
// multiply-adds of 4 x 4 scores a thread (2 x 4: 10 for 32).  8.5 ms = 57 TFLOP/s
// for the backward of 32 heads of 64 and 4096 tokens (seven products of a triangle).
// ---------------------------------------------------------------------------
template <int TM_, int TN_, int DM_, int GT_, int G_> struct Tile {
  static constexpr int TM = TM_, TN = TN_, DM = DM_, GT = GT_, G = G_;
  static constexpr int RS = DM + 4;     // operand row stride
  static constexpr int PS = TN + 4;     // score row stride
  static constexpr int RW = GT / 16;    // rows a step of i covers
  static constexpr int R = TM / RW;     // rows per thread
  static constexpr int S = TN / 16;     // score columns per thread
  static constexpr int C = DM / 64;     // float4 output columns per thread
  static constexpr int NT = GT * G;
  static constexpr int kFetch = TN * DM / GT;  // elements of an operand tile per thread
  // backward: a lone group's next loads run under its own products (of several groups,
  // one loads under another's)
  static constexpr bool kAhead = G == 1;
  // floats of shared memory: of the CTA, and of each group
  static constexpr int fwd_all() { return TM * RS; }
  static constexpr int fwd_group() { return TN * RS + TM * PS; }
  static constexpr int bwd_all() { return 2 * TM * RS; }
  static constexpr int bwd_group() { return 2 * TN * RS + 2 * TM * PS; }
};

struct Place {
  int g, t, ty, tx;  // group, thread in it, its row and column
};
template <typename Z>
__device__ __forceinline__ Place place() {
  const int t = threadIdx.x % Z::GT;
  return {(int)threadIdx.x / Z::GT, t, t >> 4, t & 15};
}
template <typename Z>
__device__ __forceinline__ void group_sync(int g) {
  if constexpr (Z::G == 1) __syncthreads();
  else asm volatile("bar.sync %0, %1;" ::"r"(1 + g), "n"(Z::GT) : "memory");
}

// Elements d .. d + 3 of a D-element row, zeros past its end (and for a row that is
// not there); vec: rows start on 4 elements and are a multiple of 4 long.
template <typename T>
__device__ __forceinline__ float4 load4(const T* x, int d, int D, bool there, bool vec) {
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  if (vec) {
    if (there && d < D) {
      using Raw = typename std::conditional<sizeof(T) == 4, uint4, uint2>::type;
      const Raw r = *reinterpret_cast<const Raw*>(x + d);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = to_f(reinterpret_cast<const T*>(&r)[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (there && d + i < D) v[i] = to_f(x[d + i]);
  }
  return make_float4(v[0], v[1], v[2], v[3]);
}

// Rows [r0, r0 + ROWS) of a head, zeros outside [0, N) x [0, D), by THREADS threads.
// fetch_tile and put_tile (backward of one group): into registers, so that the loads
// run under products, and from there into shared memory.
template <typename T, typename Z>
__device__ __forceinline__ void fetch_tile(float4* r, const void* x, int64_t base, int64_t sn, int r0, int N, int D, int t,
                                           bool vec) {
  const T* src = static_cast<const T*>(x) + base;
#pragma unroll
  for (int j = 0; j < Z::kFetch / 4; ++j) {
    const int i = (t + j * Z::GT) * 4, row = r0 + i / Z::DM;
    r[j] = load4<T>(src + (int64_t)row * sn, i % Z::DM, D, row < N, vec);
  }
}
template <typename Z>
__device__ __forceinline__ void put_tile(float* s, const float4* r, int t) {
#pragma unroll
  for (int j = 0; j < Z::kFetch / 4; ++j) {
    const int i = (t + j * Z::GT) * 4;
    *reinterpret_cast<float4*>(s + i / Z::DM * Z::RS + i % Z::DM) = r[j];
  }
}
template <typename T, int ROWS, int DM, int THREADS>
__device__ __forceinline__ void load_tile(float* s, const void* x, int64_t base, int64_t sn, int r0, int N, int D, int t,
                                          bool vec) {
  const T* src = static_cast<const T*>(x) + base;
#pragma unroll 8
  for (int i = 4 * t; i < ROWS * DM; i += 4 * THREADS) {
    const int row = r0 + i / DM, d = i % DM;
    *reinterpret_cast<float4*>(s + i / DM * (DM + 4) + d) = load4<T>(src + (int64_t)row * sn, d, D, row < N, vec);
  }
}

// acc[i][j] = a row (ty + RW i) . b row (tx + 16 j)
template <typename Z>
__device__ __forceinline__ void dot_tile(const float* a, const float* b, int D, const Place& w, float (*acc)[Z::S]) {
#pragma unroll
  for (int i = 0; i < Z::R; ++i)
#pragma unroll
    for (int j = 0; j < Z::S; ++j) acc[i][j] = 0.f;
#pragma unroll 2
  for (int d = 0; d < D; d += 4) {
    float4 x[Z::R], y[Z::S];
#pragma unroll
    for (int i = 0; i < Z::R; ++i) x[i] = *reinterpret_cast<const float4*>(a + (w.ty + Z::RW * i) * Z::RS + d);
#pragma unroll
    for (int j = 0; j < Z::S; ++j) y[j] = *reinterpret_cast<const float4*>(b + (w.tx + 16 * j) * Z::RS + d);
#pragma unroll
    for (int i = 0; i < Z::R; ++i)
#pragma unroll
      for (int j = 0; j < Z::S; ++j)
        acc[i][j] += x[i].x * y[j].x + x[i].y * y[j].y + x[i].z * y[j].z + x[i].w * y[j].w;
  }
}

// acc[i][j] += sum_c f[ty + RW i][c] m[c][4 tx + 64 j ..]
template <typename Z>
__device__ __forceinline__ void mul_tile(const float* f, const float* m, const Place& w, float4 (*acc)[Z::C]) {
#pragma unroll 1
  for (int c = 0; c < Z::TN; c += 4) {
    float4 x[Z::R];
#pragma unroll
    for (int i = 0; i < Z::R; ++i) x[i] = *reinterpret_cast<const float4*>(f + (w.ty + Z::RW * i) * Z::PS + c);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
#pragma unroll
      for (int j = 0; j < Z::C; ++j) {
        const float4 y = *reinterpret_cast<const float4*>(m + (c + k) * Z::RS + 4 * w.tx + 64 * j);
#pragma unroll
        for (int i = 0; i < Z::R; ++i) {
          const float e = k == 0 ? x[i].x : k == 1 ? x[i].y : k == 2 ? x[i].z : x[i].w;
          acc[i][j].x += e * y.x;
          acc[i][j].y += e * y.y;
          acc[i][j].z += e * y.z;
          acc[i][j].w += e * y.w;
        }
      }
    }
  }
}

// Group g > 0 leaves `n` floats a thread in its own shared memory; behind a CTA
// barrier the first group reads them: value i of thread t at [i][t].
template <typename Z>
__device__ __forceinline__ float& left(float* group, int i, int t) { return group[i * Z::GT + t]; }

// Adds the other groups' acc to the first's, in order.  true: this thread is in
// the first group.
template <typename Z, int PER>
__device__ __forceinline__ bool join_sums(float* groups, int stride, const Place& w, float4 (*acc)[Z::C], int at) {
  if constexpr (Z::G > 1) {
    static_assert((PER + 1) * Z::R * Z::C * 4 * Z::GT <= Z::bwd_group(), "sums fit the group's operands");
    if (w.g > 0) {
      float* s = groups + w.g * stride;
#pragma unroll
      for (int i = 0; i < Z::R; ++i)
#pragma unroll
        for (int j = 0; j < Z::C; ++j) {
          const int k = at + (i * Z::C + j) * 4;
          left<Z>(s, k, w.t) = acc[i][j].x, left<Z>(s, k + 1, w.t) = acc[i][j].y;
          left<Z>(s, k + 2, w.t) = acc[i][j].z, left<Z>(s, k + 3, w.t) = acc[i][j].w;
        }
    }
    __syncthreads();
    if (w.g > 0) return false;
    for (int g = 1; g < Z::G; ++g) {
      float* s = groups + g * stride;
#pragma unroll
      for (int i = 0; i < Z::R; ++i)
#pragma unroll
        for (int j = 0; j < Z::C; ++j) {
          const int k = at + (i * Z::C + j) * 4;
          acc[i][j].x += left<Z>(s, k, w.t), acc[i][j].y += left<Z>(s, k + 1, w.t);
          acc[i][j].z += left<Z>(s, k + 2, w.t), acc[i][j].w += left<Z>(s, k + 3, w.t);
        }
    }
  }
  return true;
}

template <typename T, typename Z>
__device__ __forceinline__ void store_rows(T* out, int64_t row_stride, int r0, int N, int D, float mul, const Place& w,
                                           float4 (*acc)[Z::C], T* low = nullptr) {
#pragma unroll
  for (int i = 0; i < Z::R; ++i) {
    const int r = r0 + w.ty + Z::RW * i;
    if (r >= N) continue;
#pragma unroll
    for (int j = 0; j < Z::C; ++j) {
      const float v[4] = {acc[i][j].x, acc[i][j].y, acc[i][j].z, acc[i][j].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int d = 4 * w.tx + 64 * j + k;
        if (d >= D) continue;
        const T y = from_f<T>(v[k] * mul);
        out[(int64_t)r * row_stride + d] = y;
        if (low) low[(int64_t)r * row_stride + d] = from_f<T>(v[k] * mul - to_f(y));
      }
    }
  }
}

template <typename T, typename Z>
__global__ void __launch_bounds__(Z::NT) fwd_cores(CausalParams p) {
  constexpr int TM = Z::TM, TN = Z::TN, DM = Z::DM;
  extern __shared__ __align__(16) float sm[];
  const Place w = place<Z>();
  float* groups = sm + Z::fwd_all();
  float* q_s = sm;                               // [TM][RS]
  float* kv_s = groups + w.g * Z::fwd_group();     // [TN][RS] keys, then values
  float* p_s = kv_s + TN * Z::RS;                // [TM][PS]
  const int q0 = (gridDim.x - 1 - blockIdx.x) * TM, hq = blockIdx.y, b = blockIdx.z, hkv = hq / p.E;
  load_tile<T, TM, DM, Z::NT>(q_s, p.q, b * p.q_sb + hq * p.q_sh, p.q_sn, q0, p.N, p.Dk, threadIdx.x, p.vec4);
  int lo[Z::R];
  float m[Z::R], l[Z::R];
  float4 o[Z::R][Z::C];
#pragma unroll
  for (int i = 0; i < Z::R; ++i) {
    const int q = q0 + w.ty + Z::RW * i;
    lo[i] = q < p.N ? first_key(p, b, q) : p.N;
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int j = 0; j < Z::C; ++j) o[i][j] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  const int end = min(q0 + TM, p.N), begin = first_key(p, b, q0) / 16 * 16 + w.g * TN, step = Z::G * TN;
  const int64_t kb = b * p.k_sb + hkv * p.k_sh, vb = b * p.v_sb + hkv * p.v_sh;
  __syncthreads();
  for (int k0 = begin; k0 < end; k0 += step) {
    group_sync<Z>(w.g);
    load_tile<T, TN, DM, Z::GT>(kv_s, p.k, kb, p.k_sn, k0, p.N, p.Dk, w.t, p.vec4);
    group_sync<Z>(w.g);
    float s[Z::R][Z::S];
    dot_tile<Z>(q_s, kv_s, p.Dk, w, s);
#pragma unroll
    for (int i = 0; i < Z::R; ++i) {
      const int row = w.ty + Z::RW * i, q = q0 + row;
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < Z::S; ++j) {
        const int k = k0 + w.tx + 16 * j;
        float x = s[i][j] * p.scale;
        if (p.has_cap) x = p.cap * tanhf(x / p.cap);
        s[i][j] = k >= lo[i] && k <= q ? x : -INFINITY;
        mx = fmaxf(mx, s[i][j]);
      }
#pragma unroll
      for (int x = 8; x; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
      const float mn = fmaxf(m[i], mx), me = mn == -INFINITY ? 0.f : mn;
      const float c = expf(m[i] - me);
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < Z::S; ++j) {
        // a NaN score (a NaN in a visible key) stays one; a masked one is 0
        const float e = expf(s[i][j] - me);
        sum += e;
        p_s[row * Z::PS + w.tx + 16 * j] = e;
      }
#pragma unroll
      for (int x = 8; x; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
      l[i] = l[i] * c + sum;
      m[i] = mn;
#pragma unroll
      for (int j = 0; j < Z::C; ++j) o[i][j].x *= c, o[i][j].y *= c, o[i][j].z *= c, o[i][j].w *= c;
    }
    group_sync<Z>(w.g);
    load_tile<T, TN, DM, Z::GT>(kv_s, p.v, vb, p.v_sn, k0, p.N, p.Dv, w.t, p.vec4);
    group_sync<Z>(w.g);
    mul_tile<Z>(p_s, kv_s, w, o);
  }
  if constexpr (Z::G > 1) {
    // joint maximum, then sums and O weighted by it, in the order of the groups
    constexpr int kPer = 2 + 4 * Z::C;
    static_assert(Z::R * kPer * Z::GT <= Z::fwd_group(), "a group's state fits its operands");
    group_sync<Z>(w.g);
    if (w.g > 0) {
#pragma unroll
      for (int i = 0; i < Z::R; ++i) {
        left<Z>(kv_s, i * kPer, w.t) = m[i], left<Z>(kv_s, i * kPer + 1, w.t) = l[i];
#pragma unroll
        for (int j = 0; j < Z::C; ++j) {
          const int k = i * kPer + 2 + 4 * j;
          left<Z>(kv_s, k, w.t) = o[i][j].x, left<Z>(kv_s, k + 1, w.t) = o[i][j].y;
          left<Z>(kv_s, k + 2, w.t) = o[i][j].z, left<Z>(kv_s, k + 3, w.t) = o[i][j].w;
        }
      }
    }
    __syncthreads();
    if (w.g > 0) return;
#pragma unroll
    for (int i = 0; i < Z::R; ++i) {
      float mn = m[i];
      for (int g = 1; g < Z::G; ++g) mn = fmaxf(mn, left<Z>(groups + g * Z::fwd_group(), i * kPer, w.t));
      const float me = mn == -INFINITY ? 0.f : mn;
      const float c = expf(m[i] - me);
      l[i] *= c;
#pragma unroll
      for (int j = 0; j < Z::C; ++j) o[i][j].x *= c, o[i][j].y *= c, o[i][j].z *= c, o[i][j].w *= c;
      for (int g = 1; g < Z::G; ++g) {
        float* s = groups + g * Z::fwd_group();
        const float e = expf(left<Z>(s, i * kPer, w.t) - me);
        l[i] += e * left<Z>(s, i * kPer + 1, w.t);
#pragma unroll
        for (int j = 0; j < Z::C; ++j) {
          const int k = i * kPer + 2 + 4 * j;
          o[i][j].x += e * left<Z>(s, k, w.t), o[i][j].y += e * left<Z>(s, k + 1, w.t);
          o[i][j].z += e * left<Z>(s, k + 2, w.t), o[i][j].w += e * left<Z>(s, k + 3, w.t);
        }
      }
      m[i] = mn;
    }
  }
#pragma unroll
  for (int i = 0; i < Z::R; ++i) {
    const float inv = l[i] != 0.f ? 1.f / l[i] : 0.f;
#pragma unroll
    for (int j = 0; j < Z::C; ++j) o[i][j].x *= inv, o[i][j].y *= inv, o[i][j].z *= inv, o[i][j].w *= inv;
    const int q = q0 + w.ty + Z::RW * i;
    if (w.tx == 0 && q < p.N)
      p.lse[((int64_t)b * p.N + q) * p.Hq + hq] = l[i] != 0.f ? m[i] + logf(l[i]) : -INFINITY;
  }
  const int64_t at = ((int64_t)b * p.N * p.Hq + hq) * p.Dv;
  store_rows<T, Z>(static_cast<T*>(p.out) + at, (int64_t)p.Hq * p.Dv, q0, p.N, p.Dv, 1.f, w, o,
                   p.out_low ? static_cast<T*>(p.out_low) + at : nullptr);
}

// P and dX of a score tile whose rows are queries (ROWS_Q) or keys.
struct RowStat {
  float lse, delta;
  int lo, q;  // query q sees keys lo .. q
};
__device__ __forceinline__ RowStat row_stat(const CausalParams& p, int b, int hq, int q) {
  RowStat r{0.f, 0.f, 1, 0};  // sees nothing
  if (q < p.N) {
    const int64_t i = ((int64_t)b * p.N + q) * p.Hq + hq;
    r.lse = p.lse[i];
    r.delta = p.delta[i];
    r.lo = first_key(p, b, q);
    r.q = q;
  }
  return r;
}
__device__ __forceinline__ void grad_of(const CausalParams& p, const RowStat& r, int k, float s, float dp, float* pr,
                                        float* dx) {
  float x = s * p.scale, g = 1.f;
  if (p.has_cap) {
    const float t = tanhf(x / p.cap);
    x = p.cap * t;
    g = 1.f - t * t;
  }
  const bool see = k >= r.lo && k <= r.q;
  *pr = see ? expf(x - r.lse) : 0.f;
  *dx = see ? *pr * (dp - r.delta) * g : 0.f;
}

template <typename T, typename Z>
__device__ __forceinline__ void dq_cores(const CausalParams& p, float* sm, int q0, int hq, int b) {
  constexpr int TM = Z::TM, TN = Z::TN, DM = Z::DM;
  constexpr bool kAhead = Z::kAhead;
  const Place w = place<Z>();
  float* groups = sm + Z::bwd_all();
  float* q_s = sm;
  float* g_s = q_s + TM * Z::RS;
  float* k_s = groups + w.g * Z::bwd_group();
  float* v_s = k_s + TN * Z::RS;
  float* x_s = v_s + TN * Z::RS;
  const int hkv = hq / p.E;
  const int64_t gb = ((int64_t)b * p.N * p.Hq + hq) * p.Dv, gn = (int64_t)p.Hq * p.Dv;
  load_tile<T, TM, DM, Z::NT>(q_s, p.q, b * p.q_sb + hq * p.q_sh, p.q_sn, q0, p.N, p.Dk, threadIdx.x, p.vec4);
  load_tile<T, TM, DM, Z::NT>(g_s, p.dout, gb, gn, q0, p.N, p.Dv, threadIdx.x, p.vec4);
  RowStat st[Z::R];
  float4 acc[Z::R][Z::C];
#pragma unroll
  for (int i = 0; i < Z::R; ++i) {
    st[i] = row_stat(p, b, hq, q0 + w.ty + Z::RW * i);
#pragma unroll
    for (int j = 0; j < Z::C; ++j) acc[i][j] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  const int end = min(q0 + TM, p.N), begin = first_key(p, b, q0) / 16 * 16 + w.g * TN, step = Z::G * TN;
  const int64_t kb = b * p.k_sb + hkv * p.k_sh, vb = b * p.v_sb + hkv * p.v_sh;
  float4 kr[kAhead ? Z::kFetch / 4 : 1], vr[kAhead ? Z::kFetch / 4 : 1];
  if (kAhead && begin < end) {
    fetch_tile<T, Z>(kr, p.k, kb, p.k_sn, begin, p.N, p.Dk, w.t, p.vec4);
    fetch_tile<T, Z>(vr, p.v, vb, p.v_sn, begin, p.N, p.Dv, w.t, p.vec4);
  }
  __syncthreads();
  for (int k0 = begin; k0 < end; k0 += step) {
    group_sync<Z>(w.g);
    if constexpr (kAhead) {
      put_tile<Z>(k_s, kr, w.t);
      put_tile<Z>(v_s, vr, w.t);
    } else {
      load_tile<T, TN, DM, Z::GT>(k_s, p.k, kb, p.k_sn, k0, p.N, p.Dk, w.t, p.vec4);
      load_tile<T, TN, DM, Z::GT>(v_s, p.v, vb, p.v_sn, k0, p.N, p.Dv, w.t, p.vec4);
    }
    group_sync<Z>(w.g);
    if (kAhead && k0 + step < end) {
      fetch_tile<T, Z>(kr, p.k, kb, p.k_sn, k0 + step, p.N, p.Dk, w.t, p.vec4);
      fetch_tile<T, Z>(vr, p.v, vb, p.v_sn, k0 + step, p.N, p.Dv, w.t, p.vec4);
    }
    float s[Z::R][Z::S], d[Z::R][Z::S];
    dot_tile<Z>(q_s, k_s, p.Dk, w, s);
    dot_tile<Z>(g_s, v_s, p.Dv, w, d);
#pragma unroll
    for (int i = 0; i < Z::R; ++i)
#pragma unroll
      for (int j = 0; j < Z::S; ++j) {
        float pr, dx;
        grad_of(p, st[i], k0 + w.tx + 16 * j, s[i][j], d[i][j], &pr, &dx);
        x_s[(w.ty + Z::RW * i) * Z::PS + w.tx + 16 * j] = dx;
      }
    group_sync<Z>(w.g);
    mul_tile<Z>(x_s, k_s, w, acc);
  }
  group_sync<Z>(w.g);
  if (!join_sums<Z, 0>(groups, Z::bwd_group(), w, acc, 0)) return;
  store_rows<T, Z>(static_cast<T*>(p.dq) + ((int64_t)b * p.N * p.Hq + hq) * p.Dk, (int64_t)p.Hq * p.Dk, q0, p.N, p.Dk,
                   p.scale, w, acc);
}

// dK, dV of TM keys of one key head: the queries that see them, head by head of
// the group, in order (no atomics: the sum's order is fixed).
template <typename T, typename Z>
__device__ __forceinline__ void dkv_cores(const CausalParams& p, float* sm, int k0, int hkv, int b) {
  constexpr int TM = Z::TM, TN = Z::TN, DM = Z::DM;
  constexpr bool kAhead = Z::kAhead;
  __shared__ RowStat st_all[Z::G][TN];
  const Place w = place<Z>();
  float* groups = sm + Z::bwd_all();
  float* k_s = sm;
  float* v_s = k_s + TM * Z::RS;
  float* q_s = groups + w.g * Z::bwd_group();
  float* g_s = q_s + TN * Z::RS;
  float* p_s = g_s + TN * Z::RS;
  float* x_s = p_s + TM * Z::PS;
  RowStat* st_s = st_all[w.g];
  load_tile<T, TM, DM, Z::NT>(k_s, p.k, b * p.k_sb + hkv * p.k_sh, p.k_sn, k0, p.N, p.Dk, threadIdx.x, p.vec4);
  load_tile<T, TM, DM, Z::NT>(v_s, p.v, b * p.v_sb + hkv * p.v_sh, p.v_sn, k0, p.N, p.Dv, threadIdx.x, p.vec4);
  float4 dk[Z::R][Z::C], dv[Z::R][Z::C];
#pragma unroll
  for (int i = 0; i < Z::R; ++i)
#pragma unroll
    for (int j = 0; j < Z::C; ++j) dk[i][j] = dv[i][j] = make_float4(0.f, 0.f, 0.f, 0.f);
  // tile i: queries k0 + i % steps TN of head i / steps
  const int end = query_end(p, b, min(k0 + TM, p.N) - 1);
  const int steps = max(0, (end - k0 + TN - 1) / TN), tiles = steps * p.E;
  float4 qr[kAhead ? Z::kFetch / 4 : 1], gr[kAhead ? Z::kFetch / 4 : 1];
  const int64_t qb = b * p.q_sb, gb = (int64_t)b * p.N * p.Hq * p.Dv, gn = (int64_t)p.Hq * p.Dv;
  auto fetch = [&](int i) {
    const int hq = hkv * p.E + i / steps, q0 = k0 + i % steps * TN;
    fetch_tile<T, Z>(qr, p.q, qb + hq * p.q_sh, p.q_sn, q0, p.N, p.Dk, w.t, p.vec4);
    fetch_tile<T, Z>(gr, p.dout, gb + hq * p.Dv, gn, q0, p.N, p.Dv, w.t, p.vec4);
  };
  if (kAhead && w.g < tiles) fetch(w.g);
  __syncthreads();
  for (int i0 = w.g; i0 < tiles; i0 += Z::G) {
    const int hq = hkv * p.E + i0 / steps, q0 = k0 + i0 % steps * TN;
    group_sync<Z>(w.g);
    if constexpr (kAhead) {
      put_tile<Z>(q_s, qr, w.t);
      put_tile<Z>(g_s, gr, w.t);
    } else {
      load_tile<T, TN, DM, Z::GT>(q_s, p.q, qb + hq * p.q_sh, p.q_sn, q0, p.N, p.Dk, w.t, p.vec4);
      load_tile<T, TN, DM, Z::GT>(g_s, p.dout, gb + hq * p.Dv, gn, q0, p.N, p.Dv, w.t, p.vec4);
    }
    if (w.t < TN) st_s[w.t] = row_stat(p, b, hq, q0 + w.t);
    group_sync<Z>(w.g);
    if (kAhead && i0 + Z::G < tiles) fetch(i0 + Z::G);
    float s[Z::R][Z::S], d[Z::R][Z::S];
    dot_tile<Z>(k_s, q_s, p.Dk, w, s);
    dot_tile<Z>(v_s, g_s, p.Dv, w, d);
#pragma unroll
    for (int i = 0; i < Z::R; ++i)
#pragma unroll
      for (int j = 0; j < Z::S; ++j) {
        float pr, dx;
        grad_of(p, st_s[w.tx + 16 * j], k0 + w.ty + Z::RW * i, s[i][j], d[i][j], &pr, &dx);
        p_s[(w.ty + Z::RW * i) * Z::PS + w.tx + 16 * j] = pr;
        x_s[(w.ty + Z::RW * i) * Z::PS + w.tx + 16 * j] = dx;
      }
    group_sync<Z>(w.g);
    mul_tile<Z>(p_s, g_s, w, dv);
    mul_tile<Z>(x_s, q_s, w, dk);
  }
  group_sync<Z>(w.g);
  constexpr int kAt = Z::R * Z::C * 4;
  const bool first = join_sums<Z, 0>(groups, Z::bwd_group(), w, dk, 0);
  if (!join_sums<Z, 1>(groups, Z::bwd_group(), w, dv, kAt) || !first) return;
  store_rows<T, Z>(static_cast<T*>(p.dk) + ((int64_t)b * p.N * p.Hkv + hkv) * p.Dk, (int64_t)p.Hkv * p.Dk, k0, p.N, p.Dk,
                   p.scale, w, dk);
  store_rows<T, Z>(static_cast<T*>(p.dv) + ((int64_t)b * p.N * p.Hkv + hkv) * p.Dv, (int64_t)p.Hkv * p.Dv, k0, p.N, p.Dv,
                   1.f, w, dv);
}

// Both passes in one launch, the dK/dV blocks first (they do four products a tile
// to the other's three), each from its longest: a small problem's blocks of both
// share the SMs.
template <typename T, typename Z>
__global__ void __launch_bounds__(Z::NT) bwd_cores(const __grid_constant__ CausalParams p) {
  extern __shared__ __align__(16) float sm[];
  const int tiles = (p.N + Z::TM - 1) / Z::TM, x = blockIdx.x, b = blockIdx.y;
  if (x < tiles * p.Hkv) {
    dkv_cores<T, Z>(p, sm, x / p.Hkv * Z::TM, x % p.Hkv, b);
  } else {
    const int y = x - tiles * p.Hkv;
    dq_cores<T, Z>(p, sm, (tiles - 1 - y / p.Hq) * Z::TM, y % p.Hq, b);
  }
}

template <typename K>
int launch_cores(K kernel, dim3 grid, int threads, size_t smem, const CausalParams& p, cudaStream_t st) {
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    return TC_ERR_CUDA;
  kernel<<<grid, threads, smem, st>>>(p);
  return launch_status();
}

template <typename T, typename Z>
int fwd_cores_launch(const CausalParams& p, cudaStream_t st) {
  constexpr size_t smem = sizeof(float) * (Z::fwd_all() + Z::G * Z::fwd_group());
  static_assert(smem <= 227 * 1024, "forward shared memory exceeds the per-CTA limit");
  return launch_cores(fwd_cores<T, Z>, dim3((p.N + Z::TM - 1) / Z::TM, p.Hq, p.B), Z::NT, smem, p, st);
}
template <typename T, typename Z>
int bwd_cores_launch(const CausalParams& p, cudaStream_t st) {
  constexpr size_t smem = sizeof(float) * (Z::bwd_all() + Z::G * Z::bwd_group());
  static_assert(smem + Z::G * Z::TN * sizeof(RowStat) <= 227 * 1024, "backward shared memory exceeds the per-CTA limit");
  const int64_t blocks = (int64_t)((p.N + Z::TM - 1) / Z::TM) * (p.Hq + p.Hkv);
  if (blocks > INT32_MAX) return TC_ERR_UNSUPPORTED;
  return launch_cores(bwd_cores<T, Z>, dim3((unsigned)blocks, p.B), Z::NT, smem, p, st);
}

// Blocks of 32 rows whose four groups of 128 threads share the tiles (two groups in
// the backward of D > 64, whose operands are wider; one of 256 threads above 128).
// Against blocks of 64 rows with one group of 256, fp32: 4 heads of 64 and 1024
// tokens 54 and 94 us forward and backward against 107 and 193, 4 key heads of 128
// there 85 and 198 against 169 and 312 us; 32 heads of 4096 tokens the same forward
// (2605 / 2580 us at 64, 4460 / 4516 at 128) and 8.5 against 9.1 ms backward at 64.
// Only the backward of D > 64 is faster in blocks of 64 once they give every SM two:
// 15.0 against 19.3 ms (its two groups are one block's threads on half the rows).
template <typename T>
int fwd_cores_any(const CausalParams& p, cudaStream_t st) {
  const int D = imax(p.Dk, p.Dv);
  if (D <= 64) return fwd_cores_launch<T, Tile<32, 64, 64, 128, 4>>(p, st);
  if (D <= 128) return fwd_cores_launch<T, Tile<32, 64, 128, 128, 4>>(p, st);
  return fwd_cores_launch<T, Tile<32, 32, 256, 256, 1>>(p, st);
}
template <typename T>
int bwd_cores_any(const CausalParams& p, cudaStream_t st) {
  const int D = imax(p.Dk, p.Dv);
  if (D <= 64) return bwd_cores_launch<T, Tile<32, 64, 64, 128, 4>>(p, st);
  if (D > 128) return bwd_cores_launch<T, Tile<32, 32, 256, 256, 1>>(p, st);
  const bool wide = (int64_t)((p.N + 63) / 64) * p.Hkv * p.B >= 2 * 148;
  return wide ? bwd_cores_launch<T, Tile<64, 64, 128, 256, 1>>(p, st) : bwd_cores_launch<T, Tile<32, 64, 128, 128, 2>>(p, st);
}

int make_params(const tc_causal_args* a, CausalParams* p) {
  if (!a || a->B < 0 || a->N < 0 || a->Hq <= 0 || a->Hkv <= 0 || a->Hq % a->Hkv || a->Dk <= 0 || a->Dv <= 0)
    return TC_ERR_ARG;
  if ((a->starts == nullptr) != (a->ends == nullptr)) return TC_ERR_ARG;
  if (a->dtype != TC_F32 && a->dtype != TC_BF16 && a->dtype != TC_F16) return TC_ERR_ARG;
  if (a->impl < 0 || a->impl > 2 || !std::isfinite(a->scale)) return TC_ERR_ARG;
  if (a->has_softcap && !(a->softcap > 0.f && std::isfinite(a->softcap))) return TC_ERR_ARG;
  if (a->B > 65535 || a->Hq > 65535) return TC_ERR_UNSUPPORTED;
  p->B = a->B, p->N = a->N, p->Hq = a->Hq, p->Hkv = a->Hkv, p->E = a->Hq / a->Hkv, p->Dk = a->Dk, p->Dv = a->Dv;
  p->scale = a->scale, p->cap = a->has_softcap ? a->softcap : 1.f, p->has_cap = a->has_softcap != 0;
  p->q = a->q, p->k = a->k, p->v = a->v;
  p->q_sb = a->q_stride_b, p->q_sn = a->q_stride_n, p->q_sh = a->q_stride_h;
  p->k_sb = a->k_stride_b, p->k_sn = a->k_stride_n, p->k_sh = a->k_stride_h;
  p->v_sb = a->v_stride_b, p->v_sn = a->v_stride_n, p->v_sh = a->v_stride_h;
  p->starts = a->starts, p->ends = a->ends;
  p->out = a->out, p->lse = a->lse, p->out_low = a->out_low;
  p->o = a->o, p->o_low = a->o_low, p->dout = a->dout, p->dlse = a->dlse, p->delta = a->delta;
  p->dq = a->dq, p->dk = a->dk, p->dv = a->dv;
  p->status = a->dev_status;
  const int unit = a->dtype == TC_F32 ? 16 : 8;
  const int64_t strides = a->q_stride_b | a->q_stride_n | a->q_stride_h | a->k_stride_b | a->k_stride_n | a->k_stride_h |
                          a->v_stride_b | a->v_stride_n | a->v_stride_h | a->Dk | a->Dv;
  const uintptr_t starts = (uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->dout;
  p->vec4 = strides % 4 == 0 && starts % unit == 0;
  return TC_OK;
}

}  // namespace

namespace tc {
int causal_delta(const CausalParams& p, int dtype, cudaStream_t st) {
  TC_DISPATCH(dtype, T, return launch_delta<T>(p, st));
}
}  // namespace tc

extern "C" int tc_segment_bounds(int32_t B, int32_t N, const int32_t* seq_idx, int32_t* starts, int32_t* ends,
                                 void* stream) {
  return launch_bounds(B, N, seq_idx, starts, ends, (cudaStream_t)stream);
}

extern "C" int tc_segment_bounds_i64(int32_t B, int32_t N, const int64_t* seq_idx, int32_t* starts, int32_t* ends,
                                     void* stream) {
  return launch_bounds(B, N, seq_idx, starts, ends, (cudaStream_t)stream);
}

extern "C" int tc_causal_fwd(const tc_causal_args* a, void* stream) {
  CausalParams p;
  if (int rc = make_params(a, &p)) return rc;
  if ((int64_t)a->B * a->N == 0) return TC_OK;
  if (!a->q || !a->k || !a->v || !a->out || !a->lse) return TC_ERR_ARG;
  cudaStream_t st = (cudaStream_t)stream;
  const bool tensor = a->impl != 1 && causal_tc_supported(p, a->dtype);
  if (tensor) return causal_fwd_tc(p, a->dtype, st);
  if (a->impl == 2 || p.Dk > 256 || p.Dv > 256) return TC_ERR_UNSUPPORTED;
  TC_DISPATCH(a->dtype, T, return fwd_cores_any<T>(p, st));
}

extern "C" int tc_causal_bwd(const tc_causal_args* a, void* stream) {
  CausalParams p;
  if (int rc = make_params(a, &p)) return rc;
  if ((int64_t)a->B * a->N == 0) return TC_OK;
  if (!a->q || !a->k || !a->v || !a->o || !a->dout || !a->lse || !a->delta || !a->dq || !a->dk || !a->dv)
    return TC_ERR_ARG;
  cudaStream_t st = (cudaStream_t)stream;
  const bool tensor = a->impl != 1 && causal_bwd_tc_supported(p, a->dtype);
  if (!tensor && (a->impl == 2 || p.Dk > 256 || p.Dv > 256)) return TC_ERR_UNSUPPORTED;
  if (int rc = causal_delta(p, a->dtype, st)) return rc;
  if (tensor) return causal_bwd_tc(p, a->dtype, st);
  TC_DISPATCH(a->dtype, T, return bwd_cores_any<T>(p, st));
}

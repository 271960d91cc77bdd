// 8-bit key / value cache: quantising rows as they are written, reading them
// back, and single-token attention over the codes (sm_100a).
//
// A row (one token's key or value of one head) is kept as D codes and one fp32
// scale:  scale = amax / top,  code = round(x (top / amax)),  with top 127 and
// the code + 128 in a byte (TC_KV_INT8), or top 448 and an e4m3 float
// (TC_KV_FP8).  Quotients and products are the rounded IEEE ones, so the codes
// of a value do not depend on which kernel wrote it.  Rows with amax < 1e-30
// are zeros; a row with a NaN or an infinity reads back as NaN.
//
// Layout [rows, Hkv, capacity, D]: a head's tokens are consecutive, so a split
// of a sequence streams one contiguous range of codes.
#include <cuda_fp8.h>
#include <float.h>

#include <cmath>
#include <type_traits>

#include "rotary.cuh"
#include "tc_common.cuh"

using namespace tc;
using namespace tc::ptx;
using tc::tcx::kLn2;
using tc::tcx::kLog2e;

namespace {

constexpr float kTiny = 1e-30f;

template <int STORE> struct Codec;
template <> struct Codec<TC_KV_INT8> {
  static constexpr float kTop = 127.f;
  // y + 1.5 2^23 rounds y to an integer (nearest even) into the low mantissa bits:
  // an add where the float-to-int conversion runs at a quarter of its rate
  static __device__ __forceinline__ uint32_t code(float y) { return __float_as_uint(y + (12582912.f + 128.f)) & 255u; }
  static __device__ __forceinline__ uint32_t code4(const float* y) {
    uint32_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = __float_as_uint(y[i] + (12582912.f + 128.f));
    return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
  }
  // byte i of w: 2^23 + u exactly, then u - 128
  static __device__ __forceinline__ float value(uint32_t c) { return __uint_as_float(0x4B000000u | c) - (8388608.f + 128.f); }
  static __device__ __forceinline__ void value4(uint32_t w, float* v) {
    v[0] = __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7440)) - (8388608.f + 128.f);
    v[1] = __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7441)) - (8388608.f + 128.f);
    v[2] = __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7442)) - (8388608.f + 128.f);
    v[3] = __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7443)) - (8388608.f + 128.f);
  }
  // The same two bytes as f16 subnormals u 2^-24, u = code + 128: a sum of their
  // products is (sum code q + 128 sum q) 2^-24.  One instruction where pair takes
  // two; for the keys, where the second sum is of the first one's size.  (For the
  // values it would be: 128 sum p against a sum of p v that averages out.)
  static constexpr float kMul = 16777216.f, kOff = 128.f;
  template <bool HI> static __device__ __forceinline__ uint32_t raw_pair(uint32_t x) {
    return __byte_perm(x, 0u, HI ? 0x4342 : 0x4140);
  }
  // bytes 0, 1 (hi: 2, 3) of x as two f16 values: 0x6400 | u is 1024 + u exactly
  template <bool HI> static __device__ __forceinline__ uint32_t pair(uint32_t x) {
    const uint32_t r = __byte_perm(x, 0x64646464u, HI ? 0x4342 : 0x4140);
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&r), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};
template <> struct Codec<TC_KV_FP8> {
  static constexpr float kTop = 448.f;
  static constexpr float kMul = 1.f, kOff = 0.f;
  template <bool HI> static __device__ __forceinline__ uint32_t raw_pair(uint32_t x) { return pair<HI>(x); }
  static __device__ __forceinline__ uint32_t code(float y) {
    return __nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
  }
  static __device__ __forceinline__ uint32_t code4(const float* y) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[0], y[1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[2], y[3]), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
  }
  static __device__ __forceinline__ float value(uint32_t c) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E4M3)));
  }
  static __device__ __forceinline__ void value4(uint32_t w, float* v) {
    const uint32_t lo = pair<false>(w), hi = pair<true>(w);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
  }
  template <bool HI> static __device__ __forceinline__ uint32_t pair(uint32_t x) {
    const __half2_raw v = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(HI ? x >> 16 : x & 0xffffu), __NV_E4M3);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};

// scale and top / amax of a row from its amax; the scale of a row with an infinity
// is NaN as that of one with a NaN is, so that all of it reads back as NaN.
template <int STORE>
__device__ __forceinline__ void row_scale(float amax, float* scale, float* inv) {
  const bool tiny = amax < kTiny;
  *scale = tiny ? 0.f : amax <= FLT_MAX ? __fdiv_rn(amax, Codec<STORE>::kTop) : NAN;
  *inv = tiny ? 0.f : __fdiv_rn(Codec<STORE>::kTop, amax);
}

// The 16 bytes of w as floats, and floats as 16 bytes.
template <typename T>
__device__ __forceinline__ void unpack16(const uint4& w, float* x) {
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, float>::value) {
      x[i] = __uint_as_float(v[i]);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      x[2 * i] = __uint_as_float(v[i] << 16);
      x[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack16(const float* x) {
  if constexpr (std::is_same<T, float>::value)
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  else
    return tcx::pack8<T>(x, 1.f);
}

// Largest |x| of the 16 bytes of w, as the bits of its type (16-bit types: two to
// a register, joined at the end), and as float bits.
template <typename T>
__device__ __forceinline__ uint32_t amax16(const uint4& w) {
  if constexpr (std::is_same<T, float>::value) {
    const uint32_t m = 0x7fffffffu;
    return max(max(w.x & m, w.y & m), max(w.z & m, w.w & m));
  } else {
    const uint32_t m = 0x7fff7fffu;
    return __vmaxu2(__vmaxu2(w.x & m, w.y & m), __vmaxu2(w.z & m, w.w & m));
  }
}
template <typename T>
__device__ __forceinline__ uint32_t amax_join(uint32_t a, uint32_t b) {
  return std::is_same<T, float>::value ? max(a, b) : __vmaxu2(a, b);
}
template <typename T>
__device__ __forceinline__ float amax_float(uint32_t a) {
  if constexpr (std::is_same<T, float>::value) return __uint_as_float(a);
  const uint32_t h = max(a & 0xffffu, a >> 16);
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return __uint_as_float(h << 16);
  return __half2float(__ushort_as_half((unsigned short)h));
}

// |x| as bits: ordered as the floats are, with every NaN above infinity.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The value of a code: NaN only where the scale is, never infinite (127 times a
// scale that was rounded up may pass the largest float).
__device__ __forceinline__ float held(float v, float scale) {
  v *= scale;
  return scale <= FLT_MAX ? fminf(fmaxf(v, -FLT_MAX), FLT_MAX) : v;
}
template <int STORE>
__device__ __forceinline__ float dequant(uint32_t c, float scale) {
  return held(Codec<STORE>::value(c), scale);
}

// ---------------------------------------------------------------------------
// write
// ---------------------------------------------------------------------------
struct WriteSide {  // keys or values
  const void* src;
  int64_t sb, sn, sh;
  uint8_t* codes;
  float* scales;
  int dim;
};
struct WriteParams {
  int B, N, H, rows, fresh;
  int64_t cap;
  WriteSide k, v;
  int32_t* lengths;
  const int32_t* seq;     // [B, N] or null: token (b, n) belongs to cache row b
  const int32_t* starts;  // [B, N] first token of each run of equal ids (with seq)
  int32_t* status;
};

// Cache row and slot of token (b, n); row -1 where it is not written.
__device__ __forceinline__ void place(const WriteParams& p, int b, int n, int* row, int64_t* slot) {
  int r = b, first = 0;
  if (p.seq) {
    r = p.seq[(int64_t)b * p.N + n];
    first = p.starts[(int64_t)b * p.N + n];
  }
  *row = -1;
  if (r < 0) return;
  if (r >= p.rows) {
    if (p.status) atomicOr(p.status, TC_DEV_BAD_INDEX);
    return;
  }
  const int64_t s = (int64_t)(p.fresh ? 0 : p.lengths[r]) + (n - first);
  if (s < 0 || s >= p.cap) {
    if (p.status) atomicOr(p.status, TC_DEV_BAD_INDEX);
    return;
  }
  *row = r;
  *slot = s;
}

// A row's new length is set where its run ends; with fresh nothing else reads
// the lengths, so the write kernel does it, otherwise a kernel behind it.
__device__ __forceinline__ void advance_row(const WriteParams& p, int b, int n) {
  int r = b, first = 0;
  if (p.seq) {
    const int64_t i = (int64_t)b * p.N + n;
    r = p.seq[i];
    if (r < 0 || r >= p.rows || (n + 1 < p.N && p.seq[i + 1] == r)) return;
    first = p.starts[i];
  } else if (n + 1 < p.N) {
    return;
  }
  const int64_t len = (int64_t)(p.fresh ? 0 : p.lengths[r]) + (n + 1 - first);
  p.lengths[r] = (int32_t)(len < p.cap ? len : p.cap);
}

__global__ void __launch_bounds__(256) advance_kernel(WriteParams p) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i < (int64_t)p.B * p.N) advance_row(p, (int)(i / p.N), (int)(i % p.N));
}

// LANES lanes per row, 16 bytes each; blockIdx.y: 0 keys, 1 values.  The row is read
// once and the codes leave as 8-byte (fp32: 4-byte) pieces of whole 32-byte sectors.
// A lane group takes kTok consecutive tokens of one head.  Their loads go out before
// the places are known (a dependent read away), so tokens that go nowhere are read
// too: 144 us for 161 without padding, 120 for 118 with one half padding.  The kTok
// maxima are found together, half of the lanes going on with half of the tokens, and
// each is divided by once.
// Bound by HBM and issue alike: 4 x 16384 tokens of 16 heads of 128, bf16 to int8, 0.8
// GB of values and codes in 144 us, 5.6 TB/s; one eighth of them padding: 138 us (maxima
// one by one and a division a lane 171, the conversion instruction in place of the add
// in code() and two tokens a group 254; eight tokens a group as four).
constexpr int kTok = 4;
template <typename T, int STORE, int LANES>
__global__ void __launch_bounds__(256) write_vec(const __grid_constant__ WriteParams p) {
  constexpr int VE = 16 / sizeof(T);
  const bool keys = blockIdx.y == 0;
  const WriteSide& w = keys ? p.k : p.v;
  const int b = blockIdx.z, lane = threadIdx.x % LANES;
  const int group = blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  const int tile = group / p.H, h = group - tile * p.H, n0 = tile * kTok;
  if (n0 >= p.N) return;  // whole lane groups leave; the shuffles below name their own lanes
  const uint32_t mask = LANES == 32 ? 0xffffffffu : ((1u << LANES) - 1u) << ((threadIdx.x & 31) / LANES * LANES);
  // lane j: row of codes of token n0 + j (rows of 64 or more bytes: 32 bits count
  // more of them than the memory holds)
  const T* src = static_cast<const T*>(w.src) + b * w.sb + h * w.sh + lane * VE;
  uint4 raw[kTok];
#pragma unroll
  for (int j = 0; j < kTok; ++j) {
    raw[j] = make_uint4(0u, 0u, 0u, 0u);
    if (n0 + j < p.N) raw[j] = *reinterpret_cast<const uint4*>(src + (int64_t)(n0 + j) * w.sn);
  }
  uint32_t at = 0xffffffffu;
  if (lane < kTok && n0 + lane < p.N) {
    int row;
    int64_t slot = 0;
    place(p, b, n0 + lane, &row, &slot);
    if (row >= 0) at = (uint32_t)(((int64_t)row * p.H + h) * p.cap + slot);
    if (p.fresh && keys && h == 0) advance_row(p, b, n0 + lane);
  }
  uint32_t to[kTok], m[kTok];
#pragma unroll
  for (int j = 0; j < kTok; ++j) {
    to[j] = __shfl_sync(mask, at, j, LANES);
  }
#pragma unroll
  for (int j = 0; j < kTok; ++j) m[j] = amax16<T>(raw[j]);
  int o = LANES / 2;
#pragma unroll
  for (int n = kTok / 2; n; n /= 2, o /= 2) {
    const bool up = lane & o;
#pragma unroll
    for (int j = 0; j < n; ++j)
      m[j] = amax_join<T>(up ? m[j + n] : m[j], __shfl_xor_sync(mask, up ? m[j] : m[j + n], o));
  }
#pragma unroll
  for (; o; o /= 2) m[0] = amax_join<T>(m[0], __shfl_xor_sync(mask, m[0], o));
  constexpr int kShare = LANES / kTok;  // lanes that hold one token's maximum
  float scale, inv;
  row_scale<STORE>(amax_float<T>(m[0]), &scale, &inv);
#pragma unroll
  for (int j = 0; j < kTok; ++j) {
    const float by = __shfl_sync(mask, inv, j * kShare, LANES);
    if (to[j] == 0xffffffffu) continue;
    float x[VE];
    unpack16<T>(raw[j], x);
#pragma unroll
    for (int i = 0; i < VE; ++i) x[i] = __fmul_rn(x[i], by);
    uint8_t* dst = w.codes + (int64_t)to[j] * (LANES * VE) + lane * VE;
    if constexpr (VE == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(Codec<STORE>::code4(x), Codec<STORE>::code4(x + 4));
    else *reinterpret_cast<uint32_t*>(dst) = Codec<STORE>::code4(x);
    if (lane == j * kShare) w.scales[to[j]] = scale;
  }
}

// Any head dim and strides: a warp per row, two passes over it.
template <typename T, int STORE>
__global__ void __launch_bounds__(256) write_any(const __grid_constant__ WriteParams p) {
  const bool keys = blockIdx.y == 0;
  const WriteSide& w = keys ? p.k : p.v;
  const int lane = threadIdx.x & 31;
  const int64_t i = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int h = (int)(i % p.H);
  const int64_t tok = i / p.H;
  if (tok >= (int64_t)p.B * p.N) return;
  const int b = (int)(tok / p.N), n = (int)(tok % p.N);
  int row;
  int64_t slot = 0;
  place(p, b, n, &row, &slot);
  if (p.fresh && keys && h == 0 && lane == 0) advance_row(p, b, n);
  if (row < 0) return;
  const T* src = static_cast<const T*>(w.src) + b * w.sb + (int64_t)n * w.sn + h * w.sh;
  const int D = w.dim;
  uint32_t m = 0;
  for (int d = lane; d < D; d += 32) m = max(m, abs_bits(to_f(src[d])));
#pragma unroll
  for (int o = 16; o; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  float scale, inv;
  row_scale<STORE>(__uint_as_float(m), &scale, &inv);
  const int64_t at = ((int64_t)row * p.H + h) * p.cap + slot;
  for (int d = lane; d < D; d += 32) w.codes[at * D + d] = (uint8_t)Codec<STORE>::code(__fmul_rn(to_f(src[d]), inv));
  if (lane == 0) w.scales[at] = scale;
}

template <typename T, int STORE>
int launch_write(const WriteParams& p, cudaStream_t st) {
  constexpr int VE = 16 / sizeof(T);
  bool vec = p.k.dim == p.v.dim;
  for (const WriteSide* w : {&p.k, &p.v})
    vec = vec && (uintptr_t)w->src % 16 == 0 && w->sb % VE == 0 && w->sn % VE == 0 && w->sh % VE == 0 &&
          (uintptr_t)w->codes % 8 == 0;
  const int lanes = p.k.dim / VE;
  vec = vec && p.k.dim % VE == 0 && (lanes == 8 || lanes == 16 || lanes == 32);
  vec = vec && p.B <= 65535;
  const int64_t units = vec ? (int64_t)((p.N + kTok - 1) / kTok) * p.H * lanes : (int64_t)p.B * p.N * p.H * 32;
  const int64_t grid = (units + 255) / 256;
  if (grid > INT32_MAX) return TC_ERR_UNSUPPORTED;
  const dim3 g((unsigned)grid, 2, vec ? p.B : 1);
  if (!vec) write_any<T, STORE><<<g, 256, 0, st>>>(p);
  else if (lanes == 8) write_vec<T, STORE, 8><<<g, 256, 0, st>>>(p);
  else if (lanes == 16) write_vec<T, STORE, 16><<<g, 256, 0, st>>>(p);
  else write_vec<T, STORE, 32><<<g, 256, 0, st>>>(p);
  if (int rc = launch_status()) return rc;
  if (!p.fresh) {
    advance_kernel<<<(unsigned)(((int64_t)p.B * p.N + 255) / 256), 256, 0, st>>>(p);
    return launch_status();
  }
  return TC_OK;
}

// ---------------------------------------------------------------------------
// read back
// ---------------------------------------------------------------------------
struct ReadSide {
  const uint8_t* codes;
  const float* scales;
  int dim;
  void* out;  // [rows, L, H, D]
};
struct ReadParams {
  int rows, H, L;
  int64_t cap;
  ReadSide k, v;
  const int32_t* lengths;
};

// A thread per V codes of one row (V = 16 / element size, or 1) and kReadTok
// tokens; a CTA's threads run over the heads and dims of a token, so the output
// is written in order.  Slots past a row's length are zeros and read nothing.  Bound
// by HBM: the cache of the write's case (0.77 GB of codes and values) in 128 us, 6.0
// TB/s (one token a thread: 190).
constexpr int kReadTok = 8;
template <typename T, int STORE, int V>
__global__ void __launch_bounds__(256) read_kernel(const __grid_constant__ ReadParams p) {
  const ReadSide& w = blockIdx.y == 0 ? p.k : p.v;
  const int D = w.dim, per = p.H * (D / V);  // threads per token
  const int b = blockIdx.z, len = (int)min((int64_t)p.lengths[b], p.cap);
  const int64_t first = (int64_t)blockIdx.x * blockDim.x;
  const int t0 = (int)(first / per), off = (int)(first - (int64_t)t0 * per) + threadIdx.x;  // one wide division a CTA
  const int tile = t0 + off / per, rest = off % per;
  const int h = rest / (D / V), d = (rest - h * (D / V)) * V;
  const int n0 = tile * kReadTok;
  using Raw = typename std::conditional<V == 8, uint2, typename std::conditional<V == 4, uint32_t, uint8_t>::type>::type;
  Raw raw[kReadTok];
  float sc[kReadTok];
  const int64_t at0 = ((int64_t)b * p.H + h) * p.cap;
#pragma unroll
  for (int j = 0; j < kReadTok; ++j) {
    const int n = n0 + j;
    sc[j] = 0.f;
    if (n < len && n < p.L) {
      raw[j] = *reinterpret_cast<const Raw*>(w.codes + (at0 + n) * D + d);
      sc[j] = w.scales[at0 + n];
    }
  }
#pragma unroll
  for (int j = 0; j < kReadTok; ++j) {
    const int n = n0 + j;
    if (n >= p.L) return;
    T* out = static_cast<T*>(w.out) + (((int64_t)b * p.L + n) * p.H + h) * D + d;
    float v[V];
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = 0.f;
    if (n < len) {
      if constexpr (V == 8) {
        Codec<STORE>::value4(raw[j].x, v);
        Codec<STORE>::value4(raw[j].y, v + 4);
      } else if constexpr (V == 4) {
        Codec<STORE>::value4(raw[j], v);
      } else {
        v[0] = Codec<STORE>::value(raw[j]);
      }
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] = held(v[k], sc[j]);
    }
    if constexpr (V == 1) out[0] = from_f<T>(v[0]);
    else *reinterpret_cast<uint4*>(out) = pack16<T>(v);
  }
}

template <typename T, int STORE>
int launch_read(const ReadParams& p, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  bool vec = true;
  for (const ReadSide* w : {&p.k, &p.v})
    vec = vec && w->dim % V == 0 && (uintptr_t)w->codes % V == 0 && (uintptr_t)w->out % 16 == 0;
  const int D = p.k.dim > p.v.dim ? p.k.dim : p.v.dim;
  const int64_t units = (int64_t)((p.L + kReadTok - 1) / kReadTok) * p.H * (vec ? D / V : D);
  const int64_t grid = (units + 255) / 256;
  if (grid > INT32_MAX || p.rows > 65535) return TC_ERR_UNSUPPORTED;
  const dim3 g((unsigned)grid, 2, p.rows);
  if (vec) read_kernel<T, STORE, V><<<g, 256, 0, st>>>(p);
  else read_kernel<T, STORE, 1><<<g, 256, 0, st>>>(p);
  return launch_status();
}

// ---------------------------------------------------------------------------
// single-token attention over the codes
// ---------------------------------------------------------------------------
struct AttendParams {
  int B, Hq, Hkv, E, groups;   // groups: eights of query heads per key head
  int Dk, Dv;
  int64_t cap;
  uint8_t* k;
  uint8_t* v;
  float* ks;
  float* vs;
  int32_t* lengths;
  const void* q;
  int64_t q_sb, q_sh;
  const void* k_t;             // step: the new token's key and value
  const void* v_t;
  int64_t k_sb, k_sh, v_sb, v_sh;
  const float* cos_t;          // step: [n_pos, R / 2] or null
  const float* sin_t;
  int R, interleaved, n_pos;
  float qscale, softcap;       // logit = qscale q.k (1 / sqrt(Dk) unless given)
  int has_cap, advance;
  void* out;                   // [B, Hq, Dv]
  float* lse;                  // [B, Hq]
  void* k_new;                 // step: the values as stored, [B, Hkv, D], or null
  void* v_new;
  int new_dtype;
  int chunk, splits;           // tokens per CTA, CTAs per (sequence, head group)
  float* part;                 // [B * Hkv * groups * splits][8][Dv] unnormalised O
  float2* ml;                  // [B * Hkv * groups * splits][8] their maximum (log2 units) and sum
  int32_t* done;               // [B * Hkv * groups + B] arrival counts, zero between calls
  int32_t* status;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float2 unpack_h2(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
  for (int o = 16; o; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}
__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// Dims of pair u of a D-dim head whose first R dims rotate: the rotary pair for
// u < R / 2, else two neighbours behind them (an odd last dim pairs with itself).
__device__ __forceinline__ void pair_dims(int u, int R, int interleaved, int D, int* i1, int* i2) {
  const int half = R / 2;
  if (u < half) {
    *i1 = interleaved ? 2 * u : u;
    *i2 = interleaved ? 2 * u + 1 : u + half;
  } else {
    *i1 = R + 2 * (u - half);
    *i2 = *i1 + 1 < D ? *i1 + 1 : *i1;
  }
}

// Pair u of a head's row x, rotated to position pos where the step has tables.
template <typename T>
__device__ __forceinline__ void load_pair(const AttendParams& p, const T* x, int u, int D, int R, int pos, int* i1,
                                          int* i2, float* y1, float* y2) {
  pair_dims(u, R, p.interleaved, D, i1, i2);
  const float x1 = to_f(x[*i1]), x2 = to_f(x[*i2]);
  *y1 = x1;
  *y2 = x2;
  if (u < R / 2) {
    float c = NAN, s = NAN;
    if (pos < p.n_pos) {
      c = p.cos_t[(int64_t)pos * (R / 2) + u];
      s = p.sin_t[(int64_t)pos * (R / 2) + u];
    }
    rotate_pair(x1, x2, c, s, y1, y2);
  }
}

// One warp quantises the new token's row into slot `pos` of its head, and into
// `copy` (byte place(d) for dim d) with its scale.
template <typename T, int STORE, typename F>
__device__ void write_token(const AttendParams& p, const T* x, int D, int R, int pos, int64_t head, uint8_t* codes,
                            float* scales, void* stored, uint8_t* copy, float* copy_scale, F place) {
  const int lane = threadIdx.x & 31, pairs = (D + 1) / 2;
  uint32_t m = 0;
  for (int u = lane; u < pairs; u += 32) {
    int i1, i2;
    float y1, y2;
    load_pair(p, x, u, D, R, pos, &i1, &i2, &y1, &y2);
    m = max(m, max(abs_bits(y1), abs_bits(y2)));
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  float scale, inv;
  row_scale<STORE>(__uint_as_float(m), &scale, &inv);
  const int64_t at = head * p.cap + pos;
  for (int u = lane; u < pairs; u += 32) {
    int i[2];
    float y[2];
    load_pair(p, x, u, D, R, pos, &i[0], &i[1], &y[0], &y[1]);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint32_t c = Codec<STORE>::code(__fmul_rn(y[k], inv));
      codes[at * D + i[k]] = (uint8_t)c;
      if (copy) copy[place(i[k])] = (uint8_t)c;
      if (stored) store_any(stored, head * D + i[k], p.new_dtype, dequant<STORE>(c, scale));
    }
  }
  if (lane == 0) {
    scales[at] = scale;
    if (copy) *copy_scale = scale;
  }
}

// Joins the partials of `active` splits of nE heads and writes out, lse.  A warp
// takes a head (with fewer than four heads, the warps of one share its splits): it
// finds the joint maximum and sum, then reads the splits' O, four consecutive dims
// a lane and sixteen splits in flight.  The last CTA runs this alone, so what
// counts is how few rounds of loads follow one another.
constexpr int kAtWarps = 4;
template <typename TQ>
__device__ void join_splits(const AttendParams& p, int b, int hkv, int e0, int nE, int64_t slot0, int active,
                            float* red /* [kAtWarps][Dv] */) {
  constexpr int kFly = 16;
  __shared__ float inv_s[kAtWarps];
  const int D = p.Dv, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int heads = nE >= 3 ? 4 : nE, shares = kAtWarps / heads, share = warp / heads;  // heads at a time
  const int64_t head0 = (int64_t)b * p.Hq + hkv * p.E + e0;
  const bool quad = D % 4 == 0;
  for (int e1 = 0; e1 < nE; e1 += heads) {
    const int e = e1 + warp % heads;
    if (e < nE) {
      const float2* ml = p.ml + slot0 * 8 + e;
      const float* part = p.part + (slot0 * 8 + e) * D;
      float m = -INFINITY, l = 0.f;  // over this lane's splits
      for (int s = lane; s < active; s += 32) {
        const float2 v = __ldcg(ml + (int64_t)s * 8);
        const float mn = fmaxf(m, v.x), ref = mn == -INFINITY ? 0.f : mn;
        l = l * ex2(m - ref) + v.y * ex2(v.x - ref);
        m = mn;
      }
      const float top = warp_max(m), M = top == -INFINITY ? 0.f : top;
      l = warp_sum(l * ex2(m - M));
      if (lane == 0 && share == 0) {
        inv_s[warp] = l != 0.f ? 1.f / l : 0.f;
        p.lse[head0 + e] = l != 0.f ? (top + log2f(l)) * kLn2 : -INFINITY;
      }
      for (int d0 = 0; d0 < D; d0 += 128) {
        const int d = quad ? d0 + 4 * lane : d0 + lane;
        float o[4] = {0.f, 0.f, 0.f, 0.f};
        for (int s0 = share; s0 < active; s0 += kFly * shares) {
          float4 v[kFly];
          float w[kFly];
#pragma unroll
          for (int j = 0; j < kFly; ++j) {
            const int s = s0 + j * shares;
            v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
            w[j] = -INFINITY;
            if (s < active) {
              w[j] = __ldcg(ml + (int64_t)s * 8).x;
              const float* q = part + (int64_t)s * 8 * D + d;
              if (quad) {
                if (d < D) v[j] = __ldcg(reinterpret_cast<const float4*>(q));
              } else {
                if (d < D) v[j].x = __ldcg(q);
                if (d + 32 < D) v[j].y = __ldcg(q + 32);
                if (d + 64 < D) v[j].z = __ldcg(q + 64);
                if (d + 96 < D) v[j].w = __ldcg(q + 96);
              }
            }
          }
#pragma unroll
          for (int j = 0; j < kFly; ++j) {
            const float c = ex2(w[j] - M);
            o[0] += c * v[j].x, o[1] += c * v[j].y, o[2] += c * v[j].z, o[3] += c * v[j].w;
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int di = quad ? d + i : d + 32 * i;
          if (di < D) red[warp * D + di] = o[i];
        }
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < heads * D; i += kAtWarps * 32) {
      const int h = i / D, d = i - h * D;
      if (e1 + h >= nE) break;
      float o = 0.f;
      for (int k = 0; k < shares; ++k) o += red[(h + k * heads) * D + d];
      static_cast<TQ*>(p.out)[(head0 + e1 + h) * D + d] = from_f<TQ>(inv_s[h] != 0.f ? o * inv_s[h] : 0.f);
    }
    __syncthreads();
  }
}

// Every CTA's last act, behind its global writes: the last split of a (sequence,
// head group) to arrive joins the partials, and the last head group of a
// sequence moves its length on.  With `advance` the splits without tokens of
// their own arrive too: each CTA must have read the old length before it moves.
// The counts return to zero.
template <typename TQ>
__device__ void close_split(const AttendParams& p, int b, int hg, int e0, int nE, int64_t slot0, int active, int pos,
                            int* flag, float* red) {
  const int total = p.advance ? p.splits : active, per = p.Hkv * p.groups;
  if (total > 1) {
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
      int32_t* d = p.done + (int64_t)b * per + hg;
      const bool last = atomicAdd(d, 1) == total - 1;
      if (last) *d = 0;
      *flag = last;
    }
    __syncthreads();
    if (!*flag) return;
    __threadfence();
    if (active > 1) join_splits<TQ>(p, b, hg / p.groups, e0, nE, slot0, active, red);
  }
  if (p.advance && threadIdx.x == 0) {
    int32_t* d = p.done + (int64_t)p.B * per + b;
    if (atomicAdd(d, 1) == per - 1) {
      *d = 0;
      p.lengths[b] = (int32_t)min((int64_t)pos + 1, p.cap);
    }
  }
}

// tanh to 1e-6 of its value: the Maclaurin series through y^13 up to 1/2 (next
// term 1e-7 of the sum), beyond it 1 - 2 / (e^2y + 1) (3e-7 of at least 0.46).
__device__ __forceinline__ float tanh_rel(float y) {
  const float w = y * y;
  float s = fmaf(w, 21844.f / 6081075.f, -1382.f / 155925.f);
  s = fmaf(w, s, 62.f / 2835.f);
  s = fmaf(w, s, -17.f / 315.f);
  s = fmaf(w, s, 2.f / 15.f);
  s = fmaf(w, s, -1.f / 3.f);
  s = fmaf(y * w, s, y);
  const float t = 1.f - __fdividef(2.f, ex2(fabsf(y) * (2.f * kLog2e)) + 1.f);
  return fabsf(y) <= 0.5f ? s : copysignf(t, y);
}

// Tensor-core path, Dk = Dv = D (64 or 128).  CTA = one chunk of one sequence
// and up to eight query heads of one key head; its four warps take the chunk's
// 32-token units in turn, each through a ring of its own that TMA fills (8 KB a
// unit at D = 128; two in flight or in use per warp, twelve warps per SM), so that
// no warp waits for another.  (Stages of 64 tokens shared by the four warps cost a
// quarter of the time in their hand-over, and 16 tokens a step left a warp 3200
// clocks of dependent instructions for them.)  Products are m16n8k16 f16 with fp32
// accumulators:
//   S[head, token] = q K^T:  A = q, rows 0-7 the f16 roundings of the heads'
//     q and rows 8-15 what the roundings left over, so S = row h + row h + 8
//     has q to 22 bits; B = codes, exact in f16.
//   O[head, dim] += P V:     A = P, split in two the same way, with the value
//     rows' scales folded into it, relative to the head's largest such product so
//     far, times 2^9 (2^6 of growth fit): the f16 leftovers of one that is 2^-k of
//     the largest keep 22 - max(0, k - 12) bits.
// A dot product does not care about the order of its terms, so a lane reads 16
// consecutive codes of a token and the A operand follows that order; likewise
// output dims follow the value reads.  P leaves S's accumulator layout as the A
// operand without a shuffle.  Column n of an eight of tokens is token n or, for
// odd n, (n - 1 ^ 4) + 1: with the 128-byte swizzle the eight lanes of a shared
// memory phase then meet eight different bank groups, for keys and for values.
//
// Bound by HBM where it is long: 2 (D + 4) bytes a token and key head.  64 sequences
// of up to 32768 tokens, 16 / 4 heads of 128, int8: 210 us, 5.4 TB/s; 131072 tokens
// of one sequence, 32 / 8 heads, e4m3, softcap: 59 us, of which 42 are its reads at a
// copy's rate and the rest the start and the join; 1024 tokens: 10 us, latency alone.
// (With the values' scales relative to the largest scale, and the maxima joined in
// every unit: 211 and 65 us, and a value row 2^24 of the others' cost them their bits.)
constexpr int kAtThreads = 32 * kAtWarps;
constexpr float kUp = 512.f, kLazy = 4.f, kGrow = 64.f;
constexpr int kUnit = 32;  // tokens per stage

template <int D> struct AtSmem {
  static constexpr int kTile = kUnit * D;  // codes of one stage, keys or values
  static constexpr int kNS = D == 128 ? 2 : 3;   // stages per warp
  static constexpr int QS = D + 8;             // q row stride (halves)
  static constexpr int OS = D + D / 32 * 4;    // O row stride (floats)
  static constexpr int kBytes = kAtWarps * 2 * kNS * kTile + 1024;
};

// Byte of 16-byte chunk `c` of row `r` in a stage (TMA swizzle of D-byte rows).
template <int D>
__device__ __forceinline__ int stage_at(int r, int c) {
  return r * D + ((D == 128 ? c ^ (r & 7) : c ^ ((r >> 1) & 3)) << 4);
}
// Token of column n (0..7) of an eight.
__device__ __forceinline__ int tok_of(int n) { return n & 1 ? ((n - 1) ^ 4) | 1 : n; }

template <typename TQ, int STORE, int D, bool CAP, bool STEP>
__global__ void __launch_bounds__(kAtThreads, 3)
    attend_mma(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv,
               const __grid_constant__ AttendParams p) {
  using Z = AtSmem<D>;
  constexpr int KS = D / 16;  // k steps of S
  constexpr int ND = D / 8;   // n tiles of O
  constexpr int VB = D / 8;   // value codes per lane and token
  constexpr int NS = Z::kNS, QS = Z::QS, OS = Z::OS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ __align__(16) __half q_s[16 * QS];
  float* o_s = reinterpret_cast<float*>(sm);  // the warps' O, once every unit has been read
  static_assert(kAtWarps * 8 * OS * 4 <= kAtWarps * 2 * NS * Z::kTile, "O does not fit the ring");
  __shared__ __align__(128) uint8_t new_s[2][128];  // the new token's codes, as a stage row of its slot holds them
  __shared__ float new_scale[2], qf_s[8], qs_s[8], m_s[kAtWarps][8], l_s[kAtWarps][8];
  __shared__ uint64_t full_s[kAtWarps][NS];
  __shared__ int flag, abort_s;

  const int split = blockIdx.x;
  const int hg = blockIdx.y, b = blockIdx.z;
  const int hkv = hg / p.groups, e0 = (hg - hkv * p.groups) * 8;
  const int nE = min(8, p.E - e0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int pos = max(p.lengths[b], 0);
  if (threadIdx.x == 0) {
    prefetch_tmap(&tmk);
    prefetch_tmap(&tmv);
  }
  // the warp's query heads warp and warp + 4, on their way before the length is known
  constexpr int NP = D / 64;  // pairs per lane
  const int R = STEP ? p.R : 0;
  TQ qx[2][NP][2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int e = warp + 4 * h;
    const TQ* x = static_cast<const TQ*>(p.q) + b * p.q_sb + (int64_t)(hkv * p.E + e0 + e) * p.q_sh;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      int i1, i2;
      pair_dims(lane + 32 * j, R, p.interleaved, D, &i1, &i2);
      qx[h][j][0] = e < nE ? x[i1] : from_f<TQ>(0.f);
      qx[h][j][1] = e < nE ? x[i2] : from_f<TQ>(0.f);
    }
  }
  const int ntok = (int)min((int64_t)(STEP ? pos + 1 : pos), p.cap);
  const int active = max(1, min(p.splits, (ntok + p.chunk - 1) / p.chunk));
  const int64_t slot0 = ((int64_t)b * p.Hkv * p.groups + hg) * p.splits;
  if (split >= active) {
    if (p.advance) close_split<TQ>(p, b, hg, e0, nE, slot0, active, pos, &flag, o_s);
    return;
  }
  const int c0 = split * p.chunk, c1 = split == active - 1 ? ntok : c0 + p.chunk;
  const int units = (c1 - c0 + kUnit - 1) / kUnit, mine = (units - warp + kAtWarps - 1) / kAtWarps;
  const int64_t head = (int64_t)b * p.Hkv + hkv;
  const bool owner = STEP && split == active - 1 && pos < p.cap;  // its chunk holds the new slot
  volatile int* abort_flag = &abort_s;
  uint8_t* ring = sm + warp * NS * 2 * Z::kTile;
  uint64_t* full = full_s[warp];

  auto fill = [&](int i) {  // one lane: the warp's i-th unit
    const int st = i % NS, at = c0 + (warp + i * kAtWarps) * kUnit;
    mbar_expect_tx(&full[st], 2 * Z::kTile);
    tma_load_3d(ring + 2 * st * Z::kTile, &tmk, 0, at, (int)head, &full[st]);
    tma_load_3d(ring + (2 * st + 1) * Z::kTile, &tmv, 0, at, (int)head, &full[st]);
  };
  if (lane == 0) {
    for (int i = 0; i < NS; ++i) mbar_init(&full[i], 1);
    if (warp == 0) abort_s = 0;
    mbar_fence_init();
    fence_async_smem();
    for (int i = 0; i < NS && i < mine; ++i) fill(i);
  }
  // q: rotate, bring each head's largest element to [2^13, 2^14), split in two
  float cs[NP], sn[NP];
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    const int v = lane + 32 * j;
    cs[j] = 1.f;
    sn[j] = 0.f;
    if (STEP && v < R / 2) {
      cs[j] = pos < p.n_pos ? p.cos_t[(int64_t)pos * (R / 2) + v] : NAN;
      sn[j] = pos < p.n_pos ? p.sin_t[(int64_t)pos * (R / 2) + v] : NAN;
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int e = warp + 4 * h;
    float y1[NP], y2[NP];
    uint32_t m = 0;
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      y1[j] = to_f(qx[h][j][0]);
      y2[j] = to_f(qx[h][j][1]);
      if (STEP && lane + 32 * j < R / 2) rotate_pair(y1[j], y2[j], cs[j], sn[j], &y1[j], &y2[j]);
      if (e >= nE) y1[j] = y2[j] = 0.f;
      m = max(m, max(abs_bits(y1[j]), abs_bits(y2[j])));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const int ex = min(max((int)(m >> 23) - 127, -100), 126);
    const float up = m ? __int_as_float((127 + 13 - ex) << 23) : 1.f;
    const float down = m ? __int_as_float((127 - 13 + ex) << 23) : 1.f;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      int i1, i2;
      pair_dims(lane + 32 * j, R, p.interleaved, D, &i1, &i2);
      const float a = y1[j] * up, c = y2[j] * up;
      sum += a + c;
      const __half ah = __float2half_rn(a), ch = __float2half_rn(c);
      q_s[e * QS + i1] = ah;
      q_s[e * QS + i2] = ch;
      q_s[(e + 8) * QS + i1] = __float2half_rn(a - __half2float(ah));
      q_s[(e + 8) * QS + i2] = __float2half_rn(c - __half2float(ch));
    }
    sum = warp_sum(sum);
    if (lane == 0) {
      const float f = down * p.qscale * (CAP ? 1.f / p.softcap : kLog2e);
      qf_s[e] = Codec<STORE>::kMul * f;
      qs_s[e] = -Codec<STORE>::kOff * sum * f;
    }
  }
  if constexpr (STEP) {
    // The new token's row goes to the cache and, for this chunk's attention, to
    // new_s: the stage may have been loaded before the row was written.  (Head
    // groups of one key head write the same bytes.)
    if (owner && warp >= 2) {
      const int which = warp - 2;
      const int r = (pos - c0) % kUnit;
      const TQ* x = which ? static_cast<const TQ*>(p.v_t) + b * p.v_sb + hkv * p.v_sh
                          : static_cast<const TQ*>(p.k_t) + b * p.k_sb + hkv * p.k_sh;
      write_token<TQ, STORE>(p, x, D, which ? 0 : p.R, pos, head, which ? p.v : p.k, which ? p.vs : p.ks,
                             which ? p.v_new : p.k_new, new_s[which], &new_scale[which],
                             [&](int d) { return stage_at<D>(r, d >> 4) - r * D + (d & 15); });
    }
    if (split == active - 1 && !owner && threadIdx.x == 0 && p.status) atomicOr(p.status, TC_DEV_BAD_INDEX);
  }
  __syncthreads();

  {
    // A operand of S: k step 4 c + w covers, for lane t, the codes of word w of
    // its 16-byte chunk 4 c + t, dims 64 c + 16 t + 4 w + {0, 1 | 2, 3}
    uint32_t qa[KS][4];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = 64 * (s / 4) + 16 * t + 4 * (s % 4);
      const uint2 hi = *reinterpret_cast<const uint2*>(q_s + g * QS + d);
      const uint2 lo = *reinterpret_cast<const uint2*>(q_s + (g + 8) * QS + d);
      qa[s][0] = hi.x, qa[s][1] = lo.x, qa[s][2] = hi.y, qa[s][3] = lo.y;
    }
    const float qf = qf_s[g], qoff = qs_s[g];
    const float kc = p.softcap * kLog2e;
    float o[ND][4];
#pragma unroll
    for (int i = 0; i < ND; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m = -INFINITY, ell = 0.f, winv = 0.f;  // winv: kUp / the reference of weight times scale
    // a lane holds the key and value scale of token `lane` of the warp's unit
    const float* ksb = p.ks + head * p.cap + c0 + warp * kUnit + lane;
    const float* vsb = p.vs + head * p.cap + c0 + warp * kUnit + lane;
    float kscale = 0.f, vscale = 0.f;
    auto load_scales = [&](int i) {
      const int at = i * kAtWarps * kUnit;
      const bool ok = c0 + warp * kUnit + lane + at < c1;
      kscale = ok ? ksb[at] : 0.f;
      vscale = ok ? vsb[at] : 0.f;
    };
    // tokens of an eight that this lane's accumulator columns 2 t, 2 t + 1 stand for
    const int tk[2] = {2 * t, tok_of(2 * t + 1)};

    auto unit = [&](auto tail, int i) {
      constexpr bool TAIL = decltype(tail)::value;
      const uint8_t* kt = ring + 2 * (i % NS) * Z::kTile;
      const uint8_t* vt = kt + Z::kTile;
      const int u0 = c0 + (warp + i * kAtWarps) * kUnit;
      const int left = c1 - u0;                     // tokens of the unit that count
      const int np = TAIL && owner ? pos - u0 : -1;  // the new one among them
      float sc[4][4];
#pragma unroll
      for (int nt = 0; nt < 4; ++nt) {
        const int r = 8 * nt + tok_of(g);
        const uint8_t* row = kt;
        int at0 = stage_at<D>(r, t), at1 = D == 128 ? stage_at<D>(r, 4 + t) : 0;
        if (TAIL && np == r) {
          row = new_s[0];
          at0 -= r * D;
          at1 -= r * D;
        }
        uint4 kw[D / 64];
        kw[0] = *reinterpret_cast<const uint4*>(row + at0);
        if constexpr (D == 128) kw[1] = *reinterpret_cast<const uint4*>(row + at1);
        sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const uint4 q4 = kw[s / 4];
          const uint32_t w = (s % 4) == 0 ? q4.x : (s % 4) == 1 ? q4.y : (s % 4) == 2 ? q4.z : q4.w;
          mma16816(sc[nt], qa[s], Codec<STORE>::template raw_pair<false>(w), Codec<STORE>::template raw_pair<true>(w));
        }
      }
      float x[8], vsc[8];  // index 2 nt + c: token 8 nt + tk[c]
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int tok = 8 * (j >> 1) + tk[j & 1];
        float ks = __shfl_sync(0xffffffffu, kscale, tok);
        vsc[j] = __shfl_sync(0xffffffffu, vscale, tok);
        if (TAIL && np == tok) {
          ks = new_scale[0];
          vsc[j] = new_scale[1];
        }
        float y = fmaf(sc[j >> 1][j & 1] + sc[j >> 1][2 + (j & 1)], qf, qoff) * ks;
        if constexpr (CAP) y = kc * tanh_rel(y);
        x[j] = !TAIL || tok < left ? y : -INFINITY;
        if (TAIL && tok >= left) vsc[j] = 0.f;
      }
      if (i + 1 < mine) load_scales(i + 1);

      // m moves only where a weight would pass 2^4, winv only then or where a product of
      // weight and scale would pass 2^6 of its reference: most units after the first
      // leave the accumulators alone, and the four lanes of a head join their maxima
      // in the others only
      float mx = x[0], cm = 1.f;
#pragma unroll
      for (int j = 1; j < 8; ++j) mx = fmaxf(mx, x[j]);
      const bool moved = __any_sync(0xffffffffu, mx > m + kLazy);
      if (moved) {
#pragma unroll
        for (int d = 1; d <= 2; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
        const float mn = fmaxf(m, mx);
        cm = m == mn ? 1.f : ex2(m - mn);  // m -inf: 0
        ell *= cm;
        m = mn;
      }
      const float me = m == -INFINITY ? 0.f : m;
      float wx = 0.f;  // vsc becomes weight times scale
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float e = ex2(x[j] - me);
        ell += e;
        vsc[j] *= e;
        wx = fmaxf(wx, vsc[j]);
      }
      if (moved || __any_sync(0xffffffffu, wx * winv > kGrow * kUp)) {
#pragma unroll
        for (int d = 1; d <= 2; d <<= 1) wx = fmaxf(wx, __shfl_xor_sync(0xffffffffu, wx, d));
        const float wr = winv > 0.f ? __fdividef(kUp, winv) * cm : 0.f, wn = fmaxf(fmaxf(wr, wx), kTiny), co = wr / wn;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d][0] *= co, o[d][1] *= co, o[d][2] *= co, o[d][3] *= co;
        winv = __fdividef(kUp, wn);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // sixteen tokens: one k step of the second product
        uint32_t pa[4];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int j = 4 * h + 2 * c;
          const float p0 = vsc[j] * winv, p1 = vsc[j + 1] * winv;
          const uint32_t hi = pack_h2(p0, p1);
          const float2 h2 = unpack_h2(hi);
          pa[2 * c] = hi;
          pa[2 * c + 1] = pack_h2(p0 - h2.x, p1 - h2.y);
        }
        uint32_t vw[4][VB / 4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int r = 16 * h + 8 * (k >> 1) + tk[k & 1];
          const uint8_t* row = vt + stage_at<D>(r, D == 128 ? g : g >> 1) + (D == 128 ? 0 : (g & 1) * 8);
          if (TAIL && np == r) row = new_s[1] + (row - vt) - r * D;
          if constexpr (VB == 16) {
            uint4 w = *reinterpret_cast<const uint4*>(row);
            if (TAIL && r >= left) w = make_uint4(0, 0, 0, 0);  // an e4m3 NaN times 0 is one
            vw[k][0] = w.x, vw[k][1] = w.y, vw[k][2] = w.z, vw[k][3] = w.w;
          } else {
            uint2 w = *reinterpret_cast<const uint2*>(row);
            if (TAIL && r >= left) w = make_uint2(0, 0);
            vw[k][0] = w.x, vw[k][1] = w.y;
          }
        }
        // word j of the lane's four tokens holds output dims VB g + 4 j + 0..3
#pragma unroll
        for (int j = 0; j < VB / 4; ++j) {
          const uint32_t a0 = __byte_perm(vw[0][j], vw[1][j], 0x5140), a1 = __byte_perm(vw[0][j], vw[1][j], 0x7362);
          const uint32_t b0 = __byte_perm(vw[2][j], vw[3][j], 0x5140), b1 = __byte_perm(vw[2][j], vw[3][j], 0x7362);
          mma16816(o[4 * j], pa, Codec<STORE>::template pair<false>(a0), Codec<STORE>::template pair<false>(b0));
          mma16816(o[4 * j + 1], pa, Codec<STORE>::template pair<true>(a0), Codec<STORE>::template pair<true>(b0));
          mma16816(o[4 * j + 2], pa, Codec<STORE>::template pair<false>(a1), Codec<STORE>::template pair<false>(b1));
          mma16816(o[4 * j + 3], pa, Codec<STORE>::template pair<true>(a1), Codec<STORE>::template pair<true>(b1));
        }
      }
    };

    load_scales(0);
    bool alive = true;
    for (int i = 0; i < mine; ++i) {
      alive = __all_sync(0xffffffffu, mbar_wait(&full[i % NS], (i / NS) & 1, abort_flag, p.status));
      if (!alive) break;
      // the chunk's last unit may end inside and hold the new token
      if (warp + i * kAtWarps + 1 < units) unit(std::false_type{}, i);
      else unit(std::true_type{}, i);
      __syncwarp();
      if (lane == 0 && i + NS < mine) fill(i + NS);
    }

    // join the warps: n column 2 t + c of tile i is output dim VB (2 t + c) + i
    __syncthreads();  // every warp is through with its ring
    ell += __shfl_xor_sync(0xffffffffu, ell, 1);
    ell += __shfl_xor_sync(0xffffffffu, ell, 2);
    if (t == 0) {
      m_s[warp][g] = m;
      l_s[warp][g] = ell;
    }
    float* ow = o_s + (warp * 8 + g) * OS;
    const float vout = winv > 0.f ? 1.f / winv : 0.f;
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int i = 0; i < ND; i += 4) {
        const int d = VB * (2 * t + c) + i;
        float4 w;
        w.x = (o[i][c] + o[i][2 + c]) * vout;
        w.y = (o[i + 1][c] + o[i + 1][2 + c]) * vout;
        w.z = (o[i + 2][c] + o[i + 2][2 + c]) * vout;
        w.w = (o[i + 3][c] + o[i + 3][2 + c]) * vout;
        *reinterpret_cast<float4*>(ow + d + d / 32 * 4) = w;
      }
  }
  __syncthreads();
  // the warps' shares of each head's joint O: exp2(m_w - M) (and 1 / l where this
  // chunk is the sequence's only one)
  if (threadIdx.x < 8) {
    const int e = threadIdx.x;
    float M = m_s[0][e], l = 0.f;
#pragma unroll
    for (int w = 1; w < kAtWarps; ++w) M = fmaxf(M, m_s[w][e]);
    const float ref = M == -INFINITY ? 0.f : M;
    float c[kAtWarps];
#pragma unroll
    for (int w = 0; w < kAtWarps; ++w) {
      c[w] = ex2(m_s[w][e] - ref);
      l += c[w] * l_s[w][e];
    }
    const float f = active > 1 ? 1.f : l != 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int w = 0; w < kAtWarps; ++w) m_s[w][e] = c[w] * f;
    l_s[0][e] = l;
    if (e < nE) {
      if (active > 1) __stcg(p.ml + (slot0 + split) * 8 + e, make_float2(M, l));
      else p.lse[(int64_t)b * p.Hq + hkv * p.E + e0 + e] = l != 0.f ? (M + log2f(l)) * kLn2 : -INFINITY;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < nE * D; i += kAtThreads) {
    const int e = i / D, d = i - e * D;
    float ov = 0.f;
#pragma unroll
    for (int w = 0; w < kAtWarps; ++w) ov += m_s[w][e] * o_s[(w * 8 + e) * OS + d + d / 32 * 4];
    if (active > 1) __stcg(p.part + ((slot0 + split) * 8 + e) * D + d, ov);
    else static_cast<TQ*>(p.out)[((int64_t)b * p.Hq + hkv * p.E + e0 + e) * D + d] = from_f<TQ>(l_s[0][e] != 0.f ? ov : 0.f);
  }
  close_split<TQ>(p, b, hg, e0, nE, slot0, active, pos, &flag, o_s);
}

// Any head dims up to 256 and any head count: fp32 on the CUDA cores, a warp per
// token, lanes over dims; the same splits and the same join.
constexpr int kAnyDims = 256 / 32, kAnyThreads = 128;
template <typename TQ, int STORE, bool STEP>
__global__ void __launch_bounds__(kAnyThreads) attend_any(AttendParams p) {
  __shared__ float q_s[256], o_s[4][256], m_s[4], l_s[4];
  __shared__ int flag;
  const int split = blockIdx.x, hg = blockIdx.y, b = blockIdx.z;
  const int hkv = hg / p.groups, e0 = (hg - hkv * p.groups) * 8;
  const int nE = min(8, p.E - e0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int pos = max(p.lengths[b], 0);
  const int ntok = (int)min((int64_t)(STEP ? pos + 1 : pos), p.cap);
  const int active = max(1, min(p.splits, (ntok + p.chunk - 1) / p.chunk));
  const int64_t slot0 = ((int64_t)b * p.Hkv * p.groups + hg) * p.splits;
  if (split >= active) {
    if (p.advance) close_split<TQ>(p, b, hg, e0, nE, slot0, active, pos, &flag, &o_s[0][0]);
    return;
  }
  const int c0 = split * p.chunk, c1 = split == active - 1 ? ntok : c0 + p.chunk;
  const int64_t head = (int64_t)b * p.Hkv + hkv;
  if constexpr (STEP) {
    if (split == active - 1 && pos < p.cap) {
      if (warp == 0)
        write_token<TQ, STORE>(p, static_cast<const TQ*>(p.k_t) + b * p.k_sb + hkv * p.k_sh, p.Dk, p.R, pos, head, p.k,
                               p.ks, p.k_new, nullptr, nullptr, [](int) { return 0; });
      if (warp == 1)
        write_token<TQ, STORE>(p, static_cast<const TQ*>(p.v_t) + b * p.v_sb + hkv * p.v_sh, p.Dv, 0, pos, head, p.v,
                               p.vs, p.v_new, nullptr, nullptr, [](int) { return 0; });
    } else if (split == active - 1 && threadIdx.x == 0 && p.status) {
      atomicOr(p.status, TC_DEV_BAD_INDEX);
    }
  }
  for (int e = 0; e < nE; ++e) {
    __syncthreads();
    const TQ* x = static_cast<const TQ*>(p.q) + b * p.q_sb + (int64_t)(hkv * p.E + e0 + e) * p.q_sh;
    for (int u = threadIdx.x; u < (p.Dk + 1) / 2; u += kAnyThreads) {
      int i1, i2;
      float y1, y2;
      load_pair(p, x, u, p.Dk, STEP ? p.R : 0, pos, &i1, &i2, &y1, &y2);
      q_s[i1] = y1;
      q_s[i2] = y2;
    }
    __syncthreads();
    float m = -INFINITY, ell = 0.f, o[kAnyDims];
#pragma unroll
    for (int i = 0; i < kAnyDims; ++i) o[i] = 0.f;
    for (int tok = c0 + warp; tok < c1; tok += 4) {
      const int64_t at = head * p.cap + tok;
      float s = 0.f;
      for (int d = lane; d < p.Dk; d += 32) s += q_s[d] * Codec<STORE>::value(p.k[at * p.Dk + d]);
      float xl = warp_sum(s) * p.ks[at] * p.qscale;
      if (p.has_cap) xl = p.softcap * tanhf(xl / p.softcap);
      xl *= kLog2e;
      const float mn = fmaxf(m, xl), ref = mn == -INFINITY ? 0.f : mn;
      const float cm = m == mn ? 1.f : exp2f(m - mn);
      const float pr = exp2f(xl - ref);  // a NaN logit: NaN, with the maximum as it was
      ell = ell * cm + pr;
      m = mn;
      const float w = pr * p.vs[at];
#pragma unroll
      for (int i = 0; i < kAnyDims; ++i) {
        const int d = lane + 32 * i;
        if (d < p.Dv) o[i] = o[i] * cm + w * Codec<STORE>::value(p.v[at * p.Dv + d]);
      }
    }
#pragma unroll
    for (int i = 0; i < kAnyDims; ++i) o_s[warp][lane + 32 * i] = o[i];
    if (lane == 0) {
      m_s[warp] = m;
      l_s[warp] = ell;
    }
    __syncthreads();
    const float M = fmaxf(fmaxf(m_s[0], m_s[1]), fmaxf(m_s[2], m_s[3])), ref = M == -INFINITY ? 0.f : M;
    for (int d = threadIdx.x; d < p.Dv; d += kAnyThreads) {
      float l = 0.f, ov = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {  // no tokens: 0; NaN logits alone: NaN
        const float c = exp2f(m_s[w] - ref);
        l += c * l_s[w];
        ov += c * o_s[w][d];
      }
      if (active == 1) {
        const int64_t hq = (int64_t)b * p.Hq + hkv * p.E + e0 + e;
        static_cast<TQ*>(p.out)[hq * p.Dv + d] = from_f<TQ>(l != 0.f ? ov / l : 0.f);
        if (d == 0) p.lse[hq] = l != 0.f ? (M + log2f(l)) * kLn2 : -INFINITY;
      } else {
        const int64_t at = (slot0 + split) * 8 + e;
        __stcg(p.part + at * p.Dv + d, ov);
        if (d == 0) __stcg(p.ml + at, make_float2(M, l));
      }
    }
  }
  close_split<TQ>(p, b, hg, e0, nE, slot0, active, pos, &flag, &o_s[0][0]);
}

// Codes [rows * Hkv, capacity, D] as a 3-D map of kUnit-token boxes, slots past the
// capacity reading as zeros.
template <int D>
int code_map(CUtensorMap* m, const void* base, const AttendParams& p, int64_t heads) {
  auto fn = tcx::encode_fn();
  if (!fn) return TC_ERR_CUDA;
  cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)p.cap, (cuuint64_t)heads};
  cuuint64_t strides[2] = {(cuuint64_t)D, (cuuint64_t)D * p.cap};
  cuuint32_t box[3] = {(cuuint32_t)D, (cuuint32_t)kUnit, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? TC_OK : TC_ERR_CUDA;
}

template <typename TQ, int STORE, int D, bool CAP, bool STEP>
int launch_mma(const AttendParams& p, int64_t heads, dim3 grid, cudaStream_t st) {
  CUtensorMap mk, mv;
  if (int rc = code_map<D>(&mk, p.k, p, heads)) return rc;
  if (int rc = code_map<D>(&mv, p.v, p, heads)) return rc;
  auto k = attend_mma<TQ, STORE, D, CAP, STEP>;
  constexpr int smem = AtSmem<D>::kBytes;
  if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return TC_ERR_CUDA;
  k<<<grid, kAtThreads, smem, st>>>(mk, mv, p);
  return launch_status();
}

template <typename TQ, int STORE, bool STEP>
int launch_attend(const AttendParams& p, int64_t rows, cudaStream_t st) {
  const dim3 grid(p.splits, p.Hkv * p.groups, p.B);
  const int64_t heads = rows * p.Hkv;
  const bool mma = p.Dk == p.Dv && (p.Dk == 64 || p.Dk == 128) && (uintptr_t)p.k % 16 == 0 && (uintptr_t)p.v % 16 == 0 &&
                   heads <= INT32_MAX && p.cap * p.Dk < (int64_t(1) << 40) && !(p.has_cap && p.softcap < 1e-30f);
  if (mma && p.Dk == 128)
    return p.has_cap ? launch_mma<TQ, STORE, 128, true, STEP>(p, heads, grid, st)
                     : launch_mma<TQ, STORE, 128, false, STEP>(p, heads, grid, st);
  if (mma)
    return p.has_cap ? launch_mma<TQ, STORE, 64, true, STEP>(p, heads, grid, st)
                     : launch_mma<TQ, STORE, 64, false, STEP>(p, heads, grid, st);
  attend_any<TQ, STORE, STEP><<<grid, kAnyThreads, 0, st>>>(p);
  return launch_status();
}

bool cache_ok(const tc_kv_cache* c) {
  return c && c->rows >= 0 && c->Hkv > 0 && c->Dk > 0 && c->Dv > 0 && c->capacity > 0 &&
         (c->store == TC_KV_INT8 || c->store == TC_KV_FP8) && c->k && c->v && c->k_scale && c->v_scale && c->lengths;
}

// Tokens per CTA and CTAs per (sequence, head group) over at most `most` tokens.
// One sequence: one wave of three CTAs per SM over 148 SMs.  Several may differ
// in length: eight waves, so that they even out (64 sequences of 1 to 32768
// tokens, with the kernel as it was at 294 us: 360 us with two, 302 with four, 294
// with eight, 301 with sixteen).  A chunk is a multiple of 64 tokens.
void split_rule(int64_t most, int64_t heads, int B, int* chunk, int* splits) {
  const int64_t resident = 3 * 148;
  const int64_t want = B > 1 ? (8 * resident + heads - 1) / heads : heads < resident ? resident / heads : 1;
  int64_t c = (most + want - 1) / want;
  c = (c + 63) / 64 * 64;
  if (c < 64) c = 64;
  const int64_t s = (most + c - 1) / c;
  *chunk = (int)c;
  *splits = (int)(s < 1 ? 1 : s);
}

}  // namespace

extern "C" int tc_kv_write(const tc_kv_cache* c, const tc_kv_write_args* a, void* stream) {
  if (!cache_ok(c) || !a || a->B < 0 || a->N < 0) return TC_ERR_ARG;
  if (a->N == 0 && a->B > 0 && a->fresh && !a->seq_idx) {  // B prompts of no tokens
    if (a->B > c->rows) return TC_ERR_ARG;
    return cudaMemsetAsync(c->lengths, 0, a->B * sizeof(int32_t), (cudaStream_t)stream) == cudaSuccess ? TC_OK : TC_ERR_CUDA;
  }
  if ((int64_t)a->B * a->N == 0) return TC_OK;
  if (!a->k || !a->v || (a->seq_idx && !a->starts) || (!a->seq_idx && a->B > c->rows)) return TC_ERR_ARG;
  WriteParams p;
  p.B = a->B, p.N = a->N, p.H = c->Hkv, p.rows = c->rows, p.fresh = a->fresh != 0;
  p.cap = c->capacity;
  p.k = {a->k, a->k_stride_b, a->k_stride_n, a->k_stride_h, c->k, c->k_scale, c->Dk};
  p.v = {a->v, a->v_stride_b, a->v_stride_n, a->v_stride_h, c->v, c->v_scale, c->Dv};
  p.lengths = c->lengths;
  p.seq = a->seq_idx, p.starts = a->starts;
  p.status = a->dev_status;
  cudaStream_t st = (cudaStream_t)stream;
  if (c->store == TC_KV_INT8) { TC_DISPATCH(a->dtype, T, return launch_write<T, TC_KV_INT8>(p, st)); }
  else { TC_DISPATCH(a->dtype, T, return launch_write<T, TC_KV_FP8>(p, st)); }
}

extern "C" int tc_kv_read(const tc_kv_cache* c, int32_t length, int32_t dtype, void* k_out, void* v_out, void* stream) {
  if (!cache_ok(c) || length < 0 || !k_out || !v_out) return TC_ERR_ARG;
  if ((int64_t)c->rows * length == 0) return TC_OK;
  ReadParams p;
  p.rows = c->rows, p.H = c->Hkv, p.L = length, p.cap = c->capacity;
  p.k = {c->k, c->k_scale, c->Dk, k_out};
  p.v = {c->v, c->v_scale, c->Dv, v_out};
  p.lengths = c->lengths;
  cudaStream_t st = (cudaStream_t)stream;
  if (c->store == TC_KV_INT8) { TC_DISPATCH(dtype, T, return launch_read<T, TC_KV_INT8>(p, st)); }
  else { TC_DISPATCH(dtype, T, return launch_read<T, TC_KV_FP8>(p, st)); }
}

static int attend_shape(const tc_kv_cache* c, int32_t B, int32_t Hq, int32_t max_tokens, int* chunk, int* splits) {
  if (!cache_ok(c) || B < 0 || Hq <= 0 || Hq % c->Hkv || max_tokens < 0) return TC_ERR_ARG;
  const int groups = (Hq / c->Hkv + 7) / 8;
  split_rule(max_tokens < 1 ? 1 : max_tokens, (int64_t)(B < 1 ? 1 : B) * c->Hkv * groups, B, chunk, splits);
  return TC_OK;
}

extern "C" int64_t tc_kv_attend_scratch_floats(const tc_kv_cache* c, int32_t B, int32_t Hq, int32_t max_tokens) {
  int chunk, splits;
  if (attend_shape(c, B, Hq, max_tokens, &chunk, &splits)) return -1;
  const int groups = (Hq / c->Hkv + 7) / 8;
  return splits > 1 ? (int64_t)B * c->Hkv * groups * splits * 8 * (c->Dv + 2) : 0;
}

extern "C" int tc_kv_attend(const tc_kv_cache* c, const tc_kv_attend_args* a, void* stream) {
  if (!a) return TC_ERR_ARG;
  AttendParams p;
  if (int rc = attend_shape(c, a->B, a->Hq, a->max_tokens, &p.chunk, &p.splits)) return rc;
  if (a->B == 0) return TC_OK;
  if (a->B > c->rows || !a->q || !a->out || !a->lse || a->max_tokens > c->capacity) return TC_ERR_ARG;
  if (!std::isfinite(a->scale) || (a->has_softcap && !(a->softcap > 0.f && std::isfinite(a->softcap)))) return TC_ERR_ARG;
  if (c->Dk > 256 || c->Dv > 256 || a->B > 65535) return TC_ERR_UNSUPPORTED;
  const bool step = a->k_t != nullptr;
  if (step && !a->v_t) return TC_ERR_ARG;
  if (a->R < 0 || a->R % 2 || a->R > c->Dk || (a->R && (!a->rope_cos || !a->rope_sin || a->n_pos <= 0 || !step)))
    return TC_ERR_ARG;
  p.groups = (a->Hq / c->Hkv + 7) / 8;
  if ((int64_t)c->Hkv * p.groups > 65535) return TC_ERR_UNSUPPORTED;
  const int64_t need = p.splits > 1 ? (int64_t)a->B * c->Hkv * p.groups * p.splits * 8 * (c->Dv + 2) : 0;
  if (need && (!a->scratch || (uintptr_t)a->scratch % 16 || a->scratch_floats < need)) return TC_ERR_ARG;
  if ((p.splits > 1 || a->advance) && (!a->counters || a->num_counters < (int64_t)a->B * (c->Hkv * p.groups + 1)))
    return TC_ERR_ARG;
  p.B = a->B, p.Hq = a->Hq, p.Hkv = c->Hkv, p.E = a->Hq / c->Hkv;
  p.Dk = c->Dk, p.Dv = c->Dv, p.cap = c->capacity;
  p.k = c->k, p.v = c->v, p.ks = c->k_scale, p.vs = c->v_scale, p.lengths = c->lengths;
  p.q = a->q, p.q_sb = a->q_stride_b, p.q_sh = a->q_stride_h;
  p.k_t = a->k_t, p.v_t = a->v_t;
  p.k_sb = a->k_stride_b, p.k_sh = a->k_stride_h, p.v_sb = a->v_stride_b, p.v_sh = a->v_stride_h;
  p.cos_t = a->rope_cos, p.sin_t = a->rope_sin, p.R = a->R, p.interleaved = a->interleaved != 0, p.n_pos = a->n_pos;
  p.qscale = a->scale, p.softcap = a->softcap, p.has_cap = a->has_softcap != 0;
  p.advance = step && a->advance;
  p.out = a->out, p.lse = a->lse, p.k_new = a->k_new, p.v_new = a->v_new, p.new_dtype = a->new_dtype;
  const int64_t slots = (int64_t)a->B * c->Hkv * p.groups * p.splits;
  p.ml = reinterpret_cast<float2*>(a->scratch), p.part = a->scratch + slots * 16;
  p.done = a->counters, p.status = a->dev_status;
  cudaStream_t st = (cudaStream_t)stream;
#define TC_KV_GO(S, STEP) TC_DISPATCH(a->dtype, T, return launch_attend<T, S, STEP>(p, c->rows, st))
  if (c->store == TC_KV_INT8) {
    if (step) { TC_KV_GO(TC_KV_INT8, true); }
    else { TC_KV_GO(TC_KV_INT8, false); }
  } else {
    if (step) { TC_KV_GO(TC_KV_FP8, true); }
    else { TC_KV_GO(TC_KV_FP8, false); }
  }
#undef TC_KV_GO
}

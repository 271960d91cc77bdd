// Pieces shared by the tensor-core kernels of packed causal attention.
#pragma once

#include "causal.cuh"
#include "tc_common.cuh"

namespace tc {
namespace ctc {

using namespace ptx;
using namespace tcx;

constexpr int KT = 128;  // keys per tile of the forward

// [B, N, H, D] through its strides as a 4-D map (d, h, n, b) of 64 x 1 x rows x 1
// boxes with the 128-byte swizzle; tokens past N read as zeros.  The stride of a
// dimension of size one is never used: any valid one stands in.
inline int make_map_strided(CUtensorMap* m, const void* base, int dt, int64_t B, int64_t N, int64_t H, int D, int64_t sb,
                            int64_t sn, int64_t sh, int rows) {
  auto fn = encode_fn();
  if (!fn) return TC_ERR_CUDA;
  const CUtensorMapDataType t = dt == TC_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  if (H == 1) sh = D;
  if (N == 1) sn = D * H;
  if (B == 1) sb = sn * N;
  cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)H, (cuuint64_t)N, (cuuint64_t)B};
  cuuint64_t strides[3] = {(cuuint64_t)sh * 2, (cuuint64_t)sn * 2, (cuuint64_t)sb * 2};
  cuuint32_t box[4] = {64, 1, (cuuint32_t)rows, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  CUresult r = fn(m, t, 4, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? TC_OK : TC_ERR_CUDA;
}

// A rows x HD tile: HD / 64 swizzled blocks of rows x 64.
template <int HD, int ROWS>
__device__ __forceinline__ void load_rows(uint8_t* dst, const CUtensorMap* m, int h, int n, int b, uint64_t* bar) {
#pragma unroll
  for (int c = 0; c < HD / 64; ++c) tma_load_4d(dst + c * ROWS * 128, m, 64 * c, h, n, b, bar);
}

// MMA issue by a converged warp: every lane walks the loop, so that descriptors
// stay in uniform registers, and one elected lane issues.  (One lane alone in
// the branch had the issue of 24 products take 2200 cycles: each operand moved
// to a uniform register by itself.)  Descriptors: the low word holds the
// address and the leading offset, the high word is the same for every operand
// here (1024-byte stride of 8-row groups, 128-byte swizzle).
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(const void* s, uint32_t lbo) {
  return ((smem_addr(s) & 0x3FFFFu) >> 4) | ((lbo >> 4) << 16);
}
// K-major 128 x 16 tile without swizzle: element (r, k) at (k / 8) * kAugHalf +
// r * 16 + (k % 8) * 2.
constexpr uint32_t kAugHalf = 128 * 16, kAugTile = 2 * kAugHalf;
constexpr uint32_t kAugHi = (128u >> 4) | (1u << 14);
__device__ __forceinline__ uint32_t aug_lo(const void* s) {
  return ((smem_addr(s) & 0x3FFFFu) >> 4) | ((kAugHalf >> 4) << 16);
}
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t alo, uint32_t blo, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %5};\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d),
      "r"(alo), "r"(blo), "r"(idesc), "r"(acc), "n"(kDescHi)
      : "memory");
}
// d += A B^T of two such tiles, bf16 whatever the other operands' type.
__device__ __forceinline__ void mma_aug(uint32_t d, uint32_t alo, uint32_t blo) {
  asm volatile(
      "{\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %4};\n\t"
      "mov.b64 b, {%2, %4};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, 1;\n\t}" ::"r"(d),
      "r"(alo), "r"(blo), "r"(idesc_f16(128, 128, 1, 0, 0)), "n"(kAugHi)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t blo, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(blo), "r"(idesc), "r"(acc), "n"(kDescHi)
      : "memory");
}
// d = A B^T of two K-major 128 x HD tiles.
template <int HD>
__device__ __forceinline__ void mma_tile_ss(uint32_t d, uint32_t alo, uint32_t blo, uint32_t idesc) {
#pragma unroll
  for (int kk = 0; kk < HD / 16; ++kk) {
    const uint32_t off = ((kk >> 2) * 128 * 128 + (kk & 3) * 32) >> 4;
    mma_ss(d, alo + off, blo + off, idesc, kk > 0 ? 1u : 0u);
  }
}
// d (+)= A B of A [128 x 128] in TMEM as 16-bit pairs, STEPS 16-element steps
// (8 columns each) to every STRIDE columns, and an MN-major 128 x HD tile.
template <int STEPS, int STRIDE>
__device__ __forceinline__ void mma_tile_ts(uint32_t d, uint32_t a, uint32_t blo, uint32_t idesc, uint32_t acc) {
#pragma unroll
  for (int kk = 0; kk < 8; ++kk)
    mma_ts(d, a + (kk / STEPS) * STRIDE + (kk % STEPS) * 8, blo + ((kk * 2048) >> 4), idesc, kk > 0 ? 1u : acc);
}
// A value that every lane holds alike, known to be uniform.
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

// One arrival for the warp, behind every lane's accesses (barriers of the compute
// warps count warps: 32 arrivals on one address would be served one by one).
__device__ __forceinline__ void warp_arrive(uint64_t* bar, int lane) {
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}

// Grid of a pass whose CTAs are (block, head, sequence): blocks first, so that
// the heaviest blocks of every head start before any light one (the long
// training case ends 12% earlier), while what the heads stream, `bytes`, stays
// in half of the L2; else head by head, so that a head's blocks share it.
constexpr int64_t kShareBytes = int64_t(64) << 20;
struct GridOrder {
  int heads, by_block;
};
inline dim3 grid_order(int blocks, int heads, int B, int64_t bytes, GridOrder* o) {
  o->heads = heads;
  o->by_block = bytes <= kShareBytes && blocks <= 65535;
  return o->by_block ? dim3((unsigned)heads * B, blocks, 1) : dim3(blocks, heads, B);
}
__device__ __forceinline__ void grid_place(const GridOrder& o, int* block, int* head, int* b) {
  *block = o.by_block ? blockIdx.y : blockIdx.x;
  *head = o.by_block ? blockIdx.x % o.heads : blockIdx.y;
  *b = o.by_block ? blockIdx.x / o.heads : blockIdx.z;
}
__device__ __forceinline__ int grid_blocks(const GridOrder& o) { return o.by_block ? gridDim.y : gridDim.x; }

inline bool strides_ok(const void* p, int64_t sb, int64_t sn, int64_t sh, int64_t B, int64_t N, int64_t H) {
  const int64_t most = int64_t(1) << 38;  // elements: a map's byte stride stays below 2^40
  return (uintptr_t)p % 16 == 0 && (B == 1 || (sb % 8 == 0 && sb > 0 && sb < most)) &&
         (N == 1 || (sn % 8 == 0 && sn > 0 && sn < most)) && (H == 1 || (sh % 8 == 0 && sh > 0 && sh < most));
}

// The kernels take a row's reference from its largest raw score and divide lse by
// the scale: it is positive, and lse / scale and scale s stay in fp32's range.  Their
// tanh by 1 - 2 / (e^2y + 1) is off by 3e-7 at most, the logit by that times the
// softcap: above 2048 (6e-4) it shows in the weights.  Any other scale or softcap
// takes the CUDA cores.
inline bool logits_ok(const CausalParams& p) {
  const float kq = p.has_cap ? p.scale / p.cap : p.scale;
  return p.scale >= 1e-30f && p.scale <= 1e30f && kq <= 1e30f && (!p.has_cap || p.cap <= 2048.f);
}

inline bool tc_shape(const CausalParams& p, int dtype) {
  return logits_ok(p) && (dtype == TC_BF16 || dtype == TC_F16) && p.Dk == p.Dv && (p.Dk == 64 || p.Dk == 128) &&
         strides_ok(p.q, p.q_sb, p.q_sn, p.q_sh, p.B, p.N, p.Hq) &&
         strides_ok(p.k, p.k_sb, p.k_sn, p.k_sh, p.B, p.N, p.Hkv) &&
         strides_ok(p.v, p.v_sb, p.v_sn, p.v_sh, p.B, p.N, p.Hkv);
}

}  // namespace ctc
}  // namespace tc

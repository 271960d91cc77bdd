// Parameters of the packed causal attention kernels.
#pragma once

#include "common.cuh"

namespace tc {

struct CausalParams {
  int B, N, Hq, Hkv, E, Dk, Dv;
  float scale, cap;
  int has_cap;
  const void* q;
  const void* k;
  const void* v;
  int64_t q_sb, q_sn, q_sh, k_sb, k_sn, k_sh, v_sb, v_sn, v_sh;
  const int32_t* starts;  // [B, N] or null
  const int32_t* ends;
  void* out;
  float* lse;
  void* out_low;
  const void* o;
  const void* o_low;
  const void* dout;
  const float* dlse;
  float* delta;
  void* dq;
  void* dk;
  void* dv;
  int32_t* status;
  bool vec4;  // rows of q, k, v, dout start on four elements, and their lengths are multiples
};

// First key that query n of row b sees (its last is n itself); n + 1 where it
// sees none.  Nondecreasing in n.  Bounds may come from the caller: kept inside
// the row, where every tile that they lead to can be read.
__device__ __forceinline__ int first_key(const CausalParams& p, int b, int n) {
  return p.starts ? max(__ldg(p.starts + (int64_t)b * p.N + n), 0) : 0;
}
// End of the queries that see key n (the first is n itself); n where none do.
// Nondecreasing in n.
__device__ __forceinline__ int query_end(const CausalParams& p, int b, int n) {
  return p.ends ? min(__ldg(p.ends + (int64_t)b * p.N + n), p.N) : p.N;
}

bool causal_tc_supported(const CausalParams& p, int dtype);
int causal_fwd_tc(const CausalParams& p, int dtype, cudaStream_t st);
bool causal_bwd_tc_supported(const CausalParams& p, int dtype);
int causal_bwd_tc(const CausalParams& p, int dtype, cudaStream_t st);
int causal_delta(const CausalParams& p, int dtype, cudaStream_t st);

}  // namespace tc

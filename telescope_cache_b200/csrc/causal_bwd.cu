#include "causal_tc.cuh"
namespace tc {
bool causal_bwd_tc_supported(const CausalParams&, int) { return false; }
int causal_bwd_tc(const CausalParams&, int, cudaStream_t) { return TC_ERR_UNSUPPORTED; }
}  // namespace tc

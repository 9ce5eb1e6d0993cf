// The feed-forward products (ffn_tc.cuh) on BF16.
#include "ffn_tc.cuh"

namespace j1rt {
int launch_ffn_tc_bf16(int cfg, int layout, int gated, FfnTc& p, cudaStream_t stream) {
  return ffn::launch_tc<__nv_bfloat16>(cfg, layout, gated, p, stream);
}
cudaError_t load_ffn_tc_bf16() { return ffn::load_tc<__nv_bfloat16>(); }
}  // namespace j1rt

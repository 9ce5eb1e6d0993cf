// The feed-forward products (ffn_tc.cuh) on FP16.
#include "ffn_tc.cuh"

namespace j1rt {
int launch_ffn_tc_fp16(int cfg, int layout, int gated, FfnTc& p, cudaStream_t stream) {
  return ffn::launch_tc<__half>(cfg, layout, gated, p, stream);
}
cudaError_t load_ffn_tc_fp16() { return ffn::load_tc<__half>(); }
}  // namespace j1rt

// fms_glu_bf16.cu -- the gated feed-forward block in bfloat16 (a file per type: they compile
// side by side).
#include "fms_glu.cuh"

namespace fms {
cudaError_t run_ffn_bf16(int dtype, int act, const glu::Args& p, bool bwd, cudaStream_t s) {
  return glu::run_act<__nv_bfloat16>(dtype, act, p, bwd, s);
}
int read_ffn_bf16_error(int reset) { return gemm::read_error(reset); }
}  // namespace fms

// fms_glu_f16.cu -- the gated feed-forward block in f16 (a file per type: they compile
// side by side).
#include "fms_glu.cuh"

namespace fms {
cudaError_t run_ffn_f16(int dtype, int act, const glu::Args& p, bool bwd, cudaStream_t s) {
  return glu::run_act<__half>(dtype, act, p, bwd, s);
}
int read_ffn_f16_error(int reset) { return gemm::read_error(reset); }
}  // namespace fms

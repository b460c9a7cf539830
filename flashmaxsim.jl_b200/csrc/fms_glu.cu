// fms_glu.cu -- entry points of the gated feed-forward block (fms_glu.cuh).
#include "fms_glu.cuh"

namespace fms {

cudaError_t run_ffn_f16(int dtype, int act, const glu::Args& p, bool bwd, cudaStream_t s);
cudaError_t run_ffn_bf16(int dtype, int act, const glu::Args& p, bool bwd, cudaStream_t s);
int read_ffn_f16_error(int reset);
int read_ffn_bf16_error(int reset);

namespace glu {

static int check(int dtype, int act, int64_t rows, int dim, int hidden) {
  if (dtype != FMS_F16 && dtype != FMS_BF16) return FMS_ERR_DTYPE;
  if (act < FMS_ACT_SILU || act > FMS_ACT_RELU) return FMS_ERR_INVALID;
  // row and column coordinates of a tile are 32-bit
  if (rows < 0 || rows > INT32_MAX - 512 || dim < 0 || dim > INT32_MAX - 512 || hidden < 0 || hidden > INT32_MAX - 512)
    return FMS_ERR_INVALID;
  return FMS_OK;
}

static int launch(int dtype, int act, const Args& p, bool bwd, cudaStream_t s) {
  if (device_cc() != 100) return FMS_ERR_UNSUPPORTED;
  const cudaError_t e = dtype == FMS_F16 ? run_ffn_f16(dtype, act, p, bwd, s) : run_ffn_bf16(dtype, act, p, bwd, s);
  return e == cudaSuccess ? FMS_OK : e == cudaErrorNotSupported ? FMS_ERR_UNSUPPORTED : (int)e;
}

}  // namespace glu

int read_ffn_device_error(int reset) {
  const int a = read_ffn_f16_error(reset), b = read_ffn_bf16_error(reset);
  return a != 0 ? a : b;
}

}  // namespace fms

using namespace fms;

extern "C" {

size_t fms_gated_ffn_workspace_size(int64_t rows, int dim, int hidden, int backward) {
  if (rows <= 0 || dim <= 0 || hidden <= 0) return 0;
  return glu::space(rows, dim, hidden, backward != 0).total;
}

int fms_gated_ffn_fwd(int dtype, const void* x, const void* w_gate, const void* w_up, int64_t rows, int dim,
                      int hidden, int act, void* h, void* workspace, size_t ws_bytes, fms_stream_t stream) {
  const int st = glu::check(dtype, act, rows, dim, hidden);
  if (st != FMS_OK) return st;
  if (rows == 0 || hidden == 0) return FMS_OK;
  if (!h || (dim > 0 && (!x || !w_gate || !w_up))) return FMS_ERR_INVALID;
  if (dim == 0) {  // empty sums
    const cudaError_t e = cudaMemsetAsync(h, 0, (size_t)rows * hidden * 2, (cudaStream_t)stream);
    return e == cudaSuccess ? FMS_OK : (int)e;
  }
  const size_t need = fms_gated_ffn_workspace_size(rows, dim, hidden, 0);
  if (need && (!workspace || ws_bytes < need)) return FMS_ERR_WORKSPACE;
  return glu::launch(dtype, act,
                     {x, w_gate, w_up, nullptr, rows, dim, hidden, h, nullptr, nullptr, nullptr, (char*)workspace}, false,
                     (cudaStream_t)stream);
}

int fms_gated_ffn_bwd(int dtype, const void* x, const void* w_gate, const void* w_up, const void* dh, int64_t rows,
                      int dim, int hidden, int act, void* dx, void* dw_gate, void* dw_up, void* workspace,
                      size_t ws_bytes, fms_stream_t stream) {
  const int st = glu::check(dtype, act, rows, dim, hidden);
  if (st != FMS_OK) return st;
  if (dim == 0) return FMS_OK;
  if (rows == 0 || hidden == 0) {  // empty sums
    cudaError_t e = cudaSuccess;
    if (dx) e = cudaMemsetAsync(dx, 0, (size_t)rows * dim * 2, (cudaStream_t)stream);
    if (dw_gate && e == cudaSuccess) e = cudaMemsetAsync(dw_gate, 0, (size_t)hidden * dim * 2, (cudaStream_t)stream);
    if (dw_up && e == cudaSuccess) e = cudaMemsetAsync(dw_up, 0, (size_t)hidden * dim * 2, (cudaStream_t)stream);
    return e == cudaSuccess ? FMS_OK : (int)e;
  }
  if (!x || !w_gate || !w_up || !dh) return FMS_ERR_INVALID;
  if (!workspace || ws_bytes < fms_gated_ffn_workspace_size(rows, dim, hidden, 1)) return FMS_ERR_WORKSPACE;
  return glu::launch(dtype, act, {x, w_gate, w_up, dh, rows, dim, hidden, nullptr, dx, dw_gate, dw_up, (char*)workspace},
                     true, (cudaStream_t)stream);
}

}  // extern "C"

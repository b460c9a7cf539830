// fms_linear_int8.cu -- linear layer in 8-bit integers with one scale per token
// and one per output channel:
//
//   y[t,c] = (sx_t * sw_c) * float(sum_k xc[t,k] * wc[c,k]) + b_c
//
// The integer sum is exact (int32; the entry point bounds K).  Float inputs are
// quantised per token first, in float32 whatever their type: scale =
// max(absmax, 1e-8) * (1/127), code = round to nearest even of x / scale.
#include "fms_common.cuh"
#include "fms_internal.h"

namespace fms {
namespace lin8 {

// One warp per token: absmax, then codes.
template <typename T>
__global__ void __launch_bounds__(256) quantize_kernel(const T* x, int64_t rows, int K, int8_t* codes, float* scales) {
  const int lane = threadIdx.x & 31;
  const int64_t t = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (t >= rows) return;
  const T* xt = x + t * K;
  uint32_t top = 0;  // bits of the largest |x|; as whole numbers a NaN's are above infinity's
  for (int k = lane; k < K; k += 32) top = max(top, __float_as_uint(fabsf(Tr<T>::to(xt[k]))));
  top = __reduce_max_sync(0xffffffffu, top);
  const float am = __uint_as_float(top);
  // a token that holds an infinity or a NaN has no scale: all its outputs are NaN
  const float sc = am <= 3.402823466e38f ? fmaxf(am, 1e-8f) * (1.f / 127.f) : NAN;
  for (int k = lane; k < K; k += 32) {
    const float v = rintf(fminf(fmaxf(Tr<T>::to(xt[k]) / sc, -127.f), 127.f));
    codes[t * K + k] = (int8_t)v;
  }
  if (lane == 0) scales[t] = sc;
}

constexpr int TILE = 64, KT = 32, NT = 256;

template <typename T>
__global__ void __launch_bounds__(NT) linear_kernel(const int8_t* xc, const float* sx, const int8_t* wc,
                                                    const float* sw, const T* bias, int64_t rows, int K, int C, T* y) {
  __shared__ int32_t Xs[KT / 4][TILE + 1], Ws[KT / 4][TILE + 1];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int64_t m0 = (int64_t)blockIdx.x * TILE;
  const int n0 = blockIdx.y * TILE;
  int32_t acc[4][4] = {};
  for (int k0 = 0; k0 < K; k0 += KT) {
    for (int e = threadIdx.x; e < TILE * (KT / 4); e += NT) {
      const int kk = e % (KT / 4), i = e / (KT / 4);
      uint32_t xw = 0, ww = 0;
      for (int b = 0; b < 4; ++b) {
        const int k = k0 + kk * 4 + b;
        if (k < K && m0 + i < rows) xw |= (uint32_t)(uint8_t)xc[(m0 + i) * K + k] << (8 * b);
        if (k < K && n0 + i < C) ww |= (uint32_t)(uint8_t)wc[(int64_t)(n0 + i) * K + k] << (8 * b);
      }
      Xs[kk][i] = (int32_t)xw;
      Ws[kk][i] = (int32_t)ww;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < KT / 4; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(Xs[k][ty + 16 * i], Ws[k][tx + 16 * j], acc[i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t t = m0 + ty + 16 * i;
      const int c = n0 + tx + 16 * j;
      if (t >= rows || c >= C) continue;
      float v = (sx[t] * sw[c]) * (float)acc[i][j];
      if (bias) v += Tr<T>::to(bias[c]);
      y[t * C + c] = Tr<T>::from(v);
    }
}

static size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

template <typename T>
static void quantize(const void* x, int64_t rows, int K, int8_t* codes, float* scales, cudaStream_t s) {
  quantize_kernel<T><<<(unsigned)((rows + 7) / 8), 256, 0, s>>>((const T*)x, rows, K, codes, scales);
}

template <typename T>
static void linear(const int8_t* xc, const float* sx, const int8_t* wc, const float* sw, const void* bias, int64_t rows,
                   int K, int C, void* y, cudaStream_t s) {
  const dim3 grid((unsigned)((rows + TILE - 1) / TILE), (unsigned)((C + TILE - 1) / TILE));
  linear_kernel<T><<<grid, NT, 0, s>>>(xc, sx, wc, sw, (const T*)bias, rows, K, C, (T*)y);
}

}  // namespace lin8

int read_lin8_device_error(int) { return 0; }

}  // namespace fms

using namespace fms;

extern "C" {

size_t fms_int8_linear_workspace_size(int x_dtype, int64_t rows, int dim, int out) {
  if (rows <= 0 || dim <= 0 || out <= 0 || x_dtype == FMS_I8) return 0;
  return lin8::align256((size_t)rows * dim) + (size_t)rows * 4;
}

int fms_int8_linear_fwd(int x_dtype, const void* x, const float* x_scales, const int8_t* w_codes, const float* w_scales,
                        const void* bias, int64_t rows, int dim, int out, int y_dtype, void* y, void* workspace,
                        size_t ws_bytes, fms_stream_t stream) {
  if (x_dtype != FMS_I8 && x_dtype != FMS_F32 && x_dtype != FMS_F16 && x_dtype != FMS_BF16) return FMS_ERR_DTYPE;
  if (y_dtype != FMS_F32 && y_dtype != FMS_F16 && y_dtype != FMS_BF16) return FMS_ERR_DTYPE;
  if (rows < 0 || rows > INT32_MAX || dim < 1 || out < 0) return FMS_ERR_INVALID;
  if (dim > FMS_INT8_LINEAR_MAX_DIM) return FMS_ERR_TOO_LARGE;
  if (rows == 0 || out == 0) return FMS_OK;
  if (!y || !w_scales || !x || !w_codes || (x_dtype == FMS_I8 && !x_scales)) return FMS_ERR_INVALID;
  const size_t need = fms_int8_linear_workspace_size(x_dtype, rows, dim, out);
  if (need && (!workspace || ws_bytes < need)) return FMS_ERR_WORKSPACE;
  cudaStream_t s = (cudaStream_t)stream;
  const int8_t* xc = (const int8_t*)x;
  const float* sx = x_scales;
  if (x_dtype != FMS_I8) {
    int8_t* c = (int8_t*)workspace;
    float* sc = (float*)((char*)workspace + lin8::align256((size_t)rows * dim));
    if (x_dtype == FMS_F32) lin8::quantize<float>(x, rows, dim, c, sc, s);
    else if (x_dtype == FMS_F16) lin8::quantize<__half>(x, rows, dim, c, sc, s);
    else lin8::quantize<__nv_bfloat16>(x, rows, dim, c, sc, s);
    xc = c;
    sx = sc;
  }
  if (y_dtype == FMS_F32) lin8::linear<float>(xc, sx, w_codes, w_scales, bias, rows, dim, out, y, s);
  else if (y_dtype == FMS_F16) lin8::linear<__half>(xc, sx, w_codes, w_scales, bias, rows, dim, out, y, s);
  else lin8::linear<__nv_bfloat16>(xc, sx, w_codes, w_scales, bias, rows, dim, out, y, s);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? FMS_OK : (int)e;
}

}  // extern "C"

// fms_glu.cu -- the gated feed-forward block of a token encoder:
//
//   g = x Wg^T,  u = x Wu^T,  h = a(g) * u                      (forward)
//   du = dh * a(g),  dg = dh * u * a'(g)                        (backward)
//   dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x
//
// x (rows, dim), Wg and Wu (hidden, dim), h (rows, hidden), 16-bit; sums in
// float32.  g and u are not kept for the backward pass but computed again: that
// is one more pair of products, and saves rounding them to 16 bits and
// 4 * rows * hidden bytes between the passes.
#include "fms_act.cuh"
#include "fms_internal.h"

namespace fms {
namespace glu {

constexpr int TILE = 64, KT = 16, NT = 256;  // output tile, K step, threads

// One 64 x 64 tile of C = sum over the operand pairs of A(m,k) B(k,n), float32
// sums, 4 x 4 per thread.  A element (m,k) at a[m*sam + k*sak], B (k,n) at
// b[k*sbk + n*sbn].
template <typename T>
struct Strided {
  const T* a;
  const T* b;
  int64_t sam, sak, sbk, sbn;
};

template <typename T>
__device__ __forceinline__ void tile_product(const Strided<T>& s, int64_t m0, int64_t n0, int64_t M, int64_t N,
                                             int64_t K, float (*As)[TILE + 4], float (*Bs)[TILE + 4],
                                             float (&acc)[4][4]) {
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  for (int64_t k0 = 0; k0 < K; k0 += KT) {
    for (int e = threadIdx.x; e < TILE * KT; e += NT) {
      // neighbouring threads along the operand's contiguous axis
      const int mi = s.sak == 1 ? e / KT : e % TILE, ka = s.sak == 1 ? e % KT : e / TILE;
      const int ni = s.sbk == 1 ? e / KT : e % TILE, kb = s.sbk == 1 ? e % KT : e / TILE;
      As[ka][mi] = m0 + mi < M && k0 + ka < K ? Tr<T>::to(s.a[(m0 + mi) * s.sam + (k0 + ka) * s.sak]) : 0.f;
      Bs[kb][ni] = n0 + ni < N && k0 + kb < K ? Tr<T>::to(s.b[(k0 + kb) * s.sbk + (n0 + ni) * s.sbn]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < KT; ++k) {
      float a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = As[k][ty * 4 + i], b[i] = Bs[k][tx * 4 + i];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
    }
    __syncthreads();
  }
}

// Both projections and the activation; with dh the gradients of g and u instead of h.
template <typename T, int ACT, bool BWD>
__global__ void __launch_bounds__(NT) hidden_kernel(const T* x, const T* wg, const T* wu, const T* dh, int64_t rows,
                                                    int dim, int hidden, T* h, T* dg, T* du) {
  __shared__ float As[KT][TILE + 4], Bs[KT][TILE + 4];
  const int64_t m0 = (int64_t)blockIdx.x * TILE, n0 = (int64_t)blockIdx.y * TILE;
  float g[4][4] = {}, u[4][4] = {};
  tile_product<T>({x, wg, dim, 1, 1, dim}, m0, n0, rows, hidden, dim, As, Bs, g);
  tile_product<T>({x, wu, dim, 1, 1, dim}, m0, n0, rows, hidden, dim, As, Bs, u);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
      if (m >= rows || n >= hidden) continue;
      float a, da = 0.f;
      act_eval<ACT, BWD>(g[i][j], a, da);
      if (BWD) {
        const float d = Tr<T>::to(dh[m * hidden + n]);
        dg[m * hidden + n] = Tr<T>::from(d * u[i][j] * da);
        du[m * hidden + n] = Tr<T>::from(d * a);
      } else {
        h[m * hidden + n] = Tr<T>::from(a * u[i][j]);
      }
    }
}

template <typename T>
__global__ void __launch_bounds__(NT) product_kernel(Strided<T> s1, Strided<T> s2, int pairs, int64_t M, int64_t N,
                                                     int64_t K, T* c) {
  __shared__ float As[KT][TILE + 4], Bs[KT][TILE + 4];
  const int64_t m0 = (int64_t)blockIdx.x * TILE, n0 = (int64_t)blockIdx.y * TILE;
  float acc[4][4] = {};
  tile_product<T>(s1, m0, n0, M, N, K, As, Bs, acc);
  if (pairs == 2) tile_product<T>(s2, m0, n0, M, N, K, As, Bs, acc);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
      if (m < M && n < N) c[m * N + n] = Tr<T>::from(acc[i][j]);
    }
}

struct Args {
  const void *x, *wg, *wu, *dh;
  int64_t rows;
  int dim, hidden;
  void *h, *dx, *dwg, *dwu;
  void* ws;
};

static dim3 grid(int64_t M, int64_t N) { return dim3((unsigned)((M + TILE - 1) / TILE), (unsigned)((N + TILE - 1) / TILE)); }

template <typename T, int ACT>
static cudaError_t run(const Args& p, bool bwd, cudaStream_t s) {
  const T *x = (const T*)p.x, *wg = (const T*)p.wg, *wu = (const T*)p.wu;
  T* dg = (T*)p.ws;
  T* du = dg + p.rows * p.hidden;
  const int64_t R = p.rows;
  const int D = p.dim, F = p.hidden;
  if (R > 0 && F > 0) {
    if (bwd)
      hidden_kernel<T, ACT, true><<<grid(R, F), NT, 0, s>>>(x, wg, wu, (const T*)p.dh, R, D, F, nullptr, dg, du);
    else
      hidden_kernel<T, ACT, false><<<grid(R, F), NT, 0, s>>>(x, wg, wu, nullptr, R, D, F, (T*)p.h, nullptr, nullptr);
  }
  if (bwd && D > 0) {
    if (p.dx && R > 0)
      product_kernel<T><<<grid(R, D), NT, 0, s>>>({dg, wg, F, 1, D, 1}, {du, wu, F, 1, D, 1}, 2, R, D, F, (T*)p.dx);
    if (p.dwg && F > 0)
      product_kernel<T><<<grid(F, D), NT, 0, s>>>({dg, x, 1, F, D, 1}, {}, 1, F, D, R, (T*)p.dwg);
    if (p.dwu && F > 0)
      product_kernel<T><<<grid(F, D), NT, 0, s>>>({du, x, 1, F, D, 1}, {}, 1, F, D, R, (T*)p.dwu);
  }
  return cudaGetLastError();
}

template <typename T>
static cudaError_t run_act(int act, const Args& p, bool bwd, cudaStream_t s) {
  switch (act) {
    case FMS_ACT_SILU: return run<T, FMS_ACT_SILU>(p, bwd, s);
    case FMS_ACT_GELU: return run<T, FMS_ACT_GELU>(p, bwd, s);
    case FMS_ACT_GELU_TANH: return run<T, FMS_ACT_GELU_TANH>(p, bwd, s);
    default: return run<T, FMS_ACT_RELU>(p, bwd, s);
  }
}

static int check(int dtype, int act, int64_t rows, int dim, int hidden) {
  if (dtype != FMS_F16 && dtype != FMS_BF16) return FMS_ERR_DTYPE;
  if (act < FMS_ACT_SILU || act > FMS_ACT_RELU) return FMS_ERR_INVALID;
  if (rows < 0 || rows > INT32_MAX || dim < 0 || hidden < 0) return FMS_ERR_INVALID;
  return FMS_OK;
}

static int launch(int dtype, int act, const Args& p, bool bwd, cudaStream_t s) {
  const cudaError_t e = dtype == FMS_F16 ? run_act<__half>(act, p, bwd, s) : run_act<__nv_bfloat16>(act, p, bwd, s);
  return e == cudaSuccess ? FMS_OK : (int)e;
}

}  // namespace glu
}  // namespace fms

using namespace fms;

extern "C" {

size_t fms_gated_ffn_workspace_size(int64_t rows, int dim, int hidden, int backward) {
  if (rows <= 0 || dim < 0 || hidden <= 0) return 0;
  return backward ? (size_t)rows * hidden * 2 * 2 : 0;
}

int fms_gated_ffn_fwd(int dtype, const void* x, const void* w_gate, const void* w_up, int64_t rows, int dim,
                      int hidden, int act, void* h, void* workspace, size_t ws_bytes, fms_stream_t stream) {
  const int st = glu::check(dtype, act, rows, dim, hidden);
  if (st != FMS_OK) return st;
  if (rows == 0 || hidden == 0) return FMS_OK;
  if (!h || (dim > 0 && (!x || !w_gate || !w_up))) return FMS_ERR_INVALID;
  if (ws_bytes < fms_gated_ffn_workspace_size(rows, dim, hidden, 0)) return FMS_ERR_WORKSPACE;
  return glu::launch(dtype, act, {x, w_gate, w_up, nullptr, rows, dim, hidden, h, nullptr, nullptr, nullptr, workspace},
                     false, (cudaStream_t)stream);
}

int fms_gated_ffn_bwd(int dtype, const void* x, const void* w_gate, const void* w_up, const void* dh, int64_t rows,
                      int dim, int hidden, int act, void* dx, void* dw_gate, void* dw_up, void* workspace,
                      size_t ws_bytes, fms_stream_t stream) {
  const int st = glu::check(dtype, act, rows, dim, hidden);
  if (st != FMS_OK) return st;
  if (dim == 0) return FMS_OK;
  if (rows > 0 && hidden > 0 && (!x || !w_gate || !w_up || !dh)) return FMS_ERR_INVALID;
  const size_t need = fms_gated_ffn_workspace_size(rows, dim, hidden, 1);
  if (need && (!workspace || ws_bytes < need)) return FMS_ERR_WORKSPACE;
  return glu::launch(dtype, act, {x, w_gate, w_up, dh, rows, dim, hidden, nullptr, dx, dw_gate, dw_up, workspace},
                     true, (cudaStream_t)stream);
}

}  // extern "C"

// fms_norm.cu -- the norms around a block of a token encoder, with its gate and
// residual scale in the same pass:
//
//   z = scale * x + gate * N(h; w_post, b_post)      (the stream after the block)
//   y = N(z; w_pre, b_pre)                           (the next block's input)
//
// N is the root-mean-square norm v rstd w (+ b), rstd = 1/sqrt(mean(v^2) + eps),
// or the layer norm (v - mean) rstd w (+ b), rstd = 1/sqrt(var + eps).  gate is
// one vector for all rows, one per group of `per` consecutive rows, or absent.
// All statistics and sums are float32; y is the norm of z before z is rounded.
//
// Backward, with hat the normalised values and c(.) the mean over a row:
//   a = dy w_pre;   dz' = dz + rz (a - [c(a)] - zhat c(a zhat))    ([.]: layer)
//   dx = scale dz'
//   e = dz' gate w_post;   dh = rh (e - [c(e)] - hhat c(e hhat))
// and per group of rows the column sums S1 = sum dz' hhat, S0 = sum dz',
// T1 = sum dy zhat, T0 = sum dy, from which every vector's gradient follows:
//   dw_post = sum_g gate S1, db_post = sum_g gate S0, dw_pre = sum T1,
//   db_pre = sum T0, dgate = w_post S1 + b_post S0.
// A group's rows are cut into units; each unit writes its sums, and a second
// kernel adds the units in order, so that results repeat bit for bit.
#include "fms_common.cuh"
#include "fms_internal.h"

namespace fms {
namespace norm {

constexpr int NT = 256;

struct Params {
  const void *x, *h, *dz, *dy;        // rows in T; dz, dy may be NULL (zero)
  const void *w_post, *b_post, *w_pre, *b_pre, *gate;  // vectors in V; biases and gate may be NULL
  void *z, *y, *dx, *dh;              // rows in T
  void *dw_post, *db_post, *dw_pre, *db_pre, *dgate;   // vectors in V, or NULL
  float* stats;                       // (4, rows): mean and rstd of h, mean and rstd of z
  float* part;                        // (4, units, dim)
  int64_t rows, per, groups;          // rows per gate vector, gate vectors
  int64_t units;                      // units of the backward pass
  int segs;                           // units per group (0 without rows)
  int dim;
  float eps, scale;
};

template <typename V>
__device__ __forceinline__ float vec(const void* p, int64_t i, float none) {
  return p ? Tr<V>::to(static_cast<const V*>(p)[i]) : none;
}

// Sum over the block of one or two values, the same on every thread.
__device__ __forceinline__ float2 block_sum2(float2 v) {
  __shared__ float2 part[NT / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  __syncthreads();  // the last call's reads are done
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  float2 t = part[0];
#pragma unroll
  for (int i = 1; i < NT / 32; ++i) t.x += part[i].x, t.y += part[i].y;
  return t;
}

// One row per block.
template <typename T, typename V, bool LAYER>
__global__ void __launch_bounds__(NT) forward_kernel(Params p) {
  const int64_t r = blockIdx.x;
  const int D = p.dim;
  const T* x = static_cast<const T*>(p.x) + r * D;
  const T* h = static_cast<const T*>(p.h) + r * D;
  T* z = static_cast<T*>(p.z) + r * D;
  T* y = static_cast<T*>(p.y) + r * D;
  const int64_t g0 = (r / p.per) * D;
  float mh = 0.f, mz = 0.f, s = 0.f;
  if (LAYER) {
    for (int c = threadIdx.x; c < D; c += NT) s += Tr<T>::to(h[c]);
    mh = block_sum2({s, 0.f}).x / D;
  }
  s = 0.f;
  for (int c = threadIdx.x; c < D; c += NT) {
    const float v = Tr<T>::to(h[c]) - mh;
    s += v * v;
  }
  const float rh = rsqrtf(block_sum2({s, 0.f}).x / D + p.eps);
  auto zval = [&](int c) {
    const float n = (Tr<T>::to(h[c]) - mh) * rh * vec<V>(p.w_post, c, 1.f) + vec<V>(p.b_post, c, 0.f);
    return p.scale * Tr<T>::to(x[c]) + vec<V>(p.gate, g0 + c, 1.f) * n;
  };
  if (LAYER) {
    s = 0.f;
    for (int c = threadIdx.x; c < D; c += NT) s += zval(c);
    mz = block_sum2({s, 0.f}).x / D;
  }
  s = 0.f;
  for (int c = threadIdx.x; c < D; c += NT) {
    const float v = zval(c) - mz;
    s += v * v;
  }
  const float rz = rsqrtf(block_sum2({s, 0.f}).x / D + p.eps);
  for (int c = threadIdx.x; c < D; c += NT) {
    const float v = zval(c);
    z[c] = Tr<T>::from(v);
    y[c] = Tr<T>::from((v - mz) * rz * vec<V>(p.w_pre, c, 1.f) + vec<V>(p.b_pre, c, 0.f));
  }
  if (p.stats && threadIdx.x == 0) {
    p.stats[r] = mh;
    p.stats[p.rows + r] = rh;
    p.stats[2 * p.rows + r] = mz;
    p.stats[3 * p.rows + r] = rz;
  }
}

// One unit (a run of one group's rows) per block; every thread owns the columns
// threadIdx.x + i NT of the unit's sums.
template <typename T, typename V, bool LAYER>
__global__ void __launch_bounds__(NT) backward_kernel(Params p) {
  const int D = p.dim;
  const int64_t group = blockIdx.x / p.segs, seg = blockIdx.x % p.segs;
  const int64_t r0 = group * p.per + p.per * seg / p.segs, r1 = group * p.per + p.per * (seg + 1) / p.segs;
  float* S1 = p.part + (int64_t)blockIdx.x * D;
  float* S0 = S1 + p.units * D;
  float* T1 = S0 + p.units * D;
  float* T0 = T1 + p.units * D;
  for (int c = threadIdx.x; c < D; c += NT) S1[c] = S0[c] = T1[c] = T0[c] = 0.f;
  const int64_t g0 = group * D;
  for (int64_t r = r0; r < r1; ++r) {
    const T* x = static_cast<const T*>(p.x) + r * D;
    const T* h = static_cast<const T*>(p.h) + r * D;
    const float mh = p.stats[r], rh = p.stats[p.rows + r], mz = p.stats[2 * p.rows + r], rz = p.stats[3 * p.rows + r];
    auto hhat = [&](int c) { return (Tr<T>::to(h[c]) - mh) * rh; };
    auto gate = [&](int c) { return vec<V>(p.gate, g0 + c, 1.f); };
    auto zhat = [&](int c) {
      const float n = hhat(c) * vec<V>(p.w_post, c, 1.f) + vec<V>(p.b_post, c, 0.f);
      return (p.scale * Tr<T>::to(x[c]) + gate(c) * n - mz) * rz;
    };
    auto dyv = [&](int c) { return vec<T>(p.dy, r * D + c, 0.f); };
    float2 a = {0.f, 0.f};
    for (int c = threadIdx.x; c < D; c += NT) {
      const float v = dyv(c) * vec<V>(p.w_pre, c, 1.f);
      a.x += v * zhat(c);
      if (LAYER) a.y += v;
    }
    a = block_sum2(a);
    a.x /= D, a.y /= D;
    auto dzt = [&](int c) {
      return vec<T>(p.dz, r * D + c, 0.f) + rz * (dyv(c) * vec<V>(p.w_pre, c, 1.f) - a.y - zhat(c) * a.x);
    };
    float2 b = {0.f, 0.f};
    for (int c = threadIdx.x; c < D; c += NT) {
      const float v = dzt(c) * gate(c) * vec<V>(p.w_post, c, 1.f);
      b.x += v * hhat(c);
      if (LAYER) b.y += v;
    }
    b = block_sum2(b);
    b.x /= D, b.y /= D;
    for (int c = threadIdx.x; c < D; c += NT) {
      const float d = dzt(c), hh = hhat(c);
      static_cast<T*>(p.dx)[r * D + c] = Tr<T>::from(p.scale * d);
      static_cast<T*>(p.dh)[r * D + c] = Tr<T>::from(rh * (d * gate(c) * vec<V>(p.w_post, c, 1.f) - b.y - hh * b.x));
      S1[c] += d * hh;
      S0[c] += d;
      T1[c] += dyv(c) * zhat(c);
      T0[c] += dyv(c);
    }
  }
}

// The vectors' gradients from the units' sums, one column per thread.
template <typename V>
__global__ void __launch_bounds__(NT) finish_kernel(Params p) {
  const int c = blockIdx.x * NT + threadIdx.x;
  if (c >= p.dim) return;
  const int64_t n = p.units * p.dim;
  float w = 0.f, b = 0.f, t1 = 0.f, t0 = 0.f;
  for (int64_t g = 0; g < p.groups; ++g) {
    float s1 = 0.f, s0 = 0.f;
    for (int s = 0; s < p.segs; ++s) {
      const int64_t at = (g * p.segs + s) * p.dim + c;
      s1 += p.part[at];
      s0 += p.part[n + at];
      t1 += p.part[2 * n + at];
      t0 += p.part[3 * n + at];
    }
    const float gt = vec<V>(p.gate, g * p.dim + c, 1.f);
    w += gt * s1;
    b += gt * s0;
    if (p.dgate)
      static_cast<V*>(p.dgate)[g * p.dim + c] =
          Tr<V>::from(vec<V>(p.w_post, c, 1.f) * s1 + vec<V>(p.b_post, c, 0.f) * s0);
  }
  if (p.dw_post) static_cast<V*>(p.dw_post)[c] = Tr<V>::from(w);
  if (p.db_post) static_cast<V*>(p.db_post)[c] = Tr<V>::from(b);
  if (p.dw_pre) static_cast<V*>(p.dw_pre)[c] = Tr<V>::from(t1);
  if (p.db_pre) static_cast<V*>(p.db_pre)[c] = Tr<V>::from(t0);
}

// Units per group: enough for four blocks on every SM, none without a row.
static int segments(int64_t rows, int64_t groups) {
  if (groups <= 0 || rows <= 0) return 1;
  const int64_t per = rows / groups;
  int64_t s = ((int64_t)device_sm_count() * 4 + groups - 1) / groups;
  if (s > per) s = per;
  return s < 1 ? 1 : (int)s;
}

template <typename T, typename V, bool LAYER>
static void run(const Params& p, bool bwd, cudaStream_t s) {
  if (!bwd) {
    forward_kernel<T, V, LAYER><<<(unsigned)p.rows, NT, 0, s>>>(p);
  } else {
    if (p.rows > 0) backward_kernel<T, V, LAYER><<<(unsigned)p.units, NT, 0, s>>>(p);
    finish_kernel<V><<<(p.dim + NT - 1) / NT, NT, 0, s>>>(p);
  }
}

template <typename T, typename V>
static void run_kind(int kind, const Params& p, bool bwd, cudaStream_t s) {
  if (kind == FMS_NORM_LAYER) run<T, V, true>(p, bwd, s);
  else run<T, V, false>(p, bwd, s);
}

static int launch(int dtype, int vdtype, int kind, const Params& p, bool bwd, cudaStream_t s) {
  const bool same = dtype == vdtype;
  if (dtype == FMS_F32) run_kind<float, float>(kind, p, bwd, s);
  else if (dtype == FMS_F16 && same) run_kind<__half, __half>(kind, p, bwd, s);
  else if (dtype == FMS_F16) run_kind<__half, float>(kind, p, bwd, s);
  else if (same) run_kind<__nv_bfloat16, __nv_bfloat16>(kind, p, bwd, s);
  else run_kind<__nv_bfloat16, float>(kind, p, bwd, s);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? FMS_OK : (int)e;
}

static int check(int dtype, int vdtype, int kind, int64_t rows, int64_t groups, int dim, float eps) {
  if (dtype != FMS_F32 && dtype != FMS_F16 && dtype != FMS_BF16) return FMS_ERR_DTYPE;
  if (vdtype != dtype && vdtype != FMS_F32) return FMS_ERR_DTYPE;
  if (kind != FMS_NORM_RMS && kind != FMS_NORM_LAYER) return FMS_ERR_INVALID;
  if (rows < 0 || rows > INT32_MAX || dim < 1 || groups < 0 || !(eps >= 0.f)) return FMS_ERR_INVALID;
  if (groups > 0 ? rows % groups != 0 : rows > 0) return FMS_ERR_INVALID;
  return FMS_OK;
}

}  // namespace norm
}  // namespace fms

using namespace fms;

extern "C" {

int fms_norm_residual_fwd(int dtype, int vdtype, int kind, const void* x, const void* h, const void* w_post,
                          const void* b_post, const void* w_pre, const void* b_pre, const void* gate, int64_t groups,
                          int64_t rows, int dim, float eps, float scale, void* z, void* y, float* stats,
                          fms_stream_t stream) {
  const int st = norm::check(dtype, vdtype, kind, rows, groups, dim, eps);
  if (st != FMS_OK) return st;
  if (rows == 0) return FMS_OK;
  if (!x || !h || !w_post || !w_pre || !z || !y) return FMS_ERR_INVALID;
  norm::Params p{};
  p.x = x; p.h = h; p.w_post = w_post; p.b_post = b_post; p.w_pre = w_pre; p.b_pre = b_pre; p.gate = gate;
  p.z = z; p.y = y; p.stats = stats;
  p.rows = rows; p.per = rows / groups; p.dim = dim; p.eps = eps; p.scale = scale;
  return norm::launch(dtype, vdtype, kind, p, false, (cudaStream_t)stream);
}

size_t fms_norm_residual_bwd_workspace_size(int64_t rows, int64_t groups, int dim) {
  if (rows <= 0 || groups <= 0 || dim <= 0) return 0;
  return (size_t)4 * groups * norm::segments(rows, groups) * dim * sizeof(float);
}

int fms_norm_residual_bwd(int dtype, int vdtype, int kind, const void* x, const void* h, const void* w_post,
                          const void* b_post, const void* w_pre, const void* gate, int64_t groups, int64_t rows,
                          int dim, float scale, const float* stats, const void* dz, const void* dy, void* dx, void* dh,
                          void* dw_post, void* db_post, void* dw_pre, void* db_pre, void* dgate, void* workspace,
                          size_t ws_bytes, fms_stream_t stream) {
  const int st = norm::check(dtype, vdtype, kind, rows, groups, dim, 0.f);
  if (st != FMS_OK) return st;
  if (!w_post || !w_pre) return FMS_ERR_INVALID;
  if (rows > 0 && (!x || !h || !stats || !dx || !dh)) return FMS_ERR_INVALID;
  const size_t need = fms_norm_residual_bwd_workspace_size(rows, groups, dim);
  if (need && (!workspace || ws_bytes < need)) return FMS_ERR_WORKSPACE;
  norm::Params p{};
  p.x = x; p.h = h; p.w_post = w_post; p.b_post = b_post; p.w_pre = w_pre; p.gate = gate;
  p.dz = dz; p.dy = dy; p.dx = dx; p.dh = dh;
  p.dw_post = dw_post; p.db_post = db_post; p.dw_pre = dw_pre; p.db_pre = db_pre; p.dgate = dgate;
  p.stats = const_cast<float*>(stats); p.part = (float*)workspace;
  p.rows = rows; p.dim = dim; p.scale = scale;
  p.groups = groups;
  p.segs = rows > 0 ? norm::segments(rows, groups) : 0;
  p.units = groups * p.segs;
  p.per = groups > 0 ? rows / groups : 1;
  return norm::launch(dtype, vdtype, kind, p, true, (cudaStream_t)stream);
}

}  // extern "C"

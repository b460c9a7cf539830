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
// A group's rows are cut into units, one block each; a unit writes its sums, and a
// second kernel adds the units in order, so that results repeat bit for bit.
//
// All of it is bound by memory: a row is read once into registers (forward x and h,
// backward x, h, dz and dy) and written once; nothing else but the statistics and the
// units' sums goes out.
#include "fms_common.cuh"
#include "fms_internal.h"

namespace fms {
namespace norm {

struct Params {
  const void *x, *h, *dz, *dy;        // rows in T; dz, dy may be NULL (zero)
  const void *w_post, *b_post, *w_pre, *b_pre, *gate;  // vectors in vdt; biases and gate may be NULL
  void *z, *y, *dx, *dh;              // rows in T
  void *dw_post, *db_post, *dw_pre, *db_pre, *dgate;   // vectors in vdt, or NULL
  float* stats;                       // (4, rows): mean and rstd of h, mean and rstd of z
  float* part;                        // (4, units, dim): S1, T1, S0, T0
  int64_t rows, per, groups;          // rows per gate vector, gate vectors
  int64_t units;                      // units of the backward pass
  int segs;                           // units per group (0 without rows)
  int dim, vdt, layer;
  float eps, scale;
};

// VEC neighbouring values as float32: one 16-byte access, or one value (rows that do not
// start on 16 bytes).
template <typename T, int VEC>
__device__ __forceinline__ void load(const T* p, float (&f)[VEC]) {
  if constexpr (VEC == 1) {
    f[0] = Tr<T>::to(*p);
  } else {
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 4) {
        f[j] = __uint_as_float(w[j]);
      } else {
        const T* t = reinterpret_cast<const T*>(&w[j]);
        f[2 * j] = Tr<T>::to(t[0]);
        f[2 * j + 1] = Tr<T>::to(t[1]);
      }
    }
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void store(T* p, const float (&f)[VEC]) {
  if constexpr (VEC == 1) {
    *p = Tr<T>::from(f[0]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 4) {
        w[j] = __float_as_uint(f[j]);
      } else {
        T t[2] = {Tr<T>::from(f[2 * j]), Tr<T>::from(f[2 * j + 1])};
        w[j] = *reinterpret_cast<const uint32_t*>(t);
      }
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
// The same of a weight, bias or gate (in T or float32); `none` where there is none.
template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const void* p, int vdt, int64_t at, float none, float (&f)[VEC]) {
  if (p == nullptr) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[j] = none;
  } else if (vdt == FMS_F32) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[j] = __ldg(static_cast<const float*>(p) + at + j);
  } else {
    load<T, VEC>(static_cast<const T*>(p) + at, f);
  }
}
__device__ __forceinline__ float vec1(const void* p, int vdt, int64_t i, float none) {
  if (p == nullptr) return none;
  return vdt == FMS_F32   ? static_cast<const float*>(p)[i]
         : vdt == FMS_F16 ? __half2float(static_cast<const __half*>(p)[i])
                          : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void put1(void* p, int vdt, int64_t i, float v) {
  if (p == nullptr) return;
  if (vdt == FMS_F32) static_cast<float*>(p)[i] = v;
  else if (vdt == FMS_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

constexpr int MAX_WARPS = 32;

// Sums of two values over the threads of a row, the same on each of them: a warp, or
// the whole block (one barrier: the partial sums alternate between two places).
template <bool WARP>
struct RowSum {
  float2 (*part)[MAX_WARPS];
  int turn = 0;
  __device__ __forceinline__ float2 operator()(float2 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
      v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    if (WARP) return v;
    if ((threadIdx.x & 31) == 0) part[turn][threadIdx.x >> 5] = v;
    __syncthreads();
    const int n = blockDim.x >> 5;
    float2 t = part[turn][0];
    for (int i = 1; i < n; ++i) t.x += part[turn][i].x, t.y += part[turn][i].y;
    turn ^= 1;
    return t;
  }
};

// One row per warp (WARP) or block; a thread holds NV runs of VEC values.  A warp takes
// rows of up to 4 runs per lane (no barriers between the row's sums), a block the wider
// ones.
template <typename T, int VEC, int NV, bool WARP>
__global__ void __launch_bounds__(WARP ? 128 : 1024) forward_kernel(Params p) {
  __shared__ float2 part[2][MAX_WARPS];
  RowSum<WARP> sum{part};
  const int64_t r = WARP ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
  if (WARP && r >= p.rows) return;
  const int tid = WARP ? threadIdx.x & 31 : threadIdx.x, tpr = WARP ? 32 : blockDim.x;
  const int D = p.dim;
  const float inv_d = 1.f / D;
  const T* x = static_cast<const T*>(p.x) + r * D;
  const T* h = static_cast<const T*>(p.h) + r * D;
  const int64_t g0 = (r / p.per) * D;
  float z[NV][VEC], v[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * tpr + tid) * VEC;
#pragma unroll
    for (int j = 0; j < VEC; ++j) z[i][j] = v[i][j] = 0.f;
    if (c < D) {
      load<T, VEC>(h + c, v[i]);
      load<T, VEC>(x + c, z[i]);
    }
  }
  // mean, and the reciprocal deviation of the centred values (two passes over registers)
  auto stats = [&](float (&a)[NV][VEC], float& mean, float& rstd) {
    mean = 0.f;
    if (p.layer) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) s += a[i][j];
      mean = sum({s, 0.f}).x * inv_d;
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float d = (i * tpr + tid) * VEC < D ? a[i][j] - mean : 0.f;
        s += d * d;
      }
    rstd = rsqrtf(sum({s, 0.f}).x * inv_d + p.eps);
  };
  float mh, rh, mz, rz;
  stats(v, mh, rh);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * tpr + tid) * VEC;
    if (c >= D) continue;
    float w[VEC], b[VEC], g[VEC];
    load_vec<T, VEC>(p.w_post, p.vdt, c, 1.f, w);
    load_vec<T, VEC>(p.b_post, p.vdt, c, 0.f, b);
    load_vec<T, VEC>(p.gate, p.vdt, g0 + c, 1.f, g);
#pragma unroll
    for (int j = 0; j < VEC; ++j) z[i][j] = p.scale * z[i][j] + g[j] * ((v[i][j] - mh) * rh * w[j] + b[j]);
    store<T, VEC>(static_cast<T*>(p.z) + r * D + c, z[i]);
  }
  stats(z, mz, rz);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * tpr + tid) * VEC;
    if (c >= D) continue;
    float w[VEC], b[VEC];
    load_vec<T, VEC>(p.w_pre, p.vdt, c, 1.f, w);
    load_vec<T, VEC>(p.b_pre, p.vdt, c, 0.f, b);
#pragma unroll
    for (int j = 0; j < VEC; ++j) z[i][j] = (z[i][j] - mz) * rz * w[j] + b[j];
    store<T, VEC>(static_cast<T*>(p.y) + r * D + c, z[i]);
  }
  if (p.stats && tid == 0) {
    p.stats[r] = mh;
    p.stats[p.rows + r] = rh;
    p.stats[2 * p.rows + r] = mz;
    p.stats[3 * p.rows + r] = rz;
  }
}

// One unit (a run of one group's rows) per block, a row at a time; a thread owns the
// same NV runs of VEC columns in every row and keeps their sums in registers.  BIAS:
// S0 and T0 are wanted too.
template <typename T, int VEC, int NV, bool BIAS>
__global__ void __launch_bounds__(512) backward_kernel(Params p) {
  __shared__ float2 part[2][MAX_WARPS];
  RowSum<false> sum{part};
  const int D = p.dim;
  const float inv_d = 1.f / D;
  const int64_t group = blockIdx.x / p.segs, seg = blockIdx.x % p.segs;
  const int64_t r0 = group * p.per + p.per * seg / p.segs, r1 = group * p.per + p.per * (seg + 1) / p.segs;
  float gw[NV][VEC], gb[NV][VEC], wp[NV][VEC];  // gate w_post, gate b_post, w_pre
  float S1[NV][VEC], T1[NV][VEC], S0[NV][VEC], T0[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * blockDim.x + threadIdx.x) * VEC;
    float g[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      S1[i][j] = T1[i][j] = S0[i][j] = T0[i][j] = 0.f;
      gw[i][j] = gb[i][j] = wp[i][j] = g[j] = 0.f;
    }
    if (c >= D) continue;
    load_vec<T, VEC>(p.gate, p.vdt, group * D + c, 1.f, g);
    load_vec<T, VEC>(p.w_post, p.vdt, c, 1.f, gw[i]);
    if (BIAS) load_vec<T, VEC>(p.b_post, p.vdt, c, 0.f, gb[i]);
    load_vec<T, VEC>(p.w_pre, p.vdt, c, 1.f, wp[i]);
#pragma unroll
    for (int j = 0; j < VEC; ++j) gw[i][j] *= g[j], gb[i][j] *= g[j];
  }
  for (int64_t r = r0; r < r1; ++r) {
    const float mh = p.stats[r], rh = p.stats[p.rows + r], mz = p.stats[2 * p.rows + r], rz = p.stats[3 * p.rows + r];
    float hh[NV][VEC], zh[NV][VEC], dy[NV][VEC], d[NV][VEC];
    float2 a = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * blockDim.x + threadIdx.x) * VEC;
      const int64_t at = r * D + c;
#pragma unroll
      for (int j = 0; j < VEC; ++j) hh[i][j] = zh[i][j] = dy[i][j] = d[i][j] = 0.f;
      if (c >= D) continue;
      load<T, VEC>(static_cast<const T*>(p.x) + at, zh[i]);
      load<T, VEC>(static_cast<const T*>(p.h) + at, hh[i]);
      if (p.dy) load<T, VEC>(static_cast<const T*>(p.dy) + at, dy[i]);
      if (p.dz) load<T, VEC>(static_cast<const T*>(p.dz) + at, d[i]);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if ((i * (int)blockDim.x + (int)threadIdx.x) * VEC >= D) continue;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        hh[i][j] = (hh[i][j] - mh) * rh;
        zh[i][j] = (p.scale * zh[i][j] + (hh[i][j] * gw[i][j] + gb[i][j]) - mz) * rz;
        const float t = dy[i][j] * wp[i][j];
        a.x += t * zh[i][j];
        a.y += t;
      }
    }
    a = sum(a);
    a.x *= inv_d;
    a.y = p.layer ? a.y * inv_d : 0.f;
    float2 b = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        d[i][j] += rz * (dy[i][j] * wp[i][j] - a.y - zh[i][j] * a.x);
        const float e = d[i][j] * gw[i][j];  // 0 past the row's end
        b.x += e * hh[i][j];
        b.y += e;
      }
    b = sum(b);
    b.x *= inv_d;
    b.y = p.layer ? b.y * inv_d : 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * blockDim.x + threadIdx.x) * VEC;
      if (c >= D) continue;
      const int64_t at = r * D + c;
      float o[VEC], q[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        o[j] = p.scale * d[i][j];
        q[j] = rh * (d[i][j] * gw[i][j] - b.y - hh[i][j] * b.x);
        S1[i][j] += d[i][j] * hh[i][j];
        T1[i][j] += dy[i][j] * zh[i][j];
        if (BIAS) S0[i][j] += d[i][j], T0[i][j] += dy[i][j];
      }
      store<T, VEC>(static_cast<T*>(p.dx) + at, o);
      store<T, VEC>(static_cast<T*>(p.dh) + at, q);
    }
  }
  const int64_t n = p.units * D;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * blockDim.x + threadIdx.x) * VEC;
    if (c >= D) continue;
    float* o = p.part + (int64_t)blockIdx.x * D + c;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      o[j] = S1[i][j];
      o[n + j] = T1[i][j];
      if (BIAS) o[2 * n + j] = S0[i][j], o[3 * n + j] = T0[i][j];
    }
  }
}

// The vectors' gradients from the units' sums: 32 columns per block, its 32 warps take
// the groups in turn and are added in order.
template <bool BIAS>
__global__ void __launch_bounds__(1024) finish_kernel(Params p) {
  __shared__ float acc[4][32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  const int64_t n = p.units * p.dim;
  float w = 0.f, b = 0.f, t1 = 0.f, t0 = 0.f;
  if (c < p.dim) {
    // without a gate per group the units are one run, shared by all warps
    const int64_t runs = p.groups > 1 ? p.groups : p.segs;
    const int segs = p.groups > 1 ? p.segs : 1;
    for (int64_t g = warp; g < runs; g += 32) {
      float s1 = 0.f, s0 = 0.f;
      for (int s = 0; s < segs; ++s) {
        const float* q = p.part + (g * segs + s) * p.dim + c;
        s1 += q[0];
        t1 += q[n];
        if (BIAS) s0 += q[2 * n], t0 += q[3 * n];
      }
      if (p.groups > 1) {
        const float gt = vec1(p.gate, p.vdt, g * p.dim + c, 1.f);
        w += gt * s1;
        b += gt * s0;
        put1(p.dgate, p.vdt, g * p.dim + c,
             vec1(p.w_post, p.vdt, c, 1.f) * s1 + vec1(p.b_post, p.vdt, c, 0.f) * s0);
      } else {
        w += s1;
        b += s0;
      }
    }
  }
  acc[0][warp][lane] = w;
  acc[1][warp][lane] = b;
  acc[2][warp][lane] = t1;
  acc[3][warp][lane] = t0;
  __syncthreads();
  if (warp != 0 || c >= p.dim) return;
  w = b = t1 = t0 = 0.f;
  for (int i = 0; i < 32; ++i) {
    w += acc[0][i][lane];
    b += acc[1][i][lane];
    t1 += acc[2][i][lane];
    t0 += acc[3][i][lane];
  }
  if (p.groups <= 1) {
    if (p.groups == 1) put1(p.dgate, p.vdt, c, vec1(p.w_post, p.vdt, c, 1.f) * w + vec1(p.b_post, p.vdt, c, 0.f) * b);
    const float gt = p.groups == 1 ? vec1(p.gate, p.vdt, c, 1.f) : 1.f;
    w *= gt;
    b *= gt;
  }
  put1(p.dw_post, p.vdt, c, w);
  put1(p.db_post, p.vdt, c, b);
  put1(p.dw_pre, p.vdt, c, t1);
  put1(p.db_pre, p.vdt, c, t0);
}

// Units per group: about `target` units in all, none without a row.
static int segments(int64_t rows, int64_t groups) {
  if (groups <= 0 || rows <= 0) return 1;
  const int64_t per = rows / groups;
  int64_t s = ((int64_t)device_sm_count() * 6 + groups - 1) / groups;
  if (s > per) s = per;
  return s < 1 ? 1 : (int)s;
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T, int VEC, int NV, bool WARP>
static void forward(const Params& p, cudaStream_t s) {
  if (WARP) {
    forward_kernel<T, VEC, NV, true><<<(unsigned)((p.rows + 3) / 4), 128, 0, s>>>(p);
  } else {
    const int tpr = ((p.dim + VEC * NV - 1) / (VEC * NV) + 31) / 32 * 32;
    forward_kernel<T, VEC, NV, false><<<(unsigned)p.rows, tpr, 0, s>>>(p);
  }
}

template <typename T, int VEC>
static void run_forward(const Params& p, cudaStream_t s) {
  constexpr int W = 32 * VEC;  // a warp's columns per run
  if (p.dim <= W) forward<T, VEC, 1, true>(p, s);
  else if (p.dim <= 2 * W) forward<T, VEC, 2, true>(p, s);
  else if (p.dim <= 3 * W) forward<T, VEC, 3, true>(p, s);
  else if (p.dim <= 4 * W) forward<T, VEC, 4, true>(p, s);
  else if (VEC > 1 && p.dim <= 1024 * VEC) forward<T, VEC, 1, false>(p, s);
  else if (p.dim <= 4096 * VEC) forward<T, VEC, 4, false>(p, s);
  else forward<T, VEC, 16, false>(p, s);
}

template <typename T, int VEC, int NV, bool BIAS>
static void backward(const Params& p, cudaStream_t s) {
  const int tpr = ((p.dim + VEC * NV - 1) / (VEC * NV) + 31) / 32 * 32;
  backward_kernel<T, VEC, NV, BIAS><<<(unsigned)p.units, tpr, 0, s>>>(p);
}

template <typename T, int VEC, bool BIAS>
static void run_backward(const Params& p, cudaStream_t s) {
  if (VEC > 1) {
    if (p.dim <= 512 * VEC) backward<T, VEC, 1, BIAS>(p, s);
    else if (p.dim <= 1024 * VEC) backward<T, VEC, 2, BIAS>(p, s);
    else backward<T, VEC, VEC == 8 ? 4 : 8, BIAS>(p, s);
  } else {
    if (p.dim <= 256) backward<T, VEC, 1, BIAS>(p, s);
    else if (p.dim <= 2048) backward<T, VEC, 4, BIAS>(p, s);
    else backward<T, VEC, 32, BIAS>(p, s);
  }
}

template <typename T>
static void run(const Params& p, bool bwd, cudaStream_t s) {
  constexpr int VEC = 16 / sizeof(T);
  const bool vec = p.dim % VEC == 0 && aligned16(p.x) && aligned16(p.h) && aligned16(p.w_post) && aligned16(p.b_post) &&
                   aligned16(p.w_pre) && aligned16(p.b_pre) && aligned16(p.gate) &&
                   (bwd ? aligned16(p.dz) && aligned16(p.dy) && aligned16(p.dx) && aligned16(p.dh)
                        : aligned16(p.z) && aligned16(p.y));
  if (!bwd) {
    if (vec) run_forward<T, VEC>(p, s);
    else run_forward<T, 1>(p, s);
    return;
  }
  const bool bias = p.b_post || p.db_post || p.db_pre;
  if (p.rows > 0) {
    if (vec && bias) run_backward<T, VEC, true>(p, s);
    else if (vec) run_backward<T, VEC, false>(p, s);
    else if (bias) run_backward<T, 1, true>(p, s);
    else run_backward<T, 1, false>(p, s);
  }
  const unsigned blocks = (unsigned)((p.dim + 31) / 32);
  if (bias) finish_kernel<true><<<blocks, 1024, 0, s>>>(p);
  else finish_kernel<false><<<blocks, 1024, 0, s>>>(p);
}

static int launch(int dtype, const Params& p, bool bwd, cudaStream_t s) {
  if (dtype == FMS_F32) run<float>(p, bwd, s);
  else if (dtype == FMS_F16) run<__half>(p, bwd, s);
  else run<__nv_bfloat16>(p, bwd, s);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? FMS_OK : (int)e;
}

static int check(int dtype, int vdtype, int kind, int64_t rows, int64_t groups, int dim, float eps) {
  if (dtype != FMS_F32 && dtype != FMS_F16 && dtype != FMS_BF16) return FMS_ERR_DTYPE;
  if (vdtype != dtype && vdtype != FMS_F32) return FMS_ERR_DTYPE;
  if (kind != FMS_NORM_RMS && kind != FMS_NORM_LAYER) return FMS_ERR_INVALID;
  if (rows < 0 || rows > INT32_MAX || dim < 1 || groups < 0 || !(eps >= 0.f)) return FMS_ERR_INVALID;
  if (dim > FMS_NORM_MAX_DIM) return FMS_ERR_TOO_LARGE;
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
  p.vdt = vdtype; p.layer = kind == FMS_NORM_LAYER;
  return norm::launch(dtype, p, false, (cudaStream_t)stream);
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
  p.vdt = vdtype; p.layer = kind == FMS_NORM_LAYER;
  return norm::launch(dtype, p, true, (cudaStream_t)stream);
}

}  // extern "C"

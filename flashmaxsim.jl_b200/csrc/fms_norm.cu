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
// Each block takes an equal run of the rows, whatever groups they belong to, and writes
// S for every group that it meets and T once; two small kernels add these in order, so
// that results repeat bit for bit.
//
// All of it is bound by memory: a row is read once (forward x and h, backward x, h, dz
// and dy) and written once; nothing else but the statistics and the blocks' sums goes out.
// What stands in the way is the number of instructions: a row of 768 leaves an SM 270
// (forward) and 400 (backward) cycles of memory time.  So the arithmetic is in pairs
// (f32x2), and rows are read straight into registers: a ring of bulk copies was slower
// (forward 112 us against 103 at 46080 x 768, the thread that issues them holds up its
// row).
#include "fms_common.cuh"
#include "fms_internal.h"
#include "fms_launch.cuh"

#include <type_traits>

namespace fms {
namespace norm {

struct Params {
  const void *x, *h, *dz, *dy;        // rows in T; dz, dy may be NULL (zero)
  const void *w_post, *b_post, *w_pre, *b_pre, *gate;  // vectors in vdt; biases and gate may be NULL
  void *z, *y, *dx, *dh;              // rows in T
  void *dw_post, *db_post, *dw_pre, *db_pre, *dgate;   // vectors in vdt, or NULL
  float* stats;                       // (4, rows): mean and rstd of h, mean and rstd of z
  float* part;                        // S1, S0: (blocks + groups, dim); T1, T0: (blocks, dim)
  int64_t rows, per, groups;          // rows per gate vector, gate vectors
  int64_t blocks;                     // of the backward pass (0 without rows)
  int dim, vdt, layer;
  float eps, scale;
};

// A thread's values of a row: N pairs, in runs of VEC neighbours (one 16-byte access
// each; VEC 1 for rows that do not start on 16 bytes), run i at (i * tpr + tid) * VEC.
// `raw` holds them as they lie in memory.
template <typename T, int VEC, int N>
struct Raw {
  static constexpr int RUNS = 2 * N / VEC;
  using Word = typename std::conditional<VEC == 1, T, uint4>::type;
  Word w[RUNS];
  __device__ __forceinline__ void load(const T* row, int tid, int tpr, int D) {
#pragma unroll
    for (int i = 0; i < RUNS; ++i) {
      const int c = (i * tpr + tid) * VEC;
      if constexpr (VEC == 1) w[i] = c < D ? row[c] : Tr<T>::from(0.f);
      else w[i] = c < D ? *reinterpret_cast<const uint4*>(row + c) : make_uint4(0, 0, 0, 0);
    }
  }
  __device__ __forceinline__ void get(float2 (&f)[N]) const {
    if constexpr (VEC == 1) {
#pragma unroll
      for (int k = 0; k < N; ++k) f[k] = make_float2(Tr<T>::to(w[2 * k]), Tr<T>::to(w[2 * k + 1]));
    } else {
#pragma unroll
      for (int i = 0; i < RUNS; ++i) {
        const uint32_t q[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
        for (int k = 0; k < VEC / 2; ++k) f[i * (VEC / 2) + k] = pair(q, k);
      }
    }
  }
  static __device__ __forceinline__ float2 pair(const uint32_t (&q)[4], int k) {
    if constexpr (sizeof(T) == 4) {
      return make_float2(__uint_as_float(q[2 * (k & 1)]), __uint_as_float(q[2 * (k & 1) + 1]));
    } else if constexpr (std::is_same<T, __half>::value) {
      return __half22float2(*reinterpret_cast<const __half2*>(&q[k]));
    } else {
      return make_float2(__uint_as_float(q[k] << 16), __uint_as_float(q[k] & 0xffff0000u));
    }
  }
};

// The pairs of one run written to a row.
template <typename T, int VEC, int N>
__device__ __forceinline__ void store(T* row, int tid, int tpr, int D, const float2 (&f)[N]) {
#pragma unroll
  for (int i = 0; i < 2 * N / VEC; ++i) {
    const int c = (i * tpr + tid) * VEC;
    if (c >= D) continue;
    if constexpr (VEC == 1) {
      row[c] = Tr<T>::from(i & 1 ? f[i >> 1].y : f[i >> 1].x);
    } else {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 4) {
          w[j] = __float_as_uint(j & 1 ? f[i * 2 + (j >> 1)].y : f[i * 2 + (j >> 1)].x);
        } else {
          const float2 v = f[i * 4 + j];
          if constexpr (std::is_same<T, __half>::value) {
            const __half2 h = __floats2half2_rn(v.x, v.y);
            w[j] = *reinterpret_cast<const uint32_t*>(&h);
          } else {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
            w[j] = *reinterpret_cast<const uint32_t*>(&h);
          }
        }
      }
      *reinterpret_cast<uint4*>(row + c) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// The same of a weight, bias or gate (in T or float32) from element `at` on.  WIDE: it
// starts on 16 bytes where it is in T.  (Only its own loads depend on that: how a row is
// read, and so what it adds up to, must not.)
template <bool WIDE, typename T, int VEC, int N>
__device__ __forceinline__ void load_vec(const void* p, int vdt, int64_t at, int tid, int tpr, int D, float2 (&f)[N]) {
  if (WIDE && (sizeof(T) == 4 || vdt != FMS_F32)) {
    Raw<T, VEC, N> r;
    r.load(static_cast<const T*>(p) + at, tid, tpr, D);
    r.get(f);
  } else {
    const float* q = static_cast<const float*>(p) + at;
    const T* u = static_cast<const T*>(p) + at;
#pragma unroll
    for (int e = 0; e < 2 * N; ++e) {
      const int c = (e / VEC * tpr + tid) * VEC + e % VEC;
      const float v = c >= D ? 0.f : WIDE || vdt == FMS_F32 ? q[c] : Tr<T>::to(u[c]);
      if (e & 1) f[e >> 1].y = v;
      else f[e >> 1].x = v;
    }
  }
}
__device__ __forceinline__ float2 two(float v) { return make_float2(v, v); }
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

// Sums of N values over the threads of a row, the same on each of them: a warp, or the
// whole block (one barrier: the partial sums alternate between two places).
template <bool WARP, int N>
struct RowSum {
  float (*part)[MAX_WARPS * N];
  int turn = 0;
  __device__ __forceinline__ void operator()(float (&v)[N]) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    if (WARP) return;
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int k = 0; k < N; ++k) part[turn][(threadIdx.x >> 5) * N + k] = v[k];
    }
    __syncthreads();
    const int n = blockDim.x >> 5;
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = part[turn][k];
    for (int i = 1; i < n; ++i)
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] += part[turn][i * N + k];
    turn ^= 1;
  }
};

// One row per warp (WARP, rows of up to 1024) or block; a thread holds N pairs.
template <typename T, int VEC, int N, bool WIDE, bool WARP>
__global__ void __launch_bounds__(WARP ? 128 : 1024) forward_kernel(Params p) {
  __shared__ float part[2][MAX_WARPS];
  RowSum<WARP, 1> sum{part};
  const int64_t r = WARP ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
  dependency_wait();
  if (WARP && r >= p.rows) return;
  const int tid = WARP ? threadIdx.x & 31 : threadIdx.x, tpr = WARP ? 32 : blockDim.x;
  const int D = p.dim;
  const float inv_d = 1.f / D;
  float2 z[N], v[N], w[N];
  {
    Raw<T, VEC, N> h, x;
    h.load(static_cast<const T*>(p.h) + r * D, tid, tpr, D);
    x.load(static_cast<const T*>(p.x) + r * D, tid, tpr, D);
    h.get(v);
    x.get(z);
  }
  // Takes the mean off the values and gives it and their reciprocal deviation (two passes
  // over registers).  The mean comes off before that factor goes on, and is the quotient
  // that rounds right, so that a row of one value is zero whatever 1 / sqrt(eps) multiplies
  // it by; the values past the row's end are no zeros afterwards.
  auto centre = [&](float2 (&a)[N], float& mean, float& rstd) {
    float s[1];
    mean = 0.f;
    if (p.layer) {
      float2 t = a[0];
#pragma unroll
      for (int k = 1; k < N; ++k) t = __fadd2_rn(t, a[k]);
      s[0] = t.x + t.y;
      sum(s);
      mean = s[0] * inv_d;
      mean = fmaf(fmaf(-mean, (float)D, s[0]), inv_d, mean);  // the quotient, by its remainder
#pragma unroll
      for (int k = 0; k < N; ++k) a[k] = __fadd2_rn(a[k], two(-mean));
    }
    float2 t = two(0.f);
#pragma unroll
    for (int i = 0; i < 2 * N / VEC; ++i)
      if ((i * tpr + tid) * VEC < D) {
        if constexpr (VEC == 1) {
          const float d = i & 1 ? a[i >> 1].y : a[i >> 1].x;
          t.x = fmaf(d, d, t.x);
        } else {
#pragma unroll
          for (int k = 0; k < VEC / 2; ++k) t = __ffma2_rn(a[i * (VEC / 2) + k], a[i * (VEC / 2) + k], t);
        }
      }
    s[0] = t.x + t.y;
    sum(s);
    rstd = rsqrtf(s[0] * inv_d + p.eps);
  };
  // a = a rstd w + b
  auto apply = [&](float2 (&a)[N], float rstd, const void* wv, const void* bv) {
    load_vec<WIDE, T, VEC, N>(wv, p.vdt, 0, tid, tpr, D, w);
#pragma unroll
    for (int k = 0; k < N; ++k) a[k] = __fmul2_rn(__fmul2_rn(a[k], two(rstd)), w[k]);
    if (bv) {
      load_vec<WIDE, T, VEC, N>(bv, p.vdt, 0, tid, tpr, D, w);
#pragma unroll
      for (int k = 0; k < N; ++k) a[k] = __fadd2_rn(a[k], w[k]);
    }
  };
  float mh, rh, mz, rz;
  centre(v, mh, rh);
  apply(v, rh, p.w_post, p.b_post);
  if (p.gate) {
    load_vec<WIDE, T, VEC, N>(p.gate, p.vdt, (r / p.per) * D, tid, tpr, D, w);
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = __fmul2_rn(v[k], w[k]);
  }
#pragma unroll
  for (int k = 0; k < N; ++k) z[k] = __ffma2_rn(z[k], two(p.scale), v[k]);
  store<T, VEC, N>(static_cast<T*>(p.z) + r * D, tid, tpr, D, z);
  centre(z, mz, rz);
  apply(z, rz, p.w_pre, p.b_pre);
  store<T, VEC, N>(static_cast<T*>(p.y) + r * D, tid, tpr, D, z);
  if (p.stats && tid == 0) {
    p.stats[r] = mh;
    p.stats[p.rows + r] = rh;
    p.stats[2 * p.rows + r] = mz;
    p.stats[3 * p.rows + r] = rz;
  }
}

// Block k's rows start at rows k / blocks; the block that holds row r.
__device__ __forceinline__ int64_t block_of(const Params& p, int64_t r) { return ((r + 1) * p.blocks - 1) / p.rows; }

template <int VEC, int N>
__device__ __forceinline__ void put_sums(float* o, int tid, int tpr, int D, const float2 (&f)[N]) {
#pragma unroll
  for (int e = 0; e < 2 * N; ++e) {
    const int c = (e / VEC * tpr + tid) * VEC + e % VEC;
    if (c < D) o[c] = e & 1 ? f[e >> 1].y : f[e >> 1].x;
  }
}

// A run of rows per block, a row at a time with the next one's loads in flight; a thread
// owns the same N pairs of columns in every row and keeps their sums in registers.
// BIAS: S0 and T0 are wanted too.  One block an SM is asked for by name: left to itself
// the compiler gave the widest rows 32 or 64 registers a thread and spilled the rest
// (11520 x 5120 bf16 layer 1320 us, 513 with 128 registers).
template <typename T, int VEC, int N, bool WIDE, bool BIAS>
__global__ void __launch_bounds__(512, 1) backward_kernel(Params p) {
  __shared__ float part[2][MAX_WARPS * 2];
  RowSum<false, 2> sum{part};
  dependency_wait();
  const int D = p.dim, tid = threadIdx.x, tpr = blockDim.x;
  const float inv_d = 1.f / D;
  const int64_t r0 = p.rows * blockIdx.x / p.blocks, r1 = p.rows * (blockIdx.x + 1) / p.blocks;
  float* const outS = p.part;
  float* const outT = p.part + 2 * (p.blocks + p.groups) * D;
  float2 gw[N], gb[N], wp[N];  // gate w_post, gate b_post, w_pre
  float2 S1[N], T1[N], S0[N], T0[N];
  load_vec<WIDE, T, VEC, N>(p.w_pre, p.vdt, 0, tid, tpr, D, wp);
#pragma unroll
  for (int k = 0; k < N; ++k) S1[k] = T1[k] = S0[k] = T0[k] = gb[k] = two(0.f);
  int64_t group = r0 / p.per;
  auto enter = [&]() {
    load_vec<WIDE, T, VEC, N>(p.w_post, p.vdt, 0, tid, tpr, D, gw);
    if (BIAS && p.b_post) load_vec<WIDE, T, VEC, N>(p.b_post, p.vdt, 0, tid, tpr, D, gb);
    if (p.gate) {
      float2 g[N];
      load_vec<WIDE, T, VEC, N>(p.gate, p.vdt, group * D, tid, tpr, D, g);
#pragma unroll
      for (int k = 0; k < N; ++k) gw[k] = __fmul2_rn(gw[k], g[k]), gb[k] = __fmul2_rn(gb[k], g[k]);
    }
  };
  auto leave = [&]() {
    float* o = outS + (blockIdx.x + group) * D;
    put_sums<VEC, N>(o, tid, tpr, D, S1);
    if (BIAS) put_sums<VEC, N>(o + (p.blocks + p.groups) * D, tid, tpr, D, S0);
  };
  enter();
  int64_t until = (group + 1) * p.per;  // the group's last row and one
  Raw<T, VEC, N> rx, rhh, ry, rd;
  float st[4];
  auto fetch = [&](int64_t r) {
    rx.load(static_cast<const T*>(p.x) + r * D, tid, tpr, D);
    rhh.load(static_cast<const T*>(p.h) + r * D, tid, tpr, D);
    if (p.dy) ry.load(static_cast<const T*>(p.dy) + r * D, tid, tpr, D);
    if (p.dz) rd.load(static_cast<const T*>(p.dz) + r * D, tid, tpr, D);
#pragma unroll
    for (int k = 0; k < 4; ++k) st[k] = p.stats[k * p.rows + r];
  };
  fetch(r0);
  for (int64_t r = r0; r < r1; ++r) {
    if (r == until) {
      leave();
      ++group;
      until += p.per;
#pragma unroll
      for (int k = 0; k < N; ++k) S1[k] = S0[k] = two(0.f);
      enter();
    }
    const float mh = st[0], rh = st[1], mz = st[2], rz = st[3];
    float2 hh[N], zh[N], dy[N], d[N];
    rx.get(zh);
    rhh.get(hh);
#pragma unroll
    for (int k = 0; k < N; ++k) dy[k] = d[k] = two(0.f);
    if (p.dy) ry.get(dy);
    if (p.dz) rd.get(d);
    if (r + 1 < r1) fetch(r + 1);
    const float2 nh = two(-mh), nz = two(-mz);
    float2 s0 = two(0.f), s1 = two(0.f);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      hh[k] = __fmul2_rn(__fadd2_rn(hh[k], nh), two(rh));
      float2 z = __ffma2_rn(hh[k], gw[k], __fmul2_rn(zh[k], two(p.scale)));
      if (BIAS) z = __fadd2_rn(z, gb[k]);
      zh[k] = __fmul2_rn(__fadd2_rn(z, nz), two(rz));
      const float2 t = __fmul2_rn(dy[k], wp[k]);  // 0 past the row's end
      s0 = __ffma2_rn(t, zh[k], s0);
      s1 = __fadd2_rn(s1, t);
    }
    float a[2] = {s0.x + s0.y, s1.x + s1.y};
    sum(a);
    const float2 ka = two(-rz * a[0] * inv_d), km = two(p.layer ? -rz * a[1] * inv_d : 0.f);
    s0 = s1 = two(0.f);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      d[k] = __ffma2_rn(__fmul2_rn(dy[k], wp[k]), two(rz), __fadd2_rn(d[k], km));
      d[k] = __ffma2_rn(zh[k], ka, d[k]);
      const float2 e = __fmul2_rn(d[k], gw[k]);  // 0 past the row's end
      s0 = __ffma2_rn(e, hh[k], s0);
      s1 = __fadd2_rn(s1, e);
    }
    float b[2] = {s0.x + s0.y, s1.x + s1.y};
    sum(b);
    const float2 kb = two(-rh * b[0] * inv_d), kn = two(p.layer ? -rh * b[1] * inv_d : 0.f);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      S1[k] = __ffma2_rn(d[k], hh[k], S1[k]);
      T1[k] = __ffma2_rn(dy[k], zh[k], T1[k]);
      if (BIAS) S0[k] = __fadd2_rn(S0[k], d[k]), T0[k] = __fadd2_rn(T0[k], dy[k]);
      const float2 e = __fmul2_rn(d[k], gw[k]);
      hh[k] = __ffma2_rn(hh[k], kb, __ffma2_rn(e, two(rh), kn));
      d[k] = __fmul2_rn(d[k], two(p.scale));
    }
    store<T, VEC, N>(static_cast<T*>(p.dx) + r * D, tid, tpr, D, d);
    store<T, VEC, N>(static_cast<T*>(p.dh) + r * D, tid, tpr, D, hh);
  }
  leave();
  put_sums<VEC, N>(outT + (int64_t)blockIdx.x * D, tid, tpr, D, T1);
  if (BIAS) put_sums<VEC, N>(outT + (p.blocks + blockIdx.x) * D, tid, tpr, D, T0);
}

// The vectors' gradients from the blocks' sums, in two steps.  First, 32 columns per block
// and part blockIdx.y of the groups and of the backward pass's blocks, its 32 warps in
// turn, added in order; the gates' gradients are complete here.
template <bool BIAS>
__global__ void __launch_bounds__(1024) gather_kernel(Params p, float* out) {
  __shared__ float acc[4][32][33];
  dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  const float* S = p.part + c;
  const int64_t nS = (p.blocks + p.groups) * p.dim, nT = p.blocks * p.dim;
  const float* R = S + 2 * nS;
  const int64_t first = (int64_t)blockIdx.y * 32 + warp, step = gridDim.y * 32;
  float w = 0.f, b = 0.f, t1 = 0.f, t0 = 0.f;
  if (c < p.dim) {
    if (p.groups > 1) {
      for (int64_t g = first; g < p.groups; g += step) {
        float s1 = 0.f, s0 = 0.f;
        const int64_t k1 = p.blocks ? block_of(p, (g + 1) * p.per - 1) : -1;
#pragma unroll 4
        for (int64_t k = p.blocks ? block_of(p, g * p.per) : 0; k <= k1; ++k) {
          s1 += S[(k + g) * p.dim];
          if (BIAS) s0 += S[nS + (k + g) * p.dim];
        }
        const float gt = vec1(p.gate, p.vdt, g * p.dim + c, 1.f);
        w += gt * s1;
        b += gt * s0;
        put1(p.dgate, p.vdt, g * p.dim + c,
             vec1(p.w_post, p.vdt, c, 1.f) * s1 + vec1(p.b_post, p.vdt, c, 0.f) * s0);
      }
    } else {
#pragma unroll 4
      for (int64_t k = first; k < p.blocks; k += step) {
        w += S[k * p.dim];
        if (BIAS) b += S[nS + k * p.dim];
      }
    }
#pragma unroll 4
    for (int64_t k = first; k < p.blocks; k += step) {
      t1 += R[k * p.dim];
      if (BIAS) t0 += R[nT + k * p.dim];
    }
  }
  acc[0][warp][lane] = w;
  acc[1][warp][lane] = b;
  acc[2][warp][lane] = t1;
  acc[3][warp][lane] = t0;
  __syncthreads();
  if (warp >= 4 || c >= p.dim) return;
  float s = 0.f;
  for (int i = 0; i < 32; ++i) s += acc[warp][i][lane];
  out[((int64_t)blockIdx.y * 4 + warp) * p.dim + c] = s;
}

__global__ void __launch_bounds__(128) finish_kernel(Params p, const float* in, int parts) {
  const int c = blockIdx.x * 128 + threadIdx.x;
  dependency_wait();
  if (c >= p.dim) return;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 16
  for (int i = 0; i < parts; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) s[k] += in[((int64_t)i * 4 + k) * p.dim + c];
  if (p.groups == 1) {
    put1(p.dgate, p.vdt, c, vec1(p.w_post, p.vdt, c, 1.f) * s[0] + vec1(p.b_post, p.vdt, c, 0.f) * s[1]);
    const float gt = vec1(p.gate, p.vdt, c, 1.f);
    s[0] *= gt;
    s[1] *= gt;
  }
  put1(p.dw_post, p.vdt, c, s[0]);
  put1(p.db_post, p.vdt, c, s[1]);
  put1(p.dw_pre, p.vdt, c, s[2]);
  put1(p.db_pre, p.vdt, c, s[3]);
}

// Blocks of the backward pass: what the SMs hold at 128 registers a thread, and at least
// four rows each.
static int64_t blocks_of(int64_t rows, int dim) {
  const int pairs = dim <= 4096 ? 4 : dim <= 8192 ? 8 : 16;
  const int tpr = (dim + 2 * pairs * 32 - 1) / (2 * pairs * 32) * 32;
  const int64_t most = (int64_t)device_sm_count() * (512 / tpr > 8 ? 8 : 512 / tpr), n = (rows + 3) / 4;
  return n < most ? n : most;
}
constexpr int MAX_PARTS = 16;
static int parts_of(int64_t groups, int64_t blocks) {
  const int64_t n = ((groups > blocks ? groups : blocks) + 31) / 32;
  return n < 1 ? 1 : n > MAX_PARTS ? MAX_PARTS : (int)n;
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T, int VEC, int N, bool WIDE, bool WARP>
static cudaError_t forward(const Params& p, cudaStream_t s) {
  if constexpr (WARP) {
    return launch_after(forward_kernel<T, VEC, N, WIDE, true>, dim3((unsigned)((p.rows + 3) / 4)), dim3(128), 0, s, p);
  } else {
    const int tpr = (p.dim + 2 * N * 32 - 1) / (2 * N * 32) * 32;
    return launch_after(forward_kernel<T, VEC, N, WIDE, false>, dim3((unsigned)p.rows), dim3(tpr), 0, s, p);
  }
}

template <typename T, int VEC, bool WIDE>
static cudaError_t run_forward(const Params& p, cudaStream_t s) {
  if (p.dim <= 256) return forward<T, VEC, 4, WIDE, true>(p, s);
  if (p.dim <= 512) return forward<T, VEC, 8, WIDE, true>(p, s);
  if (p.dim <= 768) return forward<T, VEC, 12, WIDE, true>(p, s);
  if (p.dim <= 1024) return forward<T, VEC, 16, WIDE, true>(p, s);
  if (p.dim <= 8192) return forward<T, VEC, 4, WIDE, false>(p, s);
  return forward<T, VEC, 8, WIDE, false>(p, s);
}

template <typename T, int VEC, int N, bool WIDE, bool BIAS>
static cudaError_t backward(const Params& p, cudaStream_t s) {
  const int tpr = (p.dim + 2 * N * 32 - 1) / (2 * N * 32) * 32;
  return launch_after(backward_kernel<T, VEC, N, WIDE, BIAS>, dim3((unsigned)p.blocks), dim3(tpr), 0, s, p);
}

template <typename T, int VEC, bool WIDE, bool BIAS>
static cudaError_t run_backward(const Params& p, cudaStream_t s) {
  if (p.dim <= 4096) return backward<T, VEC, 4, WIDE, BIAS>(p, s);
  if (p.dim <= 8192) return backward<T, VEC, 8, WIDE, BIAS>(p, s);
  return backward<T, VEC, 16, WIDE, BIAS>(p, s);
}

template <typename T>
static cudaError_t run(const Params& p, bool bwd, cudaStream_t s) {
  constexpr int VEC = 16 / sizeof(T);
  const bool wide = aligned16(p.w_post) && aligned16(p.b_post) && aligned16(p.w_pre) && aligned16(p.b_pre) && aligned16(p.gate);
  const bool vec = p.dim % VEC == 0 && aligned16(p.x) && aligned16(p.h) &&
                   (bwd ? aligned16(p.dz) && aligned16(p.dy) && aligned16(p.dx) && aligned16(p.dh)
                        : aligned16(p.z) && aligned16(p.y));
  if (!bwd)
    return vec && wide ? run_forward<T, VEC, true>(p, s)
           : vec       ? run_forward<T, VEC, false>(p, s)
                       : run_forward<T, 1, true>(p, s);
  const bool bias = p.b_post || p.db_post || p.db_pre;
  cudaError_t e = cudaSuccess;
  if (p.rows > 0) {
    if (vec && wide) e = bias ? run_backward<T, VEC, true, true>(p, s) : run_backward<T, VEC, true, false>(p, s);
    else if (vec) e = bias ? run_backward<T, VEC, false, true>(p, s) : run_backward<T, VEC, false, false>(p, s);
    else e = bias ? run_backward<T, 1, true, true>(p, s) : run_backward<T, 1, true, false>(p, s);
  }
  if (e != cudaSuccess) return e;
  const int parts = parts_of(p.groups, p.blocks);
  float* sums = p.part + (4 * p.blocks + 2 * p.groups) * p.dim;
  const dim3 grid((unsigned)((p.dim + 31) / 32), (unsigned)parts);
  e = launch_after(bias ? gather_kernel<true> : gather_kernel<false>, grid, dim3(1024), 0, s, p, sums);
  if (e != cudaSuccess) return e;
  return launch_after(finish_kernel, dim3((unsigned)((p.dim + 127) / 128)), dim3(128), 0, s, p, (const float*)sums, parts);
}

static int launch(int dtype, const Params& p, bool bwd, cudaStream_t s) {
  const cudaError_t e = dtype == FMS_F32   ? run<float>(p, bwd, s)
                        : dtype == FMS_F16 ? run<__half>(p, bwd, s)
                                           : run<__nv_bfloat16>(p, bwd, s);
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
  if (rows < 0 || groups < 0 || dim <= 0) return 0;
  const int64_t blocks = norm::blocks_of(rows, dim);
  return (size_t)(4 * blocks + 2 * groups + 4 * norm::parts_of(groups, blocks)) * dim * sizeof(float);
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
  p.blocks = norm::blocks_of(rows, dim);
  p.per = groups > 0 ? rows / groups : 1;
  p.vdt = vdtype; p.layer = kind == FMS_NORM_LAYER;
  return norm::launch(dtype, p, true, (cudaStream_t)stream);
}

}  // extern "C"

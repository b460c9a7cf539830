// fms_linear_int8.cu -- linear layer in 8-bit integers with one scale per token
// and one per output channel:
//
//   y[t,c] = (sx_t * sw_c) * float(sum_k xc[t,k] * wc[c,k]) + b_c
//
// The integer sum is exact (int32; the entry point bounds K).  Float inputs are
// quantised per token first, in float32 whatever their type: scale =
// max(absmax, 1e-8) * (1/127), code = round to nearest even of x / scale.
//
// Up to FEW tokens one kernel quantises and multiplies on the CUDA cores (bound by
// reading the weights once); more go through a quantising pass and the tcgen05
// engine (kind::i8, scales in the epilogue).  (One kernel that quantises into the MMA's
// shared memory, for layers of up to 256 channels whose weights stay there, was between 18%
// faster and 28% slower over 18944 to 180000 tokens, and no faster at 46080 x 768 -> 128.)
#include "fms_gemm_tc.cuh"
#include "fms_internal.h"

#include <type_traits>

namespace fms {
namespace lin8 {

constexpr int FEW = 8;  // tokens of the CUDA-core kernel

// ------------------------------------------------------------------ quantising

// 127 / absmax and its inverse for one token.  A token that holds an infinity or a
// NaN has no scale: all its outputs are NaN.
struct Scale {
  float s, inv;
};
__device__ __forceinline__ Scale make_scale(uint32_t top_bits) {
  const float am = __uint_as_float(top_bits);
  Scale r;
  r.s = am <= 3.402823466e38f ? fmaxf(am, 1e-8f) * (1.f / 127.f) : NAN;
  r.inv = __frcp_rn(r.s);
  return r;
}
// The code of x in the low byte.  x / s as a product with the reciprocal and one
// correction by the remainder (Markstein's division step), which is the correctly
// rounded quotient; adding 1.5 * 2^23 rounds it to a whole number, ties to even.
// |x / s| <= 127 (1 + 2^-23), so no clamp is needed.
__device__ __forceinline__ uint32_t code(float x, Scale s) {
  const float q = x * s.inv;
  const float r = fmaf(-q, s.s, x);
  return __float_as_uint(fmaf(r, s.inv, q) + 12582912.f);
}
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// The values of one 16-byte vector as float32: 8 of a 16-bit type, 4 of float32.
template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  static __device__ __forceinline__ void get(uint4 v, float (&f)[N]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (N == 4) {
        f[i] = __uint_as_float(w[i]);
      } else {
        const float2 p = gemm::unpack2<T>(w[i]);
        f[2 * i] = p.x;
        f[2 * i + 1] = p.y;
      }
    }
  }
};

// W warps per token with the row in registers: NV 16-byte vectors per lane.  Bound by
// memory: the row is read once and its codes written once.  (One warp with 16 vectors a
// lane held too few rows in flight: 30 us for 8192 x 4096 against 21 with four warps.)
template <typename T, int NV, int W>
__global__ void __launch_bounds__(256) quantize_kernel(const T* x, int64_t rows, int K, int8_t* codes, int pitch,
                                                       float* scales) {
  constexpr int N = Vec<T>::N, TPR = 32 * W;
  __shared__ uint32_t part[8];
  const int warp = threadIdx.x >> 5, tid = threadIdx.x % TPR;
  const int64_t t = (int64_t)blockIdx.x * (8 / W) + threadIdx.x / TPR;
  const bool real = t < rows;
  dependency_wait();
  const uint4* xt = reinterpret_cast<const uint4*>(x + t * K);
  uint4 v[NV];
  uint32_t top = 0;  // bits of the largest |x|; as whole numbers a NaN's are above infinity's
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    v[i] = make_uint4(0, 0, 0, 0);
    if (real && (i * TPR + tid) * N < K) v[i] = xt[i * TPR + tid];
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float f[N];
    Vec<T>::get(v[i], f);
#pragma unroll
    for (int j = 0; j < N; ++j) top = max(top, abs_bits(f[j]));
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (W > 1) {
    if ((threadIdx.x & 31) == 0) part[warp] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; ++i) top = max(top, part[warp / W * W + i]);
  }
  if (!real) return;
  const Scale s = make_scale(top);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int k = (i * TPR + tid) * N;
    if (k >= K) continue;
    float f[N];
    Vec<T>::get(v[i], f);
    uint32_t c[N / 4];
#pragma unroll
    for (int j = 0; j < N / 4; ++j)
      c[j] = pack4(code(f[4 * j], s), code(f[4 * j + 1], s), code(f[4 * j + 2], s), code(f[4 * j + 3], s));
    if constexpr (N == 8) *reinterpret_cast<uint2*>(codes + t * pitch + k) = make_uint2(c[0], c[1]);
    else *reinterpret_cast<uint32_t*>(codes + t * pitch + k) = c[0];
  }
  if (tid == 0) scales[t] = s.s;
}

// Rows of up to 32 NE values that start anywhere: a warp each, a value per lane at a time.
template <typename T, int NE>
__global__ void __launch_bounds__(256) quantize_odd_kernel(const T* x, int64_t rows, int K, int8_t* codes, int pitch,
                                                           float* scales) {
  const int lane = threadIdx.x & 31;
  const int64_t t = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  dependency_wait();
  if (t >= rows) return;
  const T* xt = x + t * K;
  T v[NE];
#pragma unroll
  for (int i = 0; i < NE; ++i) v[i] = i * 32 + lane < K ? xt[i * 32 + lane] : Tr<T>::from(0.f);
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < NE; ++i) top = max(top, abs_bits(Tr<T>::to(v[i])));
  const Scale s = make_scale(__reduce_max_sync(0xffffffffu, top));
#pragma unroll
  for (int i = 0; i < NE; ++i)
    if (i * 32 + lane < K) codes[t * pitch + i * 32 + lane] = (int8_t)code(Tr<T>::to(v[i]), s);
  if (lane == 0) scales[t] = s.s;
}

// Rows of any width and start, one block each, read twice.
template <typename T>
__global__ void __launch_bounds__(256) quantize_any_kernel(const T* x, int64_t rows, int K, int8_t* codes, int pitch,
                                                           float* scales) {
  __shared__ uint32_t part[8];
  dependency_wait();
  for (int64_t t = blockIdx.x; t < rows; t += gridDim.x) {
    const T* xt = x + t * K;
    uint32_t top = 0;
    for (int k = threadIdx.x; k < K; k += 256) top = max(top, abs_bits(Tr<T>::to(xt[k])));
    top = __reduce_max_sync(0xffffffffu, top);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, part[i]);
    const Scale s = make_scale(top);
    for (int k = threadIdx.x; k < K; k += 256) codes[t * pitch + k] = (int8_t)code(Tr<T>::to(xt[k]), s);
    if (threadIdx.x == 0) scales[t] = s.s;
  }
}

// ------------------------------------------------------------------ a few tokens

// Every block quantises all tokens for itself (they are a few KB) into shared memory;
// then one warp per output channel: 16-byte pieces of the weight's row against the same
// pieces of every token, dp4a, and a sum over the lanes.  VEC: bytes of a piece that the
// weights' alignment allows.
template <typename X, typename Y, int NTOK, int VEC>
__global__ void __launch_bounds__(256) few_kernel(const X* x, const float* x_scales, const int8_t* wc, const float* sw,
                                                  const Y* bias, int rows, int K, int C, Y* y) {
  extern __shared__ __align__(16) unsigned char codes_s[];  // (rows, pitch)
  __shared__ float sx[NTOK];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int pitch = (K + 15) & ~15;
  dependency_wait();
  for (int t = warp; t < rows; t += 8) {
    unsigned char* ct = codes_s + t * pitch;
    if constexpr (sizeof(X) == 1) {
      for (int k = lane; k < pitch; k += 32) ct[k] = k < K ? (unsigned char)x[(int64_t)t * K + k] : 0;
      if (lane == 0) sx[t] = x_scales[t];
    } else {
      const X* xt = x + (int64_t)t * K;
      uint32_t top = 0;
      for (int k = lane; k < K; k += 32) top = max(top, abs_bits(Tr<X>::to(xt[k])));
      const Scale s = make_scale(__reduce_max_sync(0xffffffffu, top));
      for (int k = lane; k < pitch; k += 32) ct[k] = k < K ? (unsigned char)code(Tr<X>::to(xt[k]), s) : 0;
      if (lane == 0) sx[t] = s.s;
    }
  }
  __syncthreads();
  for (int c = blockIdx.x * 8 + warp; c < C; c += gridDim.x * 8) {
    const int8_t* w = wc + (int64_t)c * K;
    int32_t acc[NTOK];
#pragma unroll
    for (int t = 0; t < NTOK; ++t) acc[t] = 0;
#pragma unroll 2
    for (int k = lane * VEC; k < K; k += 32 * VEC) {
      if constexpr (VEC == 16) {
        const int4 v = *reinterpret_cast<const int4*>(w + k);
#pragma unroll
        for (int t = 0; t < NTOK; ++t) {
          if (t >= rows) break;
          const int4 q = *reinterpret_cast<const int4*>(codes_s + t * pitch + k);
          acc[t] = __dp4a(v.x, q.x, __dp4a(v.y, q.y, __dp4a(v.z, q.z, __dp4a(v.w, q.w, acc[t]))));
        }
      } else if constexpr (VEC == 4) {
        const int v = *reinterpret_cast<const int*>(w + k);
#pragma unroll
        for (int t = 0; t < NTOK; ++t) {
          if (t >= rows) break;
          acc[t] = __dp4a(v, *reinterpret_cast<const int*>(codes_s + t * pitch + k), acc[t]);
        }
      } else {
        const int v = w[k];
#pragma unroll
        for (int t = 0; t < NTOK; ++t) {
          if (t >= rows) break;
          acc[t] += v * (int)(int8_t)codes_s[t * pitch + k];
        }
      }
    }
    int32_t mine = 0;
#pragma unroll
    for (int t = 0; t < NTOK; ++t) {
      if (t >= rows) break;
      const int32_t sum = __reduce_add_sync(0xffffffffu, acc[t]);
      if (lane == t) mine = sum;
    }
    if (lane < rows) {
      float v = (sx[lane] * sw[c]) * (float)mine;
      if (bias) v += Tr<Y>::to(bias[c]);
      y[(int64_t)lane * C + c] = Tr<Y>::from(v);
    }
  }
}

// ------------------------------------------------------------------ the engine's epilogue

template <typename Y>
struct ScaleEpi {
  struct alignas(64) Params {
    CUtensorMap map;  // y, where `mapped`
    const float *sx, *sw;
    const Y* bias;
    Y* y;
    int64_t rows;
    int cols;
    int mapped;       // rows of y start on 16 bytes
    int wide;         // sw and bias start on 16 bytes
  };
  template <int BN>
  struct Ahead {};
  template <int BN>
  static __device__ __forceinline__ void fetch(const Params&, const gemm::Tile&, int64_t, int, Ahead<BN>&) {}
  template <int BN, class Release>
  static __device__ __forceinline__ void run(const Params& p, const gemm::Tile& t, int64_t row, int half, uint32_t addr,
                                             const Ahead<BN>&, unsigned char* stage, Release release) {
    const int lane = threadIdx.x & 31;
    const float sx = row < p.rows ? p.sx[row] : 0.f;
#pragma unroll 1
    for (int c = half * (BN / 64); c < (half + 1) * (BN / 64); ++c) {
      __syncwarp();
      uint32_t v[32];
      gemm::load32(addr + c * 32, v);
      if (c + 1 == (half + 1) * (BN / 64)) release();
      const int col = t.n * BN + c * 32;
      float f[32];
      // All lanes read the same scales and biases, so the loads are as wide as they may be:
      // 32768 x 256 -> 1024 in bfloat16 44 us, by single values 50.
      // Columns past the end take the last one's; they are not stored.
      if (p.wide && col + 32 <= p.cols) {
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const float4 w = *reinterpret_cast<const float4*>(p.sw + col + i);
          f[i] = (sx * w.x) * (float)(int32_t)v[i];
          f[i + 1] = (sx * w.y) * (float)(int32_t)v[i + 1];
          f[i + 2] = (sx * w.z) * (float)(int32_t)v[i + 2];
          f[i + 3] = (sx * w.w) * (float)(int32_t)v[i + 3];
        }
        if (p.bias) {
          constexpr int N = Vec<Y>::N;
#pragma unroll
          for (int i = 0; i < 32; i += N) {
            float b[N];
            Vec<Y>::get(*reinterpret_cast<const uint4*>(p.bias + col + i), b);
#pragma unroll
            for (int j = 0; j < N; ++j) f[i + j] += b[j];
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const int at = min(col + i, p.cols - 1);
          f[i] = (sx * p.sw[at]) * (float)(int32_t)v[i];
          if (p.bias) f[i] += Tr<Y>::to(p.bias[at]);
        }
      }
      // 128 bytes of a row at a time: every 32 columns in float32, every 64 in 16 bits
      constexpr int PER = 128 / sizeof(Y), GROUPS = BN >= 128 ? PER / 32 : 1;
      const int k = GROUPS == 2 ? c & 1 : 0;
      if (k == 0) gemm::out_free(lane);
      if constexpr (sizeof(Y) == 2) {
        uint32_t o[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = gemm::pack2<Y>(f[2 * i], f[2 * i + 1]);
        gemm::put(stage, lane, 4 * k, o);
      } else {
        uint32_t o[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(f[i]);
        gemm::put(stage, lane, 0, o);
      }
      const int col0 = col - 32 * k;
      const int64_t row0 = row - lane;
      if (k != GROUPS - 1 || col0 >= p.cols || row0 >= p.rows) continue;
      if (32 * GROUPS == PER && p.mapped) gemm::out_store(stage, &p.map, col0, (int)row0, lane);
      else
        gemm::out_rows<sizeof(Y)>(stage, p.y + row0 * p.cols + col0, p.cols, (int)min(p.rows - row0, (int64_t)32),
                                  min(p.cols - col0, 32 * GROUPS), lane);
    }
  }
};

// ------------------------------------------------------------------ host side

static size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }
static int pitch_of(int K) { return (K + 15) & ~15; }
static bool aligned(const void* p, int n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Bytes copied to rows `pitch` apart, for codes whose rows do not start on 16 bytes.
// A warp per row, four codes at a time: two neighbouring words of the source, shifted; the
// row's first and last words byte by byte, so that no byte outside it is read.
__global__ void __launch_bounds__(256) pitch_kernel(const int8_t* src, int64_t rows, int K, int8_t* dst, int pitch) {
  const int lane = threadIdx.x & 31, words = (K + 3) / 4;
  dependency_wait();
  for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < rows; r += (int64_t)gridDim.x * 8) {
    const uint8_t* a = reinterpret_cast<const uint8_t*>(src) + r * K;
    const int off = (int)(reinterpret_cast<uintptr_t>(a) & 3);
    const uint32_t* w = reinterpret_cast<const uint32_t*>(a - off);
    uint32_t* b = reinterpret_cast<uint32_t*>(dst + r * pitch);
#pragma unroll 4
    for (int c = lane; c < words; c += 32) {
      uint32_t v = 0;
      if (c > 0 && c < words - 2) {
        v = __funnelshift_r(w[c], w[c + 1], 8 * off);
      } else {
        for (int j = 0; j < 4; ++j)
          if (4 * c + j < K) v |= (uint32_t)a[4 * c + j] << (8 * j);
      }
      b[c] = v;
    }
  }
}
static cudaError_t pitched(const int8_t*& p, int64_t rows, int K, int8_t* copy, cudaStream_t s) {
  if (K % 16 == 0 && aligned(p, 16)) return cudaSuccess;
  int64_t b = (rows + 7) / 8;
  if (b > device_sm_count() * 8) b = device_sm_count() * 8;
  const cudaError_t e = launch_after(pitch_kernel, dim3((unsigned)b), dim3(256), 0, s, p, rows, K, copy, pitch_of(K));
  p = copy;
  return e;
}

template <typename T>
static cudaError_t quantize(const void* xv, int64_t rows, int K, int8_t* codes, float* scales, cudaStream_t s) {
  const T* x = (const T*)xv;
  constexpr int N = Vec<T>::N;
  const int pitch = pitch_of(K);
  if (K % N != 0 || !aligned(x, 16) || K > 32 * N * 32) {
    const dim3 warps((unsigned)((rows + 7) / 8));
    if (K <= 256) return launch_after(quantize_odd_kernel<T, 8>, warps, dim3(256), 0, s, x, rows, K, codes, pitch, scales);
    if (K <= 512) return launch_after(quantize_odd_kernel<T, 16>, warps, dim3(256), 0, s, x, rows, K, codes, pitch, scales);
    if (K <= 1024) return launch_after(quantize_odd_kernel<T, 32>, warps, dim3(256), 0, s, x, rows, K, codes, pitch, scales);
    const int64_t most = (int64_t)device_sm_count() * 8;
    return launch_after(quantize_any_kernel<T>, dim3((unsigned)(rows < most ? rows : most)), dim3(256), 0, s, x, rows, K,
                        codes, pitch, scales);
  }
  auto go = [&](auto kernel, int w) {
    return launch_after(kernel, dim3((unsigned)((rows * w + 7) / 8)), dim3(256), 0, s, x, rows, K, codes, pitch, scales);
  };
  const int nv = (K + 32 * N - 1) / (32 * N);
  if (nv <= 1) return go(quantize_kernel<T, 1, 1>, 1);
  if (nv <= 2) return go(quantize_kernel<T, 2, 1>, 1);
  if (nv <= 3) return go(quantize_kernel<T, 3, 1>, 1);
  if (nv <= 4) return go(quantize_kernel<T, 4, 1>, 1);
  if (nv <= 8) return go(quantize_kernel<T, 4, 2>, 2);
  if (nv <= 16) return go(quantize_kernel<T, 4, 4>, 4);
  return go(quantize_kernel<T, 4, 8>, 8);
}

struct Args {
  const void* x;
  const float* x_scales;
  const int8_t* wc;
  const float* sw;
  const void* bias;
  int64_t rows;
  int K, C;
  void* y;
  char* ws;
};

struct Space {
  size_t codes, scales, w, total;
};
static bool few(int64_t rows, int K) { return rows <= FEW && rows * pitch_of(K) <= 40 * 1024; }
static Space space(int x_dtype, int64_t rows, int K, int C) {
  Space s{};
  if (few(rows, K)) return s;
  s.scales = align256((size_t)rows * pitch_of(K));
  s.w = s.scales + (x_dtype == FMS_I8 ? 0 : align256((size_t)rows * 4));
  s.total = s.w + align256((size_t)C * pitch_of(K));
  return s;
}

template <typename X, typename Y, int NTOK>
static cudaError_t run_few(const Args& p, cudaStream_t s) {
  int blocks = (p.C + 7) / 8;
  const int most = device_sm_count() * 4;
  if (blocks > most) blocks = most;
  const int smem = (int)p.rows * pitch_of(p.K);
  const X* x = (const X*)p.x;
  const Y* bias = (const Y*)p.bias;
  Y* y = (Y*)p.y;
  auto go = [&](auto kernel) {
    return launch_after(kernel, dim3((unsigned)blocks), dim3(256), smem, s, x, p.x_scales, p.wc, p.sw, bias, (int)p.rows,
                        p.K, p.C, y);
  };
  if (p.K % 16 == 0 && aligned(p.wc, 16)) return go(few_kernel<X, Y, NTOK, 16>);
  if (p.K % 4 == 0 && aligned(p.wc, 4)) return go(few_kernel<X, Y, NTOK, 4>);
  return go(few_kernel<X, Y, NTOK, 1>);
}

template <typename Y, int CG, int BN>
static cudaError_t product(const int8_t* xc, const float* sx, const int8_t* wc, const Args& p, cudaStream_t s) {
  CUtensorMap a, b;
  if (!gemm::make_map(&a, FMS_I8, xc, p.K, p.rows, pitch_of(p.K), 128) ||
      !gemm::make_map(&b, FMS_I8, wc, p.K, p.C, pitch_of(p.K), BN / CG))
    return cudaErrorNotSupported;
  gemm::Work w{};
  w.mt = (int)((p.rows + 128 * CG - 1) / (128 * CG));
  w.nt = (p.C + BN - 1) / BN;
  w.splits = 1;
  w.kb = (p.K + 127) / 128;
  w.idesc = ptx::idesc_i8(128 * CG, BN);
  typename ScaleEpi<Y>::Params e{};
  e.sx = sx;
  e.sw = p.sw;
  e.bias = (const Y*)p.bias;
  e.y = (Y*)p.y;
  e.rows = p.rows;
  e.cols = p.C;
  e.wide = aligned(p.sw, 16) && (!p.bias || aligned(p.bias, 16));
  e.mapped = p.C * sizeof(Y) % 16 == 0 && aligned(p.y, 16) &&
             gemm::make_map(&e.map, sizeof(Y) == 4 ? FMS_F32 : std::is_same<Y, __half>::value ? FMS_F16 : FMS_BF16, p.y, p.C,
                            p.rows, (int64_t)p.C * sizeof(Y), 32);
  return gemm::launch<gemm::OP_ONE, CG, BN, false, false, true, ScaleEpi<Y>>(a, a, b, b, w, e, device_sm_count(), s);
}

template <typename X, typename Y>
static cudaError_t run(const Args& p, cudaStream_t s) {
  if (few(p.rows, p.K)) return p.rows == 1 ? run_few<X, Y, 1>(p, s) : run_few<X, Y, FEW>(p, s);
  const Space L = space(sizeof(X) == 1 ? FMS_I8 : FMS_F32, p.rows, p.K, p.C);
  int8_t* codes = (int8_t*)(p.ws + L.codes);
  const int8_t *xc, *wc = p.wc;
  const float* sx;
  cudaError_t e = pitched(wc, p.C, p.K, (int8_t*)(p.ws + L.w), s);
  if (e != cudaSuccess) return e;
  if constexpr (sizeof(X) == 1) {
    xc = (const int8_t*)p.x;
    e = pitched(xc, p.rows, p.K, codes, s);
    sx = p.x_scales;
  } else {
    float* sc = (float*)(p.ws + L.scales);
    e = quantize<X>(p.x, p.rows, p.K, codes, sc, s);
    xc = codes;
    sx = sc;
  }
  if (e != cudaSuccess) return e;
  switch (gemm::pick_shape(p.rows, p.C, (p.K + 127) / 128, device_sm_count())) {
    case 0: return product<Y, 2, 256>(xc, sx, wc, p, s);
    case 1: return product<Y, 2, 128>(xc, sx, wc, p, s);
    default: return product<Y, 1, 64>(xc, sx, wc, p, s);
  }
}

template <typename Y>
static cudaError_t run_x(int x_dtype, const Args& p, cudaStream_t s) {
  switch (x_dtype) {
    case FMS_I8: return run<int8_t, Y>(p, s);
    case FMS_F32: return run<float, Y>(p, s);
    case FMS_F16: return run<__half, Y>(p, s);
    default: return run<__nv_bfloat16, Y>(p, s);
  }
}

}  // namespace lin8

int read_lin8_device_error(int reset) { return gemm::read_error(reset); }

}  // namespace fms

using namespace fms;

extern "C" {

size_t fms_int8_linear_workspace_size(int x_dtype, int64_t rows, int dim, int out) {
  if (rows <= 0 || dim <= 0 || out <= 0) return 0;
  return lin8::space(x_dtype, rows, dim, out).total;
}

int fms_int8_linear_fwd(int x_dtype, const void* x, const float* x_scales, const int8_t* w_codes, const float* w_scales,
                        const void* bias, int64_t rows, int dim, int out, int y_dtype, void* y, void* workspace,
                        size_t ws_bytes, fms_stream_t stream) {
  if (x_dtype != FMS_I8 && x_dtype != FMS_F32 && x_dtype != FMS_F16 && x_dtype != FMS_BF16) return FMS_ERR_DTYPE;
  if (y_dtype != FMS_F32 && y_dtype != FMS_F16 && y_dtype != FMS_BF16) return FMS_ERR_DTYPE;
  if (rows < 0 || rows > INT32_MAX - 512 || dim < 1 || out < 0 || out > INT32_MAX - 512) return FMS_ERR_INVALID;
  if (dim > FMS_INT8_LINEAR_MAX_DIM) return FMS_ERR_TOO_LARGE;
  if (rows == 0 || out == 0) return FMS_OK;
  if (!y || !w_scales || !x || !w_codes || (x_dtype == FMS_I8 && !x_scales)) return FMS_ERR_INVALID;
  const size_t need = fms_int8_linear_workspace_size(x_dtype, rows, dim, out);
  if (need && (!workspace || ws_bytes < need)) return FMS_ERR_WORKSPACE;
  if (device_cc() != 100) return FMS_ERR_UNSUPPORTED;
  const lin8::Args p{x, x_scales, w_codes, w_scales, bias, rows, dim, out, y, (char*)workspace};
  cudaStream_t s = (cudaStream_t)stream;
  const cudaError_t e = y_dtype == FMS_F32   ? lin8::run_x<float>(x_dtype, p, s)
                        : y_dtype == FMS_F16 ? lin8::run_x<__half>(x_dtype, p, s)
                                             : lin8::run_x<__nv_bfloat16>(x_dtype, p, s);
  return e == cudaSuccess ? FMS_OK : e == cudaErrorNotSupported ? FMS_ERR_UNSUPPORTED : (int)e;
}

}  // extern "C"

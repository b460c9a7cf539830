// fms_glu.cuh -- the gated feed-forward block of a token encoder:
//
//   g = x Wg^T,  u = x Wu^T,  h = a(g) * u                      (forward)
//   du = dh * a(g),  dg = dh * u * a'(g)                        (backward)
//   dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x
//
// x (rows, dim), Wg and Wu (hidden, dim), h (rows, hidden), 16-bit; sums in
// float32.  One kernel makes both projections of a tile into one accumulator (its
// columns are those of Wg and of Wu) and applies the activation and the product as
// it leaves TMEM.  g and u are not kept for the backward pass but computed again by
// the same kernel with another epilogue: one more pair of products, against rounding
// g and u to 16 bits (which would double the gradients' error) and 4 * rows * hidden
// bytes between the passes.  dg and du are rounded to the inputs' type, the type of
// the products they enter.
#pragma once
#include "fms_act.cuh"
#include "fms_gemm_tc.cuh"
#include "fms_internal.h"

namespace fms {
namespace glu {

using gemm::Tile;

// h = a(g) u, or with BWD dg = dh u a'(g) and du = dh a(g).
template <typename T, int ACT, bool BWD>
struct HiddenEpi {
  struct alignas(64) Params {
    CUtensorMap m0, m1;  // o0 and o1, where `mapped`
    const T* dh;
    T *o0, *o1;          // h, or dg and du
    int64_t rows;
    int hidden, ldo;     // columns; elements between the rows of the outputs
    int ldd;             // and of dh
    int mapped;          // the outputs' rows start on 16 bytes, as the copy engine asks
  };
  static __host__ __device__ constexpr int GROUPS(int BN) { return BN >= 128 ? BN / 128 : 1; }  // of 32 columns of a warp
  // The cotangents of a warp's columns, on their way while the products run.
  template <int BN>
  struct Ahead {
    uint32_t d[BWD ? GROUPS(BN) : 1][16];
  };
  template <int BN>
  static __device__ __forceinline__ void fetch(const Params& p, const Tile& t, int64_t row, int half, Ahead<BN>& f) {
    if constexpr (BWD) {
#pragma unroll
      for (int k = 0; k < GROUPS(BN); ++k) {
        const int c = half * GROUPS(BN) + k, col = t.n * (BN / 2) + c * 32;
        const int n = row < p.rows && c < BN / 64 ? p.hidden - col : 0;
        gemm::load_row32(p.dh + row * p.ldd + col, f.d[k], n);
      }
    }
  }
  template <int BN, class Release>
  static __device__ __forceinline__ void run(const Params& p, const Tile& t, int64_t row, int half, uint32_t addr,
                                             const Ahead<BN>& f, unsigned char* out, Release release) {
    const int lane = threadIdx.x & 31;
    const int col0 = t.n * (BN / 2) + half * GROUPS(BN) * 32;
    uint32_t keep[GROUPS(BN)][16];
#pragma unroll
    for (int k = 0; k < GROUPS(BN); ++k) {
      const int c = half * GROUPS(BN) + k;
      if (c >= BN / 64) {
        release();
        break;
      }
      __syncwarp();
      uint32_t g[32], u[32];
      ptx::tmem_ld32(addr + c * 32, g);
      gemm::load32(addr + BN / 2 + c * 32, u);  // waits for both
      gemm::landed(g);
      if (k == GROUPS(BN) - 1) release();
      uint32_t o[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float2 a, da;
        const float2 gv = make_float2(__uint_as_float(g[2 * i]), __uint_as_float(g[2 * i + 1]));
        const float2 uv = make_float2(__uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1]));
        act_eval2<ACT, BWD>(gv, a, da);
        if (BWD) {
          const float2 e = gemm::unpack2<T>(f.d[k][i]);
          const float2 x = __fmul2_rn(__fmul2_rn(e, uv), da), y = __fmul2_rn(e, a);
          o[i] = gemm::pack2<T>(x.x, x.y);
          keep[k][i] = gemm::pack2<T>(y.x, y.y);
        } else {
          const float2 x = __fmul2_rn(a, uv);
          o[i] = gemm::pack2<T>(x.x, x.y);
        }
      }
      if (k == 0) gemm::out_free(lane);
      gemm::put(out, lane, 4 * k, o);
    }
    const int row0 = (int)(row - lane);
    const int rows = (int)min(p.rows - row0, (int64_t)32), cols = min(p.hidden - col0, 32 * GROUPS(BN));
    if (cols <= 0 || rows <= 0 || half * GROUPS(BN) >= BN / 64) return;
    auto leave = [&](const CUtensorMap* m, T* o) {
      if (GROUPS(BN) == 2 && p.mapped) gemm::out_store(out, m, col0, row0, lane);
      else gemm::out_rows<2>(out, o + (int64_t)row0 * p.ldo + col0, p.ldo, rows, cols, lane);
    };
    leave(&p.m0, p.o0);
    if (BWD) {
      gemm::out_free(lane);
#pragma unroll
      for (int k = 0; k < GROUPS(BN); ++k) gemm::put(out, lane, 4 * k, keep[k]);
      leave(&p.m1, p.o1);
    }
  }
};

// The accumulator as it is, in T, or in float32 where the sum is split (`part` then
// holds one (rows, cols) matrix after the other).  STACK: the rows are those of two
// outputs, `pad` rows of tiles each.
template <typename T, bool STACK>
struct StoreEpi {
  struct alignas(64) Params {
    CUtensorMap m0, m1;  // o0 and o1, where `mapped`
    T *o0, *o1;
    float* part;
    int64_t rows, pad;
    int cols;
    int ldp;             // elements between the rows of `part`, a multiple of 4
    int mapped;
  };
  template <int BN>
  struct Ahead {};
  template <int BN>
  static __device__ __forceinline__ void fetch(const Params&, const Tile&, int64_t, int, Ahead<BN>&) {}
  template <int BN, class Release>
  static __device__ __forceinline__ void run(const Params& p, const Tile& t, int64_t row, int half, uint32_t addr,
                                             const Ahead<BN>&, unsigned char* stage, Release release) {
    static_assert(BN >= 128, "64 columns to a warp");
    const int lane = threadIdx.x & 31;
    T* out = p.o0;
    const CUtensorMap* map = &p.m0;
    int64_t at = t.split * (STACK ? 2 : 1) * p.rows;
    if (STACK && row >= p.pad) {
      row -= p.pad;
      out = p.o1;
      map = &p.m1;
      at += p.rows;
    }
#pragma unroll 1
    for (int c = half * (BN / 64); c < (half + 1) * (BN / 64); ++c) {
      __syncwarp();
      uint32_t v[32];
      gemm::load32(addr + c * 32, v);
      if (c + 1 == (half + 1) * (BN / 64)) release();
      const int col = t.n * BN + c * 32;
      const int n = row < p.rows ? p.cols - col : 0;
      if (p.part) {
        if (n <= 0) continue;
        float* q = p.part + (at + row) * p.ldp + col;
        if (n >= 32) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            reinterpret_cast<uint4*>(q)[i] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (i < n) q[i] = __uint_as_float(v[i]);
        }
      } else if (out) {
        uint32_t o[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = gemm::pack2<T>(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
        if ((c & 1) == 0) gemm::out_free(lane);
        gemm::put(stage, lane, 4 * (c & 1), o);
        const int64_t row0 = row - lane;
        if ((c & 1) && col - 32 < p.cols && row0 < p.rows) {
          if (p.mapped) gemm::out_store(stage, map, col - 32, (int)row0, lane);
          else
            gemm::out_rows<2>(stage, out + row0 * p.cols + col - 32, p.cols, (int)min(p.rows - row0, (int64_t)32),
                              min(p.cols - col + 32, 64), lane);
        }
      }
    }
  }
};

// Sum of the parts of a split product, in order; each part holds one or two matrices of
// rows x ldp values, of which cols count.
template <typename T>
__global__ void __launch_bounds__(256) join_kernel(const float* part, int splits, int64_t rows, int cols, int ldp,
                                                   int outputs, T* o0, T* o1) {
  dependency_wait();
  const int64_t each = rows * ldp, n = outputs * each;
  const bool wide = cols == ldp && ((reinterpret_cast<uintptr_t>(o0) | reinterpret_cast<uintptr_t>(o1)) & 7) == 0;
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < n; i += (int64_t)gridDim.x * 1024) {
    T* o = i < each ? o0 : o1;
    if (!o) continue;
    float4 s = *reinterpret_cast<const float4*>(part + i);
#pragma unroll 4
    for (int k = 1; k < splits; ++k) {
      const float4 v = *reinterpret_cast<const float4*>(part + k * n + i);
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
    const int64_t at = i < each ? i : i - each;
    if (wide) {
      *reinterpret_cast<uint2*>(o + at) = make_uint2(gemm::pack2<T>(s.x, s.y), gemm::pack2<T>(s.z, s.w));
    } else {
      const int64_t r = at / ldp;
      const int c = (int)(at - r * ldp);
      const float f[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < cols) o[r * cols + c + j] = Tr<T>::from(f[j]);
    }
  }
}

// Rows of n elements copied to rows ld apart, for operands whose rows do not start where
// TMA or a vector load asks; a warp per row, one matrix per blockIdx.y.
struct Pitch {
  const uint16_t* src;
  uint16_t* dst;
  int64_t rows;
  int n, ld;
};
struct Pitches {
  Pitch m[4];
  int count;
  // The operand with rows that start on `align` bytes: as it is, or the place of its copy.
  const void* add(const void* p, int64_t rows, int n, int ld, int align, void* copy) {
    const uintptr_t u = reinterpret_cast<uintptr_t>(p);
    if (n == ld && (u & (align - 1)) == 0) return p;
    m[count++] = {(const uint16_t*)p, (uint16_t*)copy, rows, n, ld};
    return copy;
  }
};
// Pairs of elements at a time: a row that starts on an odd element takes each pair from two
// neighbouring words, its first and last pair by themselves, so that nothing outside the row
// is read (copies are written in whole pairs: ld is even, what lies past n in a row is never
// read as an element).
static __global__ void __launch_bounds__(256) pitch_kernel(const Pitches p) {
  dependency_wait();
  const Pitch& j = p.m[blockIdx.y];
  const int lane = threadIdx.x & 31, words = j.n / 2;
  for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < j.rows; r += (int64_t)gridDim.x * 8) {
    const uint16_t* a = j.src + r * j.n;
    uint32_t* b = reinterpret_cast<uint32_t*>(j.dst + r * j.ld);
    if ((reinterpret_cast<uintptr_t>(a) & 2) == 0) {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(a);
#pragma unroll 8
      for (int c = lane; c < words; c += 32) b[c] = w[c];
    } else {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(a - 1);
#pragma unroll 8
      for (int c = lane; c < words; c += 32)
        b[c] = c > 0 && c < words - 1 ? __funnelshift_r(w[c], w[c + 1], 16) : a[2 * c] | (uint32_t)a[2 * c + 1] << 16;
    }
    if (lane == 0 && j.n % 2 != 0) b[words] = a[j.n - 1];  // the last element, alone
  }
}

struct Args {
  const void *x, *wg, *wu, *dh;
  int64_t rows;
  int dim, hidden;
  void *h, *dx, *dwg, *dwu;
  char* ws;
};

static int64_t up(int64_t n, int64_t m) { return (n + m - 1) / m * m; }
static int64_t tiles(int64_t n, int64_t t) { return (n + t - 1) / t; }

// Parts of a sum of kb blocks of 64 for `t` tiles of 256 x 256, whose parts hold `values`
// float32 each: what gives the shortest time by a pair of SMs doing a block in 0.35 us and
// starting and ending a tile in 8 blocks' time, and the parts being written and read at 5
// TB/s in a launch of 2 us more (measured: dx of 100 x 768 from 2 x 2048 columns in 25 us whole, in 17 in 16 parts).
static int parts_of(int64_t t, int kb, int64_t values) {
  const int64_t pairs = device_sm_count() / 2;
  int best = 1;
  double cost = 1e30;
  for (int s = 1; s <= 16 && (s == 1 || kb / s >= 4); ++s) {
    const double c = (double)tiles(t * s, pairs) * ((double)kb / s + 8.0) * 0.35 +
                     (s > 1 ? 2.0 + 8e-6 * (double)s * (double)values / 5.0 : 0.0);
    if (c < cost * 0.97) cost = c, best = s;
  }
  return best;
}

constexpr int FEW = 8;  // rows of the CUDA-core kernel

struct Space {
  size_t x, wg, wu, dh, dg, du, part, total;
  int ldd, ldh, splits, splits_x;  // parts of the weights' and of the input's gradients
};
// Offsets of the workspace.  The padded copies have their place whenever the width
// asks for them or a pointer might (the size is known without the pointers).
static Space space(int64_t rows, int dim, int hidden, bool bwd) {
  Space s{};
  if (!bwd && rows <= FEW) return s;
  s.ldd = (int)up(dim, 8);
  s.ldh = (int)up(hidden, 16);  // 32 bytes, for vector loads of dh
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t o = at;
    at += (size_t)up((int64_t)n, 256);
    return o;
  };
  s.x = take((size_t)rows * s.ldd * 2);
  s.wg = take((size_t)hidden * s.ldd * 2);
  s.wu = take((size_t)hidden * s.ldd * 2);
  if (bwd) {
    s.dh = take((size_t)rows * s.ldh * 2);
    s.dg = take((size_t)rows * s.ldh * 2);
    s.du = take((size_t)rows * s.ldh * 2);
    s.splits = parts_of(2 * tiles(hidden, 256) * tiles(dim, 256), (int)tiles(rows, 64), 2 * (int64_t)hidden * dim);
    s.splits_x = parts_of(tiles(rows, 256) * tiles(dim, 256), 2 * (int)tiles(hidden, 64), rows * dim);
    const size_t w = s.splits > 1 ? (size_t)s.splits * 2 * hidden * up(dim, 4) * 4 : 0;
    const size_t x = s.splits_x > 1 ? (size_t)s.splits_x * rows * up(dim, 4) * 4 : 0;
    s.part = take(w > x ? w : x);  // one after the other
  }
  s.total = at;
  return s;
}

static bool aligned(const void* p, int n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

static cudaError_t run_pitches(const Pitches& p, cudaStream_t s) {
  if (p.count == 0) return cudaSuccess;
  int64_t most = 1;
  for (int i = 0; i < p.count; ++i) most = p.m[i].rows > most ? p.m[i].rows : most;
  int64_t b = tiles(most, 8);
  if (b > device_sm_count() * 8) b = device_sm_count() * 8;
  return launch_after(pitch_kernel, dim3((unsigned)b, (unsigned)p.count), dim3(256), 0, s, p);
}

// ------------------------------------------------------------------ a few rows

// Up to FEW rows: one warp per hidden column reads its two weight rows once, 16 bytes a
// lane, against the same pieces of every row of x (from L1).  Bound by reading the
// weights; a tile of the matrix engine would leave 120 of its 128 rows empty and use
// hidden / 128 SMs only.
template <typename T, int ACT, int NR, bool WIDE>
__global__ void __launch_bounds__(128) few_kernel(const T* x, const T* wg, const T* wu, int rows, int dim, int hidden,
                                                  T* h) {
  const int lane = threadIdx.x & 31;
  const int f = blockIdx.x * 4 + (threadIdx.x >> 5);
  dependency_wait();
  if (f >= hidden) return;
  float2 g[NR], u[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) g[r] = u[r] = pair(0.f);
  if constexpr (WIDE) {
    const uint4* a = reinterpret_cast<const uint4*>(wg + (int64_t)f * dim);
    const uint4* b = reinterpret_cast<const uint4*>(wu + (int64_t)f * dim);
#pragma unroll 3
    for (int k = lane; k < dim / 8; k += 32) {
      const uint4 wa = a[k], wb = b[k];
      const uint32_t ga[4] = {wa.x, wa.y, wa.z, wa.w}, ub[4] = {wb.x, wb.y, wb.z, wb.w};
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        if (r >= rows) break;
        const uint4 xv = reinterpret_cast<const uint4*>(x + (int64_t)r * dim)[k];
        const uint32_t xs[4] = {xv.x, xv.y, xv.z, xv.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 v = gemm::unpack2<T>(xs[i]);
          g[r] = __ffma2_rn(v, gemm::unpack2<T>(ga[i]), g[r]);
          u[r] = __ffma2_rn(v, gemm::unpack2<T>(ub[i]), u[r]);
        }
      }
    }
  } else {
#pragma unroll 4
    for (int k = lane; k < dim; k += 32) {
      const float wa = Tr<T>::to(wg[(int64_t)f * dim + k]), wb = Tr<T>::to(wu[(int64_t)f * dim + k]);
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        if (r >= rows) break;
        const float v = Tr<T>::to(x[(int64_t)r * dim + k]);
        g[r].x = fmaf(v, wa, g[r].x);
        u[r].x = fmaf(v, wb, u[r].x);
      }
    }
  }
  float2 mine = pair(0.f);
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    if (r >= rows) break;
    float2 s = make_float2(g[r].x + g[r].y, u[r].x + u[r].y);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s.x += __shfl_xor_sync(0xffffffffu, s.x, o);
      s.y += __shfl_xor_sync(0xffffffffu, s.y, o);
    }
    if (lane == r) mine = s;
  }
  if (lane < rows) {
    float2 act, none;
    act_eval2<ACT, false>(pair(mine.x), act, none);
    h[(int64_t)lane * hidden + f] = Tr<T>::from(act.x * mine.y);
  }
}

template <typename T, int ACT, bool BWD, int CG, int BN>
static cudaError_t hidden_pass(int dtype, const void* x, const void* wg, const void* wu, int ldd,
                               const void* dh, int ldd_dh, const Args& p, T* o0, T* o1, int ldo, cudaStream_t s) {
  CUtensorMap a, b0, b1;
  const int box = BN / 2;
  if (!gemm::make_map(&a, dtype, x, p.dim, p.rows, (int64_t)ldd * 2, 128) ||
      !gemm::make_map(&b0, dtype, wg, p.dim, p.hidden, (int64_t)ldd * 2, box) ||
      !gemm::make_map(&b1, dtype, wu, p.dim, p.hidden, (int64_t)ldd * 2, box))
    return cudaErrorNotSupported;
  gemm::Work w{};
  w.mt = (int)tiles(p.rows, 128 * CG);
  w.nt = (int)tiles(p.hidden, BN / 2);
  w.splits = 1;
  w.kb = (int)tiles(p.dim, 64);
  w.idesc = gemm::idesc_f16(dtype, 128 * CG, BN, false, false);
  typename HiddenEpi<T, ACT, BWD>::Params e{};
  e.dh = (const T*)dh;
  e.o0 = o0;
  e.o1 = o1;
  e.rows = p.rows;
  e.hidden = p.hidden;
  e.ldo = ldo;
  e.ldd = ldd_dh;
  e.mapped = BN == 256 && ldo % 8 == 0 && aligned(o0, 16) && (!BWD || aligned(o1, 16)) &&
             gemm::make_map(&e.m0, dtype, o0, p.hidden, p.rows, (int64_t)ldo * 2, 32) &&
             (!BWD || gemm::make_map(&e.m1, dtype, o1, p.hidden, p.rows, (int64_t)ldo * 2, 32));
  return gemm::launch<gemm::OP_PAIR_B, CG, BN, false, false, false, HiddenEpi<T, ACT, BWD>>(a, a, b0, b1, w, e,
                                                                                            device_sm_count(), s);
}

template <typename T, int ACT, int NR>
static cudaError_t few_rows(const Args& p, cudaStream_t s) {
  const unsigned blocks = (unsigned)tiles(p.hidden, 4);
  const T *x = (const T*)p.x, *wg = (const T*)p.wg, *wu = (const T*)p.wu;
  if (p.dim % 8 == 0 && aligned(x, 16) && aligned(wg, 16) && aligned(wu, 16))
    return launch_after(few_kernel<T, ACT, NR, true>, dim3(blocks), dim3(128), 0, s, x, wg, wu, (int)p.rows, p.dim,
                        p.hidden, (T*)p.h);
  return launch_after(few_kernel<T, ACT, NR, false>, dim3(blocks), dim3(128), 0, s, x, wg, wu, (int)p.rows, p.dim, p.hidden,
                      (T*)p.h);
}

template <typename T, int ACT, bool BWD>
static cudaError_t hidden_any(int dtype, const void* x, const void* wg, const void* wu, int ldd, const void* dh,
                              int ldd_dh, const Args& p, T* o0, T* o1, int ldo, cudaStream_t s) {
  // the tile's columns are those of both products
  switch (gemm::pick_shape(p.rows, 2 * (int64_t)p.hidden, (int)tiles(p.dim, 64), device_sm_count())) {
    case 0: return hidden_pass<T, ACT, BWD, 2, 256>(dtype, x, wg, wu, ldd, dh, ldd_dh, p, o0, o1, ldo, s);
    case 1: return hidden_pass<T, ACT, BWD, 2, 128>(dtype, x, wg, wu, ldd, dh, ldd_dh, p, o0, o1, ldo, s);
    default: return hidden_pass<T, ACT, BWD, 1, 64>(dtype, x, wg, wu, ldd, dh, ldd_dh, p, o0, o1, ldo, s);
  }
}

template <typename T>
static cudaError_t join(const float* part, int splits, int64_t rows, int cols, int outputs, T* o0, T* o1,
                        cudaStream_t s) {
  const int ldp = (int)up(cols, 4);
  int64_t blocks = tiles(outputs * rows * ldp, 256 * 4);
  if (blocks > device_sm_count() * 8) blocks = device_sm_count() * 8;
  return launch_after(join_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, s, part, splits, rows, cols, ldp, outputs, o0,
                      o1);
}

// dx = dg Wg + du Wu: the weights as they lie are the second operand with its rows
// along the sum.
template <typename T>
static cudaError_t input_gradient(int dtype, const T* dg, const T* du, const void* wg, const void* wu, int ldd, int ldh,
                                  int splits, float* part, const Args& p, cudaStream_t s) {
  CUtensorMap a0, a1, b0, b1;
  if (!gemm::make_map(&a0, dtype, dg, p.hidden, p.rows, (int64_t)ldh * 2, 128) ||
      !gemm::make_map(&a1, dtype, du, p.hidden, p.rows, (int64_t)ldh * 2, 128) ||
      !gemm::make_map(&b0, dtype, wg, p.dim, p.hidden, (int64_t)ldd * 2, 64) ||
      !gemm::make_map(&b1, dtype, wu, p.dim, p.hidden, (int64_t)ldd * 2, 64))
    return cudaErrorNotSupported;
  gemm::Work w{};
  w.mt = (int)tiles(p.rows, 256);
  w.nt = (int)tiles(p.dim, 256);
  w.splits = splits;
  w.kb0 = (int)tiles(p.hidden, 64);
  w.kb = 2 * w.kb0;
  w.idesc = gemm::idesc_f16(dtype, 256, 256, false, true);
  typename StoreEpi<T, false>::Params e{};
  e.o0 = (T*)p.dx;
  e.rows = p.rows;
  e.cols = p.dim;
  e.part = splits > 1 ? part : nullptr;
  e.ldp = (int)up(p.dim, 4);
  e.mapped = !e.part && p.dim % 8 == 0 && aligned(p.dx, 16) &&
             gemm::make_map(&e.m0, dtype, p.dx, p.dim, p.rows, (int64_t)p.dim * 2, 32);
  const cudaError_t err = gemm::launch<gemm::OP_SUM, 2, 256, false, true, false, StoreEpi<T, false>>(
      a0, a1, b0, b1, w, e, device_sm_count(), s);
  if (err != cudaSuccess || splits == 1) return err;
  return join<T>(part, splits, p.rows, p.dim, 1, (T*)p.dx, nullptr, s);
}

// dWg = dg^T x over dWu = du^T x: both operands have their rows along the sum.
template <typename T>
static cudaError_t weight_gradients(int dtype, const T* dg, const T* du, const void* x, int ldd, int ldh, int splits,
                                    float* part, const Args& p, cudaStream_t s) {
  CUtensorMap a0, a1, b;
  if (!gemm::make_map(&a0, dtype, dg, p.hidden, p.rows, (int64_t)ldh * 2, 64) ||
      !gemm::make_map(&a1, dtype, du, p.hidden, p.rows, (int64_t)ldh * 2, 64) ||
      !gemm::make_map(&b, dtype, x, p.dim, p.rows, (int64_t)ldd * 2, 64))
    return cudaErrorNotSupported;
  gemm::Work w{};
  w.mt0 = (int)tiles(p.hidden, 256);
  w.mt = 2 * w.mt0;
  w.nt = (int)tiles(p.dim, 256);
  w.splits = splits;
  w.kb = (int)tiles(p.rows, 64);
  w.idesc = gemm::idesc_f16(dtype, 256, 256, true, true);
  typename StoreEpi<T, true>::Params e{};
  e.o0 = (T*)p.dwg;
  e.o1 = (T*)p.dwu;
  e.part = splits > 1 ? part : nullptr;
  e.rows = p.hidden;
  e.pad = (int64_t)w.mt0 * 256;
  e.cols = p.dim;
  e.ldp = (int)up(p.dim, 4);
  e.mapped = !e.part && p.dim % 8 == 0 && p.dwg && p.dwu && aligned(p.dwg, 16) && aligned(p.dwu, 16) &&
             gemm::make_map(&e.m0, dtype, p.dwg, p.dim, p.hidden, (int64_t)p.dim * 2, 32) &&
             gemm::make_map(&e.m1, dtype, p.dwu, p.dim, p.hidden, (int64_t)p.dim * 2, 32);
  const cudaError_t err = gemm::launch<gemm::OP_STACK_A, 2, 256, true, true, false, StoreEpi<T, true>>(
      a0, a1, b, b, w, e, device_sm_count(), s);
  if (err != cudaSuccess || splits == 1) return err;
  return join<T>(part, splits, p.hidden, p.dim, 2, (T*)p.dwg, (T*)p.dwu, s);
}

template <typename T, int ACT>
static cudaError_t run(int dtype, const Args& p, bool bwd, cudaStream_t s) {
  if (!bwd && p.rows <= FEW) return p.rows == 1 ? few_rows<T, ACT, 1>(p, s) : few_rows<T, ACT, FEW>(p, s);
  const Space L = space(p.rows, p.dim, p.hidden, bwd);
  Pitches c{};
  const void* x = c.add(p.x, p.rows, p.dim, L.ldd, 16, p.ws + L.x);
  const void* wg = c.add(p.wg, p.hidden, p.dim, L.ldd, 16, p.ws + L.wg);
  const void* wu = c.add(p.wu, p.hidden, p.dim, L.ldd, 16, p.ws + L.wu);
  const void* dh = bwd ? c.add(p.dh, p.rows, p.hidden, L.ldh, 32, p.ws + L.dh) : nullptr;
  cudaError_t e = run_pitches(c, s);
  if (e != cudaSuccess) return e;
  if (!bwd) return hidden_any<T, ACT, false>(dtype, x, wg, wu, L.ldd, nullptr, 0, p, (T*)p.h, nullptr, p.hidden, s);
  T *dg = (T*)(p.ws + L.dg), *du = (T*)(p.ws + L.du);
  e = hidden_any<T, ACT, true>(dtype, x, wg, wu, L.ldd, dh, L.ldh, p, dg, du, L.ldh, s);
  if (e == cudaSuccess && p.dx) e = input_gradient<T>(dtype, dg, du, wg, wu, L.ldd, L.ldh, L.splits_x, (float*)(p.ws + L.part), p, s);
  if (e == cudaSuccess && (p.dwg || p.dwu))
    e = weight_gradients<T>(dtype, dg, du, x, L.ldd, L.ldh, L.splits, (float*)(p.ws + L.part), p, s);
  return e;
}

template <typename T>
static cudaError_t run_act(int dtype, int act, const Args& p, bool bwd, cudaStream_t s) {
  switch (act) {
    case FMS_ACT_SILU: return run<T, FMS_ACT_SILU>(dtype, p, bwd, s);
    case FMS_ACT_GELU: return run<T, FMS_ACT_GELU>(dtype, p, bwd, s);
    case FMS_ACT_GELU_TANH: return run<T, FMS_ACT_GELU_TANH>(dtype, p, bwd, s);
    default: return run<T, FMS_ACT_RELU>(dtype, p, bwd, s);
  }
}

}  // namespace glu
}  // namespace fms

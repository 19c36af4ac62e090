// The training path's kernels around its matrix products: dropout, and LayerNorm alone or behind dropout and a residual, forward and
// backward.  All of them are bound by memory traffic (or, for a few rows, by the launch): each pass reads its inputs once and writes
// its outputs once, and what can be made again is not stored: the mask (philox.cuh) and the sum in front of the norm.
//
// Everything works on units of eight consecutive columns: a 16-byte load in bf16, two in fp32, and one block of random bits.
// VEC: the rows allow that (columns a multiple of eight, aligned rows); otherwise a unit is read element by element, and unless its elements share
// random bits they are not neighbours but as far apart as there are units, so that the threads' loads are.
#include "tdb_internal.h"
#include "ptx_sm100.cuh"
#include "philox.cuh"
#include <algorithm>

namespace tdb {
using namespace ptx;

namespace {

__device__ __forceinline__ void to_type(float* p, float v) { *p = v; }
__device__ __forceinline__ void to_type(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// A unit as it comes from memory: eight elements of T.
template <typename T> struct Unit { uint4 v[sizeof(T) / 2]; };

template <typename T, bool VEC>
__device__ __forceinline__ Unit<T> load_unit(const T* p, int have, int step = 1) {
  Unit<T> u;
  if (VEC) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) u.v[i] = reinterpret_cast<const uint4*>(p)[i];
  } else {
    T* e = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) { if (i < have) e[i] = p[i * step]; else to_type(e + i, 0.f); }
  }
  return u;
}
// Eight elements as four pairs: two fp32 operations go by in one instruction, which is what keeps the kernels below bound by memory.
struct Eight {
  f32x2 v[4];
  __device__ __forceinline__ void unpack(float* f) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float2 h = halves(v[i]); f[2 * i] = h.x; f[2 * i + 1] = h.y; }
  }
  __device__ __forceinline__ void pack(const float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = pair(f[2 * i], f[2 * i + 1]);
  }
};
__device__ __forceinline__ f32x2 twice(float x) { return pair(x, x); }
__device__ __forceinline__ f32x2 times(f32x2 a, f32x2 b) { mul2(a, b); return a; }
__device__ __forceinline__ f32x2 plus(f32x2 a, f32x2 b) { add2(a, b); return a; }
__device__ __forceinline__ f32x2 fused(f32x2 a, f32x2 b, f32x2 c) { fma2(c, a, b); return c; }

__device__ __forceinline__ Eight eight(const Unit<float>& u) {
  Eight e;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    e.v[2 * i] = pair(__uint_as_float(u.v[i].x), __uint_as_float(u.v[i].y));
    e.v[2 * i + 1] = pair(__uint_as_float(u.v[i].z), __uint_as_float(u.v[i].w));
  }
  return e;
}
__device__ __forceinline__ Eight eight(const Unit<__nv_bfloat16>& u) {
  const uint32_t w[4] = {u.v[0].x, u.v[0].y, u.v[0].z, u.v[0].w};
  Eight e;
#pragma unroll
  for (int i = 0; i < 4; ++i) e.v[i] = pair(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  return e;
}
template <bool VEC>
__device__ __forceinline__ void store_unit(float* p, const Eight& x, int have, int step = 1) {
  float f[8];
  x.unpack(f);
  if (VEC) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      reinterpret_cast<uint4*>(p)[i] = make_uint4(__float_as_uint(f[4 * i]), __float_as_uint(f[4 * i + 1]), __float_as_uint(f[4 * i + 2]), __float_as_uint(f[4 * i + 3]));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) if (i < have) p[i * step] = f[i];
  }
}
template <bool VEC>
__device__ __forceinline__ void store_unit(__nv_bfloat16* p, const Eight& x, int have, int step = 1) {
  float f[8];
  x.unpack(f);
  if (VEC) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) if (i < have) p[i * step] = __float2bfloat16_rn(f[i]);
  }
}
// Eight weights of either type.
template <bool VEC>
__device__ __forceinline__ Eight load_weights(const void* w, int f32, int at, int have, int step) {
  return f32 ? eight(load_unit<float, VEC>(static_cast<const float*>(w) + at, have, step))
             : eight(load_unit<__nv_bfloat16, VEC>(static_cast<const __nv_bfloat16*>(w) + at, have, step));
}
__device__ __forceinline__ void drop8(Eight& x, const uint4& bits, uint32_t above, float scale) {
  float f[8];
  x.unpack(f);
  tdb::drop8(f, bits, above, scale);
  x.pack(f);
}

// ------------------------------------------------------------------------------------------------------------------ dropout
// y = what stays of x, scaled; its backward pass is the same of dy.  PER units to a thread, all loaded before the first is used.  16384 x 1024 bf16: bound by
// the generator's instructions (154 for eight elements, 69 % of the issue slots) before memory.
template <typename T, bool VEC, int PER>
__global__ void __launch_bounds__(256) dropout_kernel(const T* __restrict__ x, T* __restrict__ y, int64_t n, Dropout key) {
  const int64_t full = VEC ? n / 8 : 0, first = (int64_t)blockIdx.x * 256 * PER + threadIdx.x;
  const uint64_t seed = dropout_seed(key);
  const uint32_t above = dropout_above(key.drop);
  auto drop = [&](const Unit<T>& u, int64_t at) {
    Eight f = eight(u);
    drop8(f, philox((uint64_t)at, (uint64_t)key.offset, seed), above, key.scale);
    return f;
  };
  if (VEC && ((int64_t)blockIdx.x + 1) * 256 * PER <= full) {        // every unit of the block is a whole one
    Unit<T> u[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) u[i] = load_unit<T, true>(x + (first + 256 * i) * 8, 8);
#pragma unroll
    for (int i = 0; i < PER; ++i) store_unit<true>(y + (first + 256 * i) * 8, drop(u[i], first + 256 * i), 8);
    return;
  }
  for (int i = 0; i < PER; ++i) {
    const int64_t at = first + 256 * i;
    if (at * 8 >= n) return;
    const int have = (int)min((int64_t)8, n - at * 8);
    if (at < full) store_unit<true>(y + at * 8, drop(load_unit<T, true>(x + at * 8, 8), at), 8);
    else store_unit<false>(y + at * 8, drop(load_unit<T, false>(x + at * 8, have), at), have);
  }
}

// ---------------------------------------------------------------------------------------------------------------- LayerNorm
// The threads that share a row are `group` threads of the block (whole warps); sums over them, in a fixed order.
struct Group {
  int threads, lane, index;               // index: which of the block's groups
  float* shared;                          // two buffers of N floats for every warp of the block
  int flip;
};
// Every lane gets the warp's sum of each of N values (1, 2 or 4).  Lanes trade values on the way, so that N sums take N - 1 exchanges more than
// one, and not five times as many.
template <int N>
__device__ __forceinline__ void warp_sums(float* v) {
  const int lane = threadIdx.x & 31;
  if constexpr (N == 4) {
    const bool up = lane & 16;
    const float a = __shfl_xor_sync(0xffffffffu, up ? v[0] : v[2], 16), b = __shfl_xor_sync(0xffffffffu, up ? v[1] : v[3], 16);
    float w[2] = {(up ? v[2] : v[0]) + a, (up ? v[3] : v[1]) + b};
    const bool odd = lane & 8;
    const float c = __shfl_xor_sync(0xffffffffu, odd ? w[0] : w[1], 8);
    float s = (odd ? w[1] : w[0]) + c;
#pragma unroll
    for (int off = 4; off >= 1; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __shfl_sync(0xffffffffu, s, 8 * i);
  } else if constexpr (N == 2) {
    const bool up = lane & 16;
    const float a = __shfl_xor_sync(0xffffffffu, up ? v[0] : v[1], 16);
    float s = (up ? v[1] : v[0]) + a;
#pragma unroll
    for (int off = 8; off >= 1; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    v[0] = __shfl_sync(0xffffffffu, s, 0);
    v[1] = __shfl_sync(0xffffffffu, s, 16);
  } else {
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], off);
  }
}
// A warp each, the whole block, or a part of the block with a barrier of its own: those come to sixteen barriers a block, of the 64 that an
// SM has, which would leave it four blocks.
enum { A_WARP, THE_BLOCK, A_PART };
template <int N, int KIND = A_PART>
__device__ __forceinline__ void group_sum(Group& g, float* v) {
  warp_sums<N>(v);
  if (KIND == A_WARP || g.threads == 32) return;
  const int warps = g.threads / 32;
  // two buffers in turn: a warp that runs ahead writes the other one, and cannot come round again before the next barrier
  float* buf = g.shared + (g.index * 2 + g.flip) * N * warps;
  g.flip ^= 1;
  if (g.lane % 32 == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) buf[g.lane / 32 * N + i] = v[i];
  }
  if (KIND == THE_BLOCK) __syncthreads();
  else asm volatile("bar.sync %0, %1;" ::"r"(g.index + 1), "r"(g.threads) : "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = 0.f;
#pragma unroll 4
  for (int w = 0; w < warps; ++w) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += buf[w * N + i];
  }
}

// JOIN: LayerNorm(dropout(x) + res), DROP: with dropout in fact; otherwise LayerNorm(x).  U units of a row to a thread.
enum { ALONE = 0, JOIN = 1, JOIN_DROP = 2 };

struct NormParams : Norm {
  int group, w_f32;                                         // threads of a row
};

// Which columns unit c is: the first, how far apart, and how many there are.
struct Columns { int first, step, have; };
template <bool VEC, int MODE>
__device__ __forceinline__ Columns columns(int c, int units, int cols) {
  if (VEC) return {c * 8, 1, 8};
  if (MODE == JOIN_DROP) return {c * 8, 1, cols - c * 8};
  return {c, units, (cols - c + units - 1) / units};
}

// Eight elements of what the norm is taken of; `bits` are those that dropped them.
template <typename T, bool VEC, int MODE>
__device__ __forceinline__ Eight joined(const NormParams& p, const Unit<T>& x, const Unit<T>& r, int64_t row, int col, uint64_t seed, uint4& bits) {
  Eight f = eight(x);
  if (MODE == JOIN_DROP) {
    bits = dropout_bits<VEC>((uint64_t)row * p.cols + col, (uint64_t)p.drop.offset, seed);
    drop8(f, bits, dropout_above(p.drop.drop), p.drop.scale);
  }
  if (MODE != ALONE) {
    const Eight g = eight(r);
#pragma unroll
    for (int e = 0; e < 4; ++e) add2(f.v[e], g.v[e]);
  }
  return f;
}
// Elements behind the last column become zero.
__device__ __forceinline__ void cut(Eight& x, int have) {
  float f[8];
  x.unpack(f);
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = e < have ? f[e] : 0.f;
  x.pack(f);
}

// One group of threads to a row, the row in registers; mean first, then the deviations from it (the sum of squares alone would lose
// the variance of rows far from zero).
// A block has at most 8 rows of a warp, or one row of up to 512 threads.  With dropout the compiler is told how many blocks an SM is to
// hold: four where warps have rows of bf16 (9216 x 1024 17.5 us, 18.3 without), one where a block has the row (2000 x 4096 in fp32 24.5, 25.0
// without).  Warps with rows of fp32 are left without (0): 64 registers do not hold a row's two units in fp32, and 16384 x 1024 takes 49.4 us so bound and
// 43.7 without, 9216 x 1024 30.9 and 28.2, 9216 x 1020 59.5 and 55.9, 9216 x 768 18.6 both.  So is the norm alone: 16384 x 1024 takes 18.4 us so, 19.0
// with four and 20.0 with one.
constexpr int forward_threads(int kind, int mode) { return kind == A_WARP && mode == JOIN_DROP ? 256 : 512; }
template <typename T> constexpr int forward_blocks(int kind, int mode) { return mode != JOIN_DROP ? 0 : kind != A_WARP ? 1 : sizeof(T) == 2 ? 4 : 0; }

template <typename T, bool VEC, int MODE, int U, int KIND>
__global__ void __launch_bounds__(forward_threads(KIND, MODE), forward_blocks<T>(KIND, MODE)) norm_forward_kernel(const NormParams p) {
  extern __shared__ __align__(16) float shared[];
  Group g{p.group, (int)threadIdx.x % p.group, (int)threadIdx.x / p.group, shared, 0};
  const int groups = blockDim.x / p.group;
  const int64_t row = (int64_t)blockIdx.x * groups + g.index;
  if (row >= p.rows) return;                                // a whole group
  const int units = (p.cols + 7) / 8;
  const uint64_t seed = MODE == JOIN_DROP ? dropout_seed(p.drop) : 0;
  const T *x = (const T*)p.x + row * p.x_stride, *res = (const T*)p.res + row * p.res_stride;
  Unit<T> xu[U], ru[MODE == ALONE ? 1 : U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int c = g.lane + p.group * i;
    if (c < units) {
      const Columns at = columns<VEC, MODE>(c, units, p.cols);
      xu[i] = load_unit<T, VEC>(x + at.first, at.have, at.step);
      if (MODE != ALONE) ru[i] = load_unit<T, VEC>(res + at.first, at.have, at.step);
    }
  }
  Eight f[U];
  f32x2 sums = twice(0.f);
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int c = g.lane + p.group * i;
    if (c < units) {
      uint4 bits;
      f[i] = joined<T, VEC, MODE>(p, xu[i], ru[MODE == ALONE ? 0 : i], row, c * 8, seed, bits);
#pragma unroll
      for (int e = 0; e < 4; ++e) add2(sums, f[i].v[e]);     // zeros behind the last column
    }
  }
  float sum = halves(sums).x + halves(sums).y;
  group_sum<1, KIND>(g, &sum);
  const f32x2 mean = twice(sum / (float)p.cols), minus = twice(-halves(mean).x);
  f32x2 squares = twice(0.f);
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int c = g.lane + p.group * i;
    if (c < units) {
#pragma unroll
      for (int e = 0; e < 4; ++e) add2(f[i].v[e], minus);
      if (!VEC) cut(f[i], columns<VEC, MODE>(c, units, p.cols).have);
#pragma unroll
      for (int e = 0; e < 4; ++e) fma2(squares, f[i].v[e], f[i].v[e]);
    }
  }
  float sq = halves(squares).x + halves(squares).y;
  group_sum<1, KIND>(g, &sq);
  const float inv = rsqrtf(sq / (float)p.cols + p.eps);
  if (p.stats && g.lane == 0) *reinterpret_cast<float2*>(p.stats + 2 * row) = make_float2(halves(mean).x, inv);
  const f32x2 scale = twice(inv);
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int c = g.lane + p.group * i;
    if (c < units) {
      const Columns at = columns<VEC, MODE>(c, units, p.cols);
      const Eight w = load_weights<VEC>(p.w, p.w_f32, at.first, at.have, at.step);
      const Eight b = load_weights<VEC>(p.b, p.w_f32, at.first, at.have, at.step);
#pragma unroll
      for (int e = 0; e < 4; ++e) f[i].v[e] = fused(times(f[i].v[e], scale), w.v[e], b.v[e]);
      store_unit<VEC>((T*)p.y + row * p.cols + at.first, f[i], at.have, at.step);
    }
  }
}

// Backward.  With g = dy w and h = (z - mean) inv:  dz = (g - mean(g) - h mean(g h)) inv, dw = sum over rows of dy h, db of dy.
// A group of threads keeps the same columns for all its rows, so the weights and both column sums stay in registers up to 8192 columns (beyond, with four
// units to a thread, 372 to 1096 bytes of each thread spill), and the 2 R sums of the R rows that it takes at once share one exchange.  A block's sums
// go to `partial` and are added up by the kernel behind this one, in a fixed order: atomics would make two runs differ.
// VEC: what a thread will read is asked for some rounds ahead, by asynchronous copies into shared memory that no other thread touches, without barriers
// or registers for it.  As the ring holds: three rounds up to 4096 columns, where an SM has some 150 KB in flight while it computes; up to 8192 three in
// bf16, two in fp32 and one with a residual in fp32; beyond, two in bf16 and one with a residual, and in fp32 none: a round waits for its own copies.
constexpr int RING_BYTES = 192 * 1024;
template <typename T, int MODE, int U, int R>
__host__ __device__ constexpr int round_bytes() { return R * U * (MODE == ALONE ? 2 : 3) * (int)sizeof(Unit<T>); }     // of one thread
template <typename T, int MODE, int U, int R>
__host__ __device__ constexpr int rounds_ahead() { return RING_BYTES / 512 / round_bytes<T, MODE, U, R>() < 4 ? RING_BYTES / 512 / round_bytes<T, MODE, U, R>() : 4; }

template <typename T, bool VEC, int MODE, int U, int R>
__global__ void __launch_bounds__(512, 1) norm_backward_kernel(const NormParams p) {
  extern __shared__ __align__(16) float shared[];
  constexpr int STAGES = VEC ? rounds_ahead<T, MODE, U, R>() : 0, NT = MODE == ALONE ? 2 : 3, PIECES = (int)sizeof(Unit<T>) / 16;
  float* ring = shared;
  float* exchange = shared + STAGES * round_bytes<T, MODE, U, R>() / 4 * blockDim.x;
  Group g{p.group, (int)threadIdx.x % p.group, (int)threadIdx.x / p.group, exchange, 0};
  const int groups = blockDim.x / p.group, units = (p.cols + 7) / 8;
  const uint64_t seed = MODE == JOIN_DROP ? dropout_seed(p.drop) : 0;
  const uint32_t above = dropout_above(p.drop.drop);
  Eight w[U], dw[U], db[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int c = g.lane + p.group * i;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[i].v[e] = dw[i].v[e] = db[i].v[e] = twice(0.f);
    const Columns at = columns<VEC, MODE>(c, units, p.cols);
    if (c < units) w[i] = load_weights<VEC>(p.w, p.w_f32, at.first, at.have, at.step);
  }
  const float over = 1.f / (float)p.cols;
  const int64_t first = ((int64_t)blockIdx.x * groups + g.index) * R, stride = (int64_t)gridDim.x * groups * R;
  // tensor k of x, residual, dy
  auto source = [&](int k, int64_t row, int col) {
    return k == 0 ? (const T*)p.x + row * p.x_stride + col : k == NT - 1 ? (const T*)p.dy + row * p.dy_stride + col : (const T*)p.res + row * p.res_stride + col;
  };
  const uint32_t mine = (uint32_t)__cvta_generic_to_shared(ring) + threadIdx.x * 16, pitch = blockDim.x * 16;
  const uint32_t stage_bytes = NT * R * U * PIECES * pitch;
  auto slot = [&](uint32_t stage, int k, int r, int i, int piece) { return stage + (uint32_t)(((k * R + r) * U + i) * PIECES + piece) * pitch; };
  auto ask = [&](int64_t row0, uint32_t stage) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (row0 + r >= p.rows) break;
#pragma unroll
      for (int k = 0; k < NT; ++k) {
        const T* row = source(k, row0 + r, g.lane * 8);
#pragma unroll
        for (int i = 0; i < U; ++i)
          if (g.lane + p.group * i < units) {
#pragma unroll
            for (int piece = 0; piece < PIECES; ++piece)
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(slot(stage, k, r, i, piece)),
                           "l"(reinterpret_cast<const uint4*>(row + p.group * i * 8) + piece) : "memory");
          }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto unit = [&](uint32_t stage, int k, int64_t row, int r, int i) {
    const int c = g.lane + p.group * i;
    Unit<T> u;
    if constexpr (VEC) {
#pragma unroll
      for (int piece = 0; piece < PIECES; ++piece) {
        uint4& v = u.v[piece];
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(slot(stage, k, r, i, piece)) : "memory");
      }
    } else {
      const Columns at = columns<VEC, MODE>(c, units, p.cols);
      u = load_unit<T, false>(source(k, row, at.first), at.have, at.step);
    }
    return u;
  };
  auto stat = [&](int64_t row) { return *reinterpret_cast<const float2*>(p.stats + 2 * (row < p.rows ? row : p.rows - 1)); };
  if constexpr (VEC) {
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) ask(first + s * stride, mine + s * stage_bytes);
  }
  float2 soon[R];
#pragma unroll
  for (int r = 0; r < R; ++r) soon[r] = stat(first + r);
  uint32_t stage = mine, before = mine + (VEC ? STAGES - 1 : 0) * stage_bytes;      // of this round, and of the one before it
  for (int64_t row0 = first; row0 < p.rows; row0 += stride) {
    if constexpr (VEC) {
      ask(row0 + (STAGES - 1) * stride, before);
      asm volatile("cp.async.wait_group %0;" ::"n"(VEC ? STAGES - 1 : 0) : "memory");
    }
    float2 st[R];
    Eight h[R][U];
    float sums[2 * R];
    uint4 bits[R][U];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      st[r] = soon[r];
      soon[r] = stat(row0 + stride + r);
      f32x2 s1 = twice(0.f), s2 = twice(0.f);
      sums[2 * r] = sums[2 * r + 1] = 0.f;
      if (row0 + r >= p.rows) continue;
      const f32x2 minus = twice(-st[r].x), inv = twice(st[r].y);
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int c = g.lane + p.group * i;
        if (c >= units) continue;
        const Unit<T> xu = unit(stage, 0, row0 + r, r, i);
        h[r][i] = joined<T, VEC, MODE>(p, xu, MODE == ALONE ? xu : unit(stage, 1, row0 + r, r, i), row0 + r, c * 8, seed, bits[r][i]);
        const Eight d = eight(unit(stage, NT - 1, row0 + r, r, i));          // zeros behind the last column, and in w too
#pragma unroll
        for (int e = 0; e < 4; ++e) h[r][i].v[e] = times(plus(h[r][i].v[e], minus), inv);
        if (!VEC) cut(h[r][i], columns<VEC, MODE>(c, units, p.cols).have);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          fma2(dw[i].v[e], d.v[e], h[r][i].v[e]);
          add2(db[i].v[e], d.v[e]);
          const f32x2 gw = times(d.v[e], w[i].v[e]);
          add2(s1, gw);
          fma2(s2, gw, h[r][i].v[e]);
        }
      }
      sums[2 * r] = halves(s1).x + halves(s1).y;
      sums[2 * r + 1] = halves(s2).x + halves(s2).y;
    }
    group_sum<2 * R>(g, sums);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = row0 + r;
      if (row >= p.rows) break;
      const f32x2 c1 = twice(-sums[2 * r] * over), c2 = twice(-sums[2 * r + 1] * over), inv = twice(st[r].y);
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int c = g.lane + p.group * i;
        if (c >= units) continue;
        Eight d = eight(unit(stage, NT - 1, row, r, i));
#pragma unroll
        for (int e = 0; e < 4; ++e) d.v[e] = times(fused(h[r][i].v[e], c2, fused(d.v[e], w[i].v[e], c1)), inv);
        const Columns to = columns<VEC, MODE>(c, units, p.cols);
        const int64_t at = row * p.cols + to.first;
        if (MODE == ALONE && p.dx) store_unit<VEC>((T*)p.dx + at, d, to.have, to.step);
        if (MODE != ALONE && p.dres) store_unit<VEC>((T*)p.dres + at, d, to.have, to.step);
        if (MODE == JOIN_DROP && p.dx) {
          drop8(d, bits[r][i], above, p.drop.scale);
          store_unit<VEC>((T*)p.dx + at, d, to.have, to.step);
        }
      }
    }
    before = stage;
    if constexpr (VEC) stage = stage + stage_bytes == mine + STAGES * stage_bytes ? mine : stage + stage_bytes;
  }
  let_next_start();
  if (!p.partial) return;
  // the block's groups add up their column sums, one after the other, where the ring was
  if constexpr (VEC) asm volatile("cp.async.wait_group 0;" ::: "memory");
  float* sum = shared;
  for (int k = 0; k < groups; ++k) {
    __syncthreads();
    if (g.index != k) continue;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int c = g.lane + p.group * i;
      if (c >= units) continue;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float* a = sum + e * units + c;                     // by element, so that neighbouring threads meet different banks
        float* b = a + 8 * units;
        const float2 w2 = halves(dw[i].v[e / 2]), b2 = halves(db[i].v[e / 2]);
        *a = (k ? *a : 0.f) + (e % 2 ? w2.y : w2.x);
        *b = (k ? *b : 0.f) + (e % 2 ? b2.y : b2.x);
      }
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < p.cols; c += blockDim.x) {
    const int at = VEC || MODE == JOIN_DROP ? (c & 7) * units + (c >> 3) : c;
    p.partial[(int64_t)blockIdx.x * 2 * p.cols + c] = sum[at];
    p.partial[((int64_t)blockIdx.x * 2 + 1) * p.cols + c] = sum[8 * units + at];
  }
}

// [blocks, 2, cols] -> dw, db.  32 columns and 16 shares of the blocks to a thread block.
__global__ void __launch_bounds__(512) norm_weights_kernel(const float* __restrict__ partial, int blocks, int cols, int w_f32, void* dw, void* db) {
  __shared__ float part[16][33];
  const int lane = threadIdx.x % 32, share = threadIdx.x / 32, c = blockIdx.x * 32 + lane;
  wait_for_stream();
  float s = 0.f;
  if (c < 2 * cols)
    for (int b = share; b < blocks; b += 16) s += *reinterpret_cast<const volatile float*>(partial + (int64_t)b * 2 * cols + c);
  part[share][lane] = s;
  __syncthreads();
  if (share || c >= 2 * cols) return;
  s = 0.f;
#pragma unroll
  for (int k = 0; k < 16; ++k) s += part[k][lane];
  void* out = c < cols ? dw : db;
  const int at = c < cols ? c : c - cols;
  if (!out) return;
  if (w_f32) static_cast<float*>(out)[at] = s;
  else static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(s);
}

// Threads of a row, and units of a thread: U at most.
int group_threads(int units, int u) { return ((units + u - 1) / u + 31) / 32 * 32; }

template <typename T, bool VEC, int MODE>
int norm_forward(NormParams p, cudaStream_t s) {
  const int units = (p.cols + 7) / 8;
  int sms = 0;
  if (const int rc = device_sms(&sms)) return rc;
  auto run = [&](auto kernel, int u) {
    p.group = group_threads(units, u);
    const int groups = p.group == 32 && p.rows >= 16 * sms ? 8 : 1;       // few rows: one to a block, so that they spread over the SMs
    const int64_t blocks = (p.rows + groups - 1) / groups;
    kernel<<<(unsigned)blocks, groups * p.group, p.group == 32 ? 0 : 2 * (p.group / 32) * sizeof(float), s>>>(p);
    return cuda_fail(cudaGetLastError(), "norm launch");
  };
  if (units <= 32) return run(norm_forward_kernel<T, VEC, MODE, 1, A_WARP>, 1);
  if (units <= 64) return run(norm_forward_kernel<T, VEC, MODE, 2, A_WARP>, 2);
  if (units <= 96) return run(norm_forward_kernel<T, VEC, MODE, 3, A_WARP>, 3);
  if (units <= 128) return run(norm_forward_kernel<T, VEC, MODE, 4, A_WARP>, 4);
  return run(norm_forward_kernel<T, VEC, MODE, 4, THE_BLOCK>, 4);
}

struct BackwardShape { int units_each, rows_each, group, groups, blocks; };

// Blocks of up to 512 threads, one to an SM, with several rows in flight to each of their groups; fewer of both where that would leave
// SMs without rows.
BackwardShape backward_shape(int64_t rows, int cols, int most_rows, int sms) {
  BackwardShape b;
  const int units = (cols + 7) / 8;
  b.units_each = units <= 512 ? 1 : units <= 1024 ? 2 : 4;
  b.group = group_threads(units, b.units_each);
  b.groups = 512 / b.group > 1 ? 512 / b.group : 1;
  b.rows_each = b.units_each == 1 && rows >= (int64_t)most_rows * b.groups * sms ? most_rows : 1;
  const int64_t each = (rows + sms - 1) / sms;
  if (b.rows_each == 1 && each < b.groups) b.groups = (int)each;
  const int64_t most = (rows + b.groups * b.rows_each - 1) / (b.groups * b.rows_each);
  b.blocks = (int)(most < sms ? most : sms);
  return b;
}

template <typename T, bool VEC, int MODE>
int norm_backward(NormParams p, cudaStream_t s) {
  constexpr int R = VEC && sizeof(T) == 2 ? 2 : 1;
  int sms = 0, rc;
  if ((rc = device_sms(&sms))) return rc;
  const BackwardShape b = backward_shape(p.rows, p.cols, R, sms);
  const int units = (p.cols + 7) / 8;
  p.group = b.group;
  auto run = [&](auto kernel, int r, int ring) -> int {       // ring: bytes of one thread
    const int exchange = b.group == 32 ? 0 : b.groups * 2 * 2 * r * (b.group / 32) * 4, threads = b.groups * b.group;
    const int bytes = std::max(VEC ? ring * threads + exchange : exchange, (VEC ? 0 : exchange) + (p.partial ? 16 * units * 4 : 0));
    if (bytes > 48 * 1024)
      if (const int rc = opt_in_smem(reinterpret_cast<const void*>(kernel), 227 * 1024)) return rc;
    kernel<<<b.blocks, threads, bytes, s>>>(p);
    return cuda_fail(cudaGetLastError(), "norm backward launch");
  };
#define TDB_BACKWARD(U, R) run(norm_backward_kernel<T, VEC, MODE, U, R>, R, rounds_ahead<T, MODE, U, R>() * round_bytes<T, MODE, U, R>())
  if (b.rows_each == R && R > 1) rc = TDB_BACKWARD(1, R);
  else if (b.units_each == 1) rc = TDB_BACKWARD(1, 1);
  else if (b.units_each == 2) rc = TDB_BACKWARD(2, 1);
  else rc = TDB_BACKWARD(4, 1);
#undef TDB_BACKWARD
  if (rc || !p.partial) return rc;
  return cuda_fail(launch_early(norm_weights_kernel, dim3((2 * p.cols + 31) / 32), 512, 0, s, (const float*)p.partial, b.blocks, p.cols, p.w_f32, p.dw, p.db),
                   "norm weights launch");
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename T>
bool vectors(const NormParams& p) {
  const int per = 16 / (int)sizeof(T);
  return p.cols % 8 == 0 && p.x_stride % per == 0 && p.res_stride % per == 0 && p.dy_stride % per == 0 && aligned(p.x) && aligned(p.res) &&
         aligned(p.dy) && aligned(p.y) && aligned(p.dx) && aligned(p.dres) && aligned(p.w) && aligned(p.b);
}

template <typename T>
int forward_t(const NormParams& p, int mode, cudaStream_t s) {
  if (vectors<T>(p))
    return mode == ALONE ? norm_forward<T, true, ALONE>(p, s) : mode == JOIN ? norm_forward<T, true, JOIN>(p, s) : norm_forward<T, true, JOIN_DROP>(p, s);
  return mode == ALONE ? norm_forward<T, false, ALONE>(p, s) : mode == JOIN ? norm_forward<T, false, JOIN>(p, s) : norm_forward<T, false, JOIN_DROP>(p, s);
}
template <typename T>
int backward_t(const NormParams& p, int mode, cudaStream_t s) {
  if (vectors<T>(p))
    return mode == ALONE ? norm_backward<T, true, ALONE>(p, s) : mode == JOIN ? norm_backward<T, true, JOIN>(p, s) : norm_backward<T, true, JOIN_DROP>(p, s);
  return mode == ALONE ? norm_backward<T, false, ALONE>(p, s) : mode == JOIN ? norm_backward<T, false, JOIN>(p, s) : norm_backward<T, false, JOIN_DROP>(p, s);
}

NormParams params(const Norm& n) {
  NormParams p{n, 0, n.w_dtype == TDB_DTYPE_F32};
  if (!n.res) p.res_stride = 0;
  if (!n.dy) p.dy_stride = 0;
  return p;
}
int mode_of(const Norm& n) { return !n.res ? ALONE : n.drop.drop ? JOIN_DROP : JOIN; }

}  // namespace
}  // namespace tdb

using namespace tdb;

extern "C" {

int tdb_dropout(const void* x, void* y, int64_t n, int dtype, const Dropout* d, void* stream) {
  if (n == 0) return TDB_OK;
  int sms = 0;
  if (const int rc = device_sms(&sms)) return rc;
  const int64_t units = (n + 7) / 8;
  const bool vec = aligned(x) && aligned(y), many = vec && units >= (int64_t)sms * 2048;
  const int64_t per = 256 * (many ? 4 : 1);
  const unsigned blocks = (unsigned)((units + per - 1) / per);
  cudaStream_t s = (cudaStream_t)stream;
#define TDB_DROPOUT(T)                                                                                  \
  (many ? dropout_kernel<T, true, 4> : vec ? dropout_kernel<T, true, 1> : dropout_kernel<T, false, 1>)  \
      <<<blocks, 256, 0, s>>>((const T*)x, (T*)y, n, *d)
  if (dtype == TDB_DTYPE_F32) TDB_DROPOUT(float);
  else TDB_DROPOUT(__nv_bfloat16);
#undef TDB_DROPOUT
  return cuda_fail(cudaGetLastError(), "dropout launch");
}

int tdb_norm_forward(const Norm* n, int dtype, void* stream) {
  if (n->rows == 0) return TDB_OK;
  const NormParams p = params(*n);
  return dtype == TDB_DTYPE_F32 ? forward_t<float>(p, mode_of(*n), (cudaStream_t)stream) : forward_t<__nv_bfloat16>(p, mode_of(*n), (cudaStream_t)stream);
}

int64_t tdb_norm_partial_floats(int64_t rows, int cols) {
  int sms = 0;
  if (rows == 0 || device_sms(&sms)) return 0;
  return (int64_t)sms * 2 * cols;                            // backward_shape: no more blocks than SMs
}

int tdb_norm_backward(const Norm* n, int dtype, void* stream) {
  if (n->rows == 0) return TDB_OK;
  const NormParams p = params(*n);
  return dtype == TDB_DTYPE_F32 ? backward_t<float>(p, mode_of(*n), (cudaStream_t)stream) : backward_t<__nv_bfloat16>(p, mode_of(*n), (cudaStream_t)stream);
}

}  // extern "C"

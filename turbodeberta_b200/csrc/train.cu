// The training path's kernels around its matrix products: dropout, and LayerNorm alone or behind dropout and a residual, forward and
// backward.  All of them are bound by memory traffic (or, for a few rows, by the launch): each pass reads its inputs once and writes
// its outputs once, and what can be made again is not stored: the mask (philox.cuh) and the sum in front of the norm.
//
// Everything works on units of eight consecutive columns: a 16-byte load in bf16, two in fp32, and one block of random bits.
// VEC: the rows allow that (columns a multiple of eight, aligned rows); otherwise a unit is read element by element.
#include "tdb_internal.h"
#include "philox.cuh"

namespace tdb {

namespace {

__device__ __forceinline__ void to_type(float* p, float v) { *p = v; }
__device__ __forceinline__ void to_type(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// A unit as it comes from memory: eight elements of T.
template <typename T> struct Unit { uint4 v[sizeof(T) / 2]; };

template <typename T, bool VEC>
__device__ __forceinline__ Unit<T> load_unit(const T* p, int have) {
  Unit<T> u;
  if (VEC) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) u.v[i] = reinterpret_cast<const uint4*>(p)[i];
  } else {
    T* e = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) { if (i < have) e[i] = p[i]; else to_type(e + i, 0.f); }
  }
  return u;
}
__device__ __forceinline__ void unpack(const Unit<float>& u, float* f) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    f[4 * i] = __uint_as_float(u.v[i].x); f[4 * i + 1] = __uint_as_float(u.v[i].y);
    f[4 * i + 2] = __uint_as_float(u.v[i].z); f[4 * i + 3] = __uint_as_float(u.v[i].w);
  }
}
__device__ __forceinline__ void unpack(const Unit<__nv_bfloat16>& u, float* f) {
  const uint32_t w[4] = {u.v[0].x, u.v[0].y, u.v[0].z, u.v[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
template <bool VEC>
__device__ __forceinline__ void store_unit(float* p, const float* f, int have) {
  if (VEC) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      reinterpret_cast<uint4*>(p)[i] = make_uint4(__float_as_uint(f[4 * i]), __float_as_uint(f[4 * i + 1]), __float_as_uint(f[4 * i + 2]), __float_as_uint(f[4 * i + 3]));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) if (i < have) p[i] = f[i];
  }
}
template <bool VEC>
__device__ __forceinline__ void store_unit(__nv_bfloat16* p, const float* f, int have) {
  if (VEC) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 t = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&t);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) if (i < have) p[i] = __float2bfloat16_rn(f[i]);
  }
}
// Eight weights of either type.
__device__ __forceinline__ void load_weights(const void* w, int f32, int64_t at, int have, float* f) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    f[i] = i < have ? (f32 ? static_cast<const float*>(w)[at + i] : __bfloat162float(static_cast<const __nv_bfloat16*>(w)[at + i])) : 0.f;
}

// ------------------------------------------------------------------------------------------------------------------ dropout
// y = what stays of x, scaled; its backward pass is the same of dy.  PER units to a thread, all loaded before the first is used.
template <typename T, bool VEC, int PER>
__global__ void __launch_bounds__(256) dropout_kernel(const T* __restrict__ x, T* __restrict__ y, int64_t n, Dropout key) {
  const int64_t units = (n + 7) / 8, first = ((int64_t)blockIdx.x * 256 * PER) + threadIdx.x;
  const uint64_t seed = dropout_seed(key);
  Unit<T> u[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int64_t at = first + 256 * i;
    if (at >= units) break;
    const int have = (int)min((int64_t)8, n - at * 8);
    u[i] = VEC && have == 8 ? load_unit<T, true>(x + at * 8, 8) : load_unit<T, false>(x + at * 8, have);
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int64_t at = first + 256 * i;
    if (at >= units) break;
    const int have = (int)min((int64_t)8, n - at * 8);
    float f[8];
    unpack(u[i], f);
    drop8(f, staying(philox((uint64_t)at, (uint64_t)key.offset, seed), key.drop), key.scale);
    if (VEC && have == 8) store_unit<true>(y + at * 8, f, 8);
    else store_unit<false>(y + at * 8, f, have);
  }
}

// ---------------------------------------------------------------------------------------------------------------- LayerNorm
// The threads that share a row are `group` threads of the block (whole warps); sums over them, in a fixed order.
struct Group {
  int threads, lane, index;               // index: which of the block's groups
  float* shared;                          // 2 buffers of 32 floats for every value that is summed at once
  int flip;
};
__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
  return x;
}
template <int N>
__device__ __forceinline__ void group_sum(Group& g, float* v) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
  if (g.threads == 32) return;
  const int warps = g.threads / 32;
  // two buffers in turn: a warp that runs ahead writes the other one, and cannot come round again before the next barrier
  float* buf = g.shared + (g.index * 2 + g.flip) * N * warps;
  g.flip ^= 1;
  if (g.lane % 32 == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) buf[i * warps + g.lane / 32] = v[i];
  }
  asm volatile("bar.sync %0, %1;" ::"r"(g.index + 1), "r"(g.threads) : "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float s = 0.f;
    for (int w = 0; w < warps; ++w) s += buf[i * warps + w];
    v[i] = s;
  }
}

// JOIN: LayerNorm(dropout(x) + res), DROP: with dropout in fact; otherwise LayerNorm(x).  U units of a row to a thread.
enum { ALONE = 0, JOIN = 1, JOIN_DROP = 2 };

struct NormParams : Norm {
  int group, w_f32;                                         // threads of a row
};

template <typename T, bool VEC, int MODE>
__device__ __forceinline__ void joined(const NormParams& p, const Unit<T>& x, const Unit<T>& r, int64_t row, int col, uint64_t seed, float* f, uint32_t& stay) {
  unpack(x, f);
  if (MODE == JOIN_DROP) {
    stay = staying(dropout_bits<VEC>((uint64_t)row * p.cols + col, (uint64_t)p.drop.offset, seed), p.drop.drop);
    drop8(f, stay, p.drop.scale);
  }
  if (MODE != ALONE) {
    float g[8];
    unpack(r, g);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] += g[e];
  }
}

// One group of threads to a row, the row in registers; mean first, then the deviations from it (the sum of squares alone would lose
// the variance of rows far from zero).
template <typename T, bool VEC, int MODE, int U>
__global__ void __launch_bounds__(512) norm_forward_kernel(const NormParams p) {
  extern __shared__ float shared[];
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
      xu[i] = load_unit<T, VEC>(x + c * 8, p.cols - c * 8);
      if (MODE != ALONE) ru[i] = load_unit<T, VEC>(res + c * 8, p.cols - c * 8);
    }
  }
  float f[U][8], sum = 0.f;
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int c = g.lane + p.group * i;
    if (c < units) {
      uint32_t stay;
      joined<T, VEC, MODE>(p, xu[i], ru[MODE == ALONE ? 0 : i], row, c * 8, seed, f[i], stay);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += VEC || c * 8 + e < p.cols ? f[i][e] : 0.f;
    }
  }
  group_sum<1>(g, &sum);
  const float mean = sum / (float)p.cols;
  float sq = 0.f;
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int c = g.lane + p.group * i;
    if (c < units) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        f[i][e] -= mean;
        sq = VEC || c * 8 + e < p.cols ? fmaf(f[i][e], f[i][e], sq) : sq;
      }
    }
  }
  group_sum<1>(g, &sq);
  const float inv = rsqrtf(sq / (float)p.cols + p.eps);
  if (p.stats && g.lane == 0) *reinterpret_cast<float2*>(p.stats + 2 * row) = make_float2(mean, inv);
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int c = g.lane + p.group * i;
    if (c < units) {
      float w[8], b[8];
      load_weights(p.w, p.w_f32, c * 8, p.cols - c * 8, w);
      load_weights(p.b, p.w_f32, c * 8, p.cols - c * 8, b);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[i][e] = fmaf(f[i][e] * inv, w[e], b[e]);
      store_unit<VEC>((T*)p.y + row * p.cols + c * 8, f[i], p.cols - c * 8);
    }
  }
}

// Backward.  With g = dy w and h = (z - mean) inv:  dz = (g - mean(g) - h mean(g h)) inv, dw = sum over rows of dy h, db of dy.
// A group of threads keeps the same columns for all its rows, so the weights and both column sums stay in registers; R rows are in
// flight at once, and their 2 R sums share one exchange.  The sums of a block go to `partial` and are added up by the kernel behind
// this one, in a fixed order: atomics would make two runs differ.
template <typename T, bool VEC, int MODE, int U, int R>
__global__ void __launch_bounds__(512, 1) norm_backward_kernel(const NormParams p) {
  extern __shared__ float shared[];
  Group g{p.group, (int)threadIdx.x % p.group, (int)threadIdx.x / p.group, shared, 0};
  const int groups = blockDim.x / p.group, units = (p.cols + 7) / 8;
  const uint64_t seed = MODE == JOIN_DROP ? dropout_seed(p.drop) : 0;
  float w[U][8], dw[U][8], db[U][8];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int c = g.lane + p.group * i;
#pragma unroll
    for (int e = 0; e < 8; ++e) w[i][e] = dw[i][e] = db[i][e] = 0.f;
    if (c < units) load_weights(p.w, p.w_f32, c * 8, p.cols - c * 8, w[i]);
  }
  const float over = 1.f / (float)p.cols;
  for (int64_t row0 = ((int64_t)blockIdx.x * groups + g.index) * R; row0 < p.rows; row0 += (int64_t)gridDim.x * groups * R) {
    Unit<T> xu[R][U], ru[MODE == ALONE ? 1 : R][U], du[R][U];
    float2 st[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = min(row0 + r, p.rows - 1);        // a row behind the last one is the last one again, and counts for nothing
      st[r] = *reinterpret_cast<const float2*>(p.stats + 2 * row);
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int c = g.lane + p.group * i;
        if (c < units) {
          xu[r][i] = load_unit<T, VEC>((const T*)p.x + row * p.x_stride + c * 8, p.cols - c * 8);
          if (MODE != ALONE) ru[r][i] = load_unit<T, VEC>((const T*)p.res + row * p.res_stride + c * 8, p.cols - c * 8);
          du[r][i] = load_unit<T, VEC>((const T*)p.dy + row * p.dy_stride + c * 8, p.cols - c * 8);
        }
      }
    }
    float h[R][U][8], sums[2 * R];
    uint32_t stay[R][U];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool real = row0 + r < p.rows;
      sums[2 * r] = sums[2 * r + 1] = 0.f;
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int c = g.lane + p.group * i;
        if (c >= units) continue;
        joined<T, VEC, MODE>(p, xu[r][i], ru[MODE == ALONE ? 0 : r][i], row0 + r, c * 8, seed, h[r][i], stay[r][i]);
        float d[8];
        unpack(du[r][i], d);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool in = real && (VEC || c * 8 + e < p.cols);
          h[r][i][e] = (h[r][i][e] - st[r].x) * st[r].y;
          dw[i][e] = in ? fmaf(d[e], h[r][i][e], dw[i][e]) : dw[i][e];
          db[i][e] = in ? db[i][e] + d[e] : db[i][e];
          const float gw = d[e] * w[i][e];                  // zero behind the last column
          sums[2 * r] += VEC || in ? gw : 0.f;
          sums[2 * r + 1] = VEC || in ? fmaf(gw, h[r][i][e], sums[2 * r + 1]) : sums[2 * r + 1];
        }
      }
    }
    group_sum<2 * R>(g, sums);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = row0 + r;
      if (row >= p.rows) break;
      const float c1 = sums[2 * r] * over, c2 = sums[2 * r + 1] * over;
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int c = g.lane + p.group * i;
        if (c >= units) continue;
        float d[8];
        unpack(du[r][i], d);
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] = (fmaf(d[e], w[i][e], -c1) - h[r][i][e] * c2) * st[r].y;
        const int64_t at = row * p.cols + c * 8;
        if (MODE == ALONE && p.dx) store_unit<VEC>((T*)p.dx + at, d, p.cols - c * 8);
        if (MODE != ALONE && p.dres) store_unit<VEC>((T*)p.dres + at, d, p.cols - c * 8);
        if (MODE == JOIN_DROP && p.dx) {
          drop8(d, stay[r][i], p.drop.scale);
          store_unit<VEC>((T*)p.dx + at, d, p.cols - c * 8);
        }
      }
    }
  }
  let_next_start();
  if (!p.partial) return;
  // the block's groups add up their column sums, one after the other
  float* sum = shared + (p.group == 32 ? 0 : groups * 2 * 2 * R * (p.group / 32));
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
        *a = k ? *a + dw[i][e] : dw[i][e];
        *b = k ? *b + db[i][e] : db[i][e];
      }
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < p.cols; c += blockDim.x) {
    const int at = (c & 7) * units + (c >> 3);
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
    const int groups = p.rows >= 16 * sms ? max(1, 128 / p.group) : 1;      // few rows: one per block, so that they spread over the SMs
    const int64_t blocks = (p.rows + groups - 1) / groups;
    kernel<<<(unsigned)blocks, groups * p.group, groups * 2 * (p.group / 32) * sizeof(float), s>>>(p);
    return cuda_fail(cudaGetLastError(), "norm launch");
  };
  if (units <= 32) return run(norm_forward_kernel<T, VEC, MODE, 1>, 1);
  if (units <= 64) return run(norm_forward_kernel<T, VEC, MODE, 2>, 2);
  if (units <= 96) return run(norm_forward_kernel<T, VEC, MODE, 3>, 3);
  return run(norm_forward_kernel<T, VEC, MODE, 4>, 4);
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
  constexpr int R = !VEC ? 1 : sizeof(T) == 2 ? 4 : 2;       // what the registers hold
  int sms = 0, rc;
  if ((rc = device_sms(&sms))) return rc;
  const BackwardShape b = backward_shape(p.rows, p.cols, R, sms);
  const int units = (p.cols + 7) / 8;
  p.group = b.group;
  auto run = [&](auto kernel, int r) -> int {
    const int exchange = b.group == 32 ? 0 : b.groups * 2 * 2 * r * (b.group / 32);
    const int bytes = (exchange + (p.partial ? 16 * units : 0)) * (int)sizeof(float);
    if (bytes > 48 * 1024)
      if (const int rc = opt_in_smem(reinterpret_cast<const void*>(kernel), 227 * 1024)) return rc;
    kernel<<<b.blocks, b.groups * b.group, bytes, s>>>(p);
    return cuda_fail(cudaGetLastError(), "norm backward launch");
  };
  if (b.rows_each == R && R > 1) rc = run(norm_backward_kernel<T, VEC, MODE, 1, R>, R);
  else if (b.units_each == 1) rc = run(norm_backward_kernel<T, VEC, MODE, 1, 1>, 1);
  else if (b.units_each == 2) rc = run(norm_backward_kernel<T, VEC, MODE, 2, 1>, 1);
  else rc = run(norm_backward_kernel<T, VEC, MODE, 4, 1>, 1);
  if (rc || !p.partial) return rc;
  return cuda_fail(launch_early(norm_weights_kernel, dim3((2 * p.cols + 31) / 32), 512, 0, s, (const float*)p.partial, b.blocks, p.cols, p.w_f32, p.dw, p.db),
                   "norm weights launch");
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename T>
bool vectors(const NormParams& p) {
  const int per = 16 / (int)sizeof(T);
  return p.cols % 8 == 0 && p.x_stride % per == 0 && p.res_stride % per == 0 && p.dy_stride % per == 0 && aligned(p.x) && aligned(p.res) &&
         aligned(p.dy) && aligned(p.y) && aligned(p.dx) && aligned(p.dres);
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

// Low-rank adapters of many requests beside a shared projection, for any type and size:
//   y[t] = x[t] W^T + b + s_a (x[t] A_a^T) B_a^T          a: the adapter of row t (none: the shared part alone)
// and coming back, with W frozen,  u[t] = s_a dy[t] B_a,  dx = dy W + u A_a,  dA_a = sum u^T x,  dB_a = sum dy^T h,  h[t] = s_a x[t] A_a^T.
//
// These are the kernels beside the shared product: `shrink` makes h or u, `expand` adds their part to the product and writes the result,
// `gather` sums the gradients.  A tile's rows may belong to several adapters: it takes one adapter after the other, with zeros in the
// place of other rows, so requests need not be sorted and a tile of one adapter costs nothing extra.
#include "tdb_internal.h"
#include "lora.cuh"
#include <algorithm>

namespace tdb {

namespace {

__device__ __forceinline__ float value(const float* p) { return *p; }
__device__ __forceinline__ float value(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

constexpr int TILE = 16, COLS = 128, STEP = 64;

// One matrix per adapter, factor j of column c at j * sj + c * sc.
template <typename T> struct Factors { const T* p; int64_t each, sj, sc; };

// The rows' adapters in shared memory; whether `row` is the first of its adapter in the tile.
__device__ __forceinline__ void load_ids(int* ids, const LoraRows& rows, int64_t t0, int count) {
  if ((int)threadIdx.x < count) ids[threadIdx.x] = t0 + threadIdx.x < rows.rows ? adapter_of(rows, t0 + threadIdx.x) : -1;
  __syncthreads();
}
__device__ __forceinline__ bool is_first(const int* ids, int row) {
  for (int i = 0; i < row; ++i)
    if (ids[i] == ids[row]) return false;
  return true;
}

// h[z][t][j] = s_a sum over this share of the columns of x[t][c] F_a(j, c).  A block: 16 rows, 64 factors.
template <typename T>
__global__ void __launch_bounds__(256) shrink_kernel(const T* __restrict__ x, int64_t stride, int cols, Factors<T> f, int rank, LoraRows rows,
                                                     int share, float* __restrict__ h) {
  __shared__ int ids[TILE];
  __shared__ float xs[TILE][STEP + 1], fs[STEP][64 + 1];
  const int64_t t0 = (int64_t)blockIdx.x * TILE;
  const int j0 = blockIdx.y * 64, jn = min(64, rank - j0), c_begin = blockIdx.z * share, c_end = min(cols, c_begin + share);
  const int row = threadIdx.x / 16, jt = threadIdx.x % 16;              // a thread: one row, factors jt, jt + 16, ...
  load_ids(ids, rows, t0, TILE);
  float out[4] = {0.f, 0.f, 0.f, 0.f};
  for (int first = 0; first < TILE; ++first) {
    const int a = ids[first];
    if (a < 0 || !is_first(ids, first)) continue;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int c0 = c_begin; c0 < c_end; c0 += STEP) {
      __syncthreads();
      for (int e = threadIdx.x; e < TILE * STEP; e += 256) {
        const int r = e / STEP, c = e % STEP;
        xs[r][c] = ids[r] == a && c0 + c < c_end ? value(x + (t0 + r) * stride + c0 + c) : 0.f;
      }
      const T* fa = f.p + a * f.each;
      for (int e = threadIdx.x; e < STEP * 64; e += 256) {
        const int j = f.sj == 1 ? e % 64 : e / STEP, c = f.sj == 1 ? e / 64 : e % STEP;
        fs[c][j] = j < jn && c0 + c < c_end ? value(fa + (j0 + j) * f.sj + (int64_t)(c0 + c) * f.sc) : 0.f;
      }
      __syncthreads();
      if (ids[row] == a) {
        for (int c = 0; c < STEP; ++c) {
          const float v = xs[row][c];
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[i] = fmaf(v, fs[c][jt + 16 * i], acc[i]);
        }
      }
    }
    if (ids[row] == a) {
#pragma unroll
      for (int i = 0; i < 4; ++i) out[i] = acc[i] * scaling_of(rows, a);
    }
  }
  if (t0 + row >= rows.rows) return;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (jt + 16 * i < jn) h[((int64_t)blockIdx.z * rows.rows + t0 + row) * rank + j0 + jt + 16 * i] = out[i];
}

// y[t][c] = base[t][c] + bias[c] + sum over j of h[t][j] F_a(j, c), one rounding.  A block: 16 rows, 128 columns, one to a thread.
template <typename T>
__global__ void __launch_bounds__(COLS) expand_kernel(const float* base, const T* __restrict__ bias, const float* __restrict__ h, int shares,
                                                      int rank, Factors<T> f, LoraRows rows, int cols, T* y) {     // base may be y
  __shared__ int ids[TILE];
  __shared__ float hs[TILE][64];
  const int64_t t0 = (int64_t)blockIdx.x * TILE;
  const int c = blockIdx.y * COLS + threadIdx.x;
  load_ids(ids, rows, t0, TILE);
  float acc[TILE];
#pragma unroll
  for (int r = 0; r < TILE; ++r) acc[r] = 0.f;
  for (int j0 = 0; j0 < rank; j0 += 64) {
    const int jn = min(64, rank - j0);
    __syncthreads();
    for (int e = threadIdx.x; e < TILE * 64; e += COLS) {
      const int r = e / 64, j = e % 64;
      float s = 0.f;
      if (j < jn && ids[r] >= 0)
        for (int z = 0; z < shares; ++z) s += h[((int64_t)z * rows.rows + t0 + r) * rank + j0 + j];
      hs[r][j] = s;
    }
    __syncthreads();
    if (c >= cols) continue;
    for (int first = 0; first < TILE; ++first) {
      const int a = ids[first];
      if (a < 0 || !is_first(ids, first)) continue;
      const T* fa = f.p + a * f.each + j0 * f.sj + (int64_t)c * f.sc;
      bool mine[TILE];
#pragma unroll
      for (int r = 0; r < TILE; ++r) mine[r] = ids[r] == a;
      for (int j = 0; j < jn; ++j) {
        const float v = value(fa + j * f.sj);
#pragma unroll
        for (int r = 0; r < TILE; ++r) acc[r] = mine[r] ? fmaf(hs[r][j], v, acc[r]) : acc[r];
      }
    }
  }
  if (c >= cols) return;
  const float b = bias ? value(bias + c) : 0.f;
#pragma unroll
  for (int r = 0; r < TILE; ++r)
    if (t0 + r < rows.rows) put(y + (t0 + r) * cols + c, base[(t0 + r) * cols + c] + b + acc[r]);
}

// part[z][a][j][c] = sum over this share of the rows t of adapter a of v[t][j] x[t][c].  A block: one adapter, 16 factors, 128 columns.
template <typename T>
__global__ void __launch_bounds__(COLS) gather_kernel(const T* __restrict__ x, int64_t stride, int cols, const float* __restrict__ v, int shares, int rank,
                                                      LoraRows rows, int64_t share, int j_blocks, float* __restrict__ part) {
  __shared__ int ids[32];
  __shared__ float vs[32][16];
  const int a = blockIdx.y / j_blocks, j0 = blockIdx.y % j_blocks * 16, jn = min(16, rank - j0), c = blockIdx.x * COLS + threadIdx.x;
  const int64_t begin = blockIdx.z * share, end = min(rows.rows, begin + share);
  float acc[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) acc[j] = 0.f;
  for (int64_t t0 = begin; t0 < end; t0 += 32) {
    const int count = (int)min((int64_t)32, end - t0);
    __syncthreads();
    int mine = 0;
    if (threadIdx.x < 32) ids[threadIdx.x] = mine = (int)threadIdx.x < count && adapter_of(rows, t0 + threadIdx.x) == a;
    if (!__syncthreads_or(mine)) continue;
    for (int e = threadIdx.x; e < 32 * 16; e += COLS) {
      const int r = e / 16, j = e % 16;
      float s = 0.f;
      if (ids[r] && j < jn)
        for (int z = 0; z < shares; ++z) s += v[((int64_t)z * rows.rows + t0 + r) * rank + j0 + j];
      vs[r][j] = s;
    }
    __syncthreads();
    if (c < cols) {
#pragma unroll 8
      for (int r = 0; r < 32; ++r) {
        if (!ids[r]) continue;
        const float xv = value(x + (t0 + r) * stride + c);
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[j] = fmaf(vs[r][j], xv, acc[j]);
      }
    }
  }
  if (c >= cols) return;
  const int n = gridDim.y / j_blocks;
#pragma unroll
  for (int j = 0; j < 16; ++j)
    if (j < jn) part[(((int64_t)blockIdx.z * n + a) * rank + j0 + j) * cols + c] = acc[j];
}

// The shares' sum, as [a][j][c] or, turned, [a][c][j].
template <typename T, bool TURNED>
__global__ void __launch_bounds__(256) gather_sum_kernel(const float* __restrict__ part, int shares, int64_t total, int rank, int cols, T* __restrict__ out) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= total) return;
  int64_t from = e;
  if (TURNED) {
    const int64_t j = e % rank, c = e / rank % cols, a = e / rank / cols;
    from = (a * rank + j) * cols + c;
  }
  float s = 0.f;
  for (int z = 0; z < shares; ++z) s += part[z * total + from];
  put(out + e, s);
}

LoraRows rows_of(const Lora& l) { return LoraRows{l.ids, l.id_bytes, l.rows_per_id, l.rows, l.n, l.scaling, l.scaling_value}; }

template <typename T>
int shrink(const Lora& l, bool back, float* h, int shares, cudaStream_t s) {
  const int cols = back ? l.features : l.cols, share = (cols + shares - 1) / shares;
  const Factors<T> f = back ? Factors<T>{(const T*)l.b, (int64_t)l.features * l.rank, 1, l.rank} : Factors<T>{(const T*)l.a, (int64_t)l.cols * l.rank, l.cols, 1};
  const dim3 grid((unsigned)((l.rows + TILE - 1) / TILE), (l.rank + 63) / 64, shares);
  shrink_kernel<T><<<grid, 256, 0, s>>>((const T*)(back ? l.dy : l.x), back ? l.dy_stride : l.x_stride, cols, f, l.rank, rows_of(l), share, h);
  return cuda_fail(cudaGetLastError(), "lora shrink launch");
}
template <typename T>
int expand(const Lora& l, bool back, const float* base, const float* h, int shares, void* y, cudaStream_t s) {
  const int cols = back ? l.cols : l.features;
  const Factors<T> f = back ? Factors<T>{(const T*)l.a, (int64_t)l.cols * l.rank, l.cols, 1} : Factors<T>{(const T*)l.b, (int64_t)l.features * l.rank, 1, l.rank};
  const dim3 grid((unsigned)((l.rows + TILE - 1) / TILE), (cols + COLS - 1) / COLS);
  expand_kernel<T><<<grid, COLS, 0, s>>>(base, back ? nullptr : (const T*)l.bias, h, shares, l.rank, f, rows_of(l), cols, (T*)y);
  return cuda_fail(cudaGetLastError(), "lora expand launch");
}
template <typename T>
int gather(const Lora& l, bool of_b, const float* v, int v_shares, float* part, int shares, cudaStream_t s) {
  const int cols = of_b ? l.features : l.cols, j_blocks = (l.rank + 15) / 16;
  const dim3 grid((cols + COLS - 1) / COLS, l.n * j_blocks, shares);
  gather_kernel<T><<<grid, COLS, 0, s>>>((const T*)(of_b ? l.dy : l.x), of_b ? l.dy_stride : l.x_stride, cols, v, v_shares, l.rank, rows_of(l),
                                         (l.rows + shares - 1) / shares, j_blocks, part);
  return cuda_fail(cudaGetLastError(), "lora gather launch");
}
template <typename T>
int gather_sum(const Lora& l, bool of_b, const float* part, int shares, void* out, cudaStream_t s) {
  const int cols = of_b ? l.features : l.cols;
  const int64_t total = (int64_t)l.n * l.rank * cols;
  const unsigned blocks = (unsigned)((total + 255) / 256);
  if (of_b) gather_sum_kernel<T, true><<<blocks, 256, 0, s>>>(part, shares, total, l.rank, cols, (T*)out);
  else gather_sum_kernel<T, false><<<blocks, 256, 0, s>>>(part, shares, total, l.rank, cols, (T*)out);
  return cuda_fail(cudaGetLastError(), "lora gather sum launch");
}

}  // namespace
}  // namespace tdb

using namespace tdb;

extern "C" {

// Few rows leave SMs idle, so their columns are shared out, down to 256 columns a block; `expand` and `gather` add the shares up.
int tdb_lora_shares(const Lora* l, int back) {
  int sms = 0;
  if (device_sms(&sms)) return 1;
  const int cols = back ? l->features : l->cols;
  const int64_t blocks = (l->rows + TILE - 1) / TILE * ((l->rank + 63) / 64);
  return (int)std::max<int64_t>(1, std::min<int64_t>({(cols + 255) / 256, sms / std::max<int64_t>(1, blocks), 8}));
}
// Likewise for the rows of a gradient, down to 128 of them a block.
int tdb_lora_gather_shares(const Lora* l, int of_b) {
  int sms = 0;
  if (device_sms(&sms)) return 1;
  const int64_t blocks = (int64_t)l->n * ((l->rank + 15) / 16) * (((of_b ? l->features : l->cols) + COLS - 1) / COLS);
  return (int)std::max<int64_t>(1, std::min<int64_t>({(l->rows + 127) / 128, 4 * sms / std::max<int64_t>(1, blocks), 32}));
}

int tdb_lora_shrink(const Lora* l, int back, float* h, int shares, void* stream) {
  return l->dtype == TDB_DTYPE_F32 ? shrink<float>(*l, back, h, shares, (cudaStream_t)stream) : shrink<__nv_bfloat16>(*l, back, h, shares, (cudaStream_t)stream);
}
int tdb_lora_expand(const Lora* l, int back, const float* base, const float* h, int shares, void* y, void* stream) {
  return l->dtype == TDB_DTYPE_F32 ? expand<float>(*l, back, base, h, shares, y, (cudaStream_t)stream)
                                   : expand<__nv_bfloat16>(*l, back, base, h, shares, y, (cudaStream_t)stream);
}
int tdb_lora_gather(const Lora* l, int of_b, const float* v, int v_shares, float* part, int shares, void* stream) {
  return l->dtype == TDB_DTYPE_F32 ? gather<float>(*l, of_b, v, v_shares, part, shares, (cudaStream_t)stream)
                                   : gather<__nv_bfloat16>(*l, of_b, v, v_shares, part, shares, (cudaStream_t)stream);
}
int tdb_lora_gather_sum(const Lora* l, int of_b, const float* part, int shares, void* out, void* stream) {
  return l->dtype == TDB_DTYPE_F32 ? gather_sum<float>(*l, of_b, part, shares, out, (cudaStream_t)stream)
                                   : gather_sum<__nv_bfloat16>(*l, of_b, part, shares, out, (cudaStream_t)stream);
}

}  // extern "C"

// Low-rank adapters of many requests beside a shared projection, for any type and size:
//   y[t] = x[t] W^T + b + s_a (x[t] A_a^T) B_a^T          a: the adapter of row t (none: the shared part alone)
// and coming back, with W frozen,  u[t] = s_a dy[t] B_a,  dx = dy W + u A_a,  dA_a = sum u^T x,  dB_a = sum dy^T h,  h[t] = s_a x[t] A_a^T.
//
// These are the kernels beside the shared product: `shrink` makes h or u, `expand` adds their part to the product and writes the result,
// `gather` sums the gradients.  A tile's rows may belong to several adapters: it takes one adapter after the other.  Where there are adapters
// and rows enough `sort` puts the rows in their order first, so that a tile hardly ever has more than one (2000 rows 2048 -> 2048 in fp32, rank 64, every
// row with another of 32 adapters: 1621 us in the order they come, 528 sorted).
#include "tdb_internal.h"
#include "lora.cuh"
#include <algorithm>

namespace tdb {

namespace {

__device__ __forceinline__ float value(const float* p) { return *p; }
__device__ __forceinline__ float value(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

constexpr int TILE = 16, COLS = 128;

// One matrix per adapter, factor j of column c at j * sj + c * sc.
template <typename T> struct Factors { const T* p; int64_t each, sj, sc; };

// The adapters of up to 32 rows, and which of them there are, by the block's first warp.
struct Present { int id[32], list[32], count; };
__device__ __forceinline__ void find_present(Present& s, const LoraRows& rows, int64_t t0, int n) {
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x, id = lane < n && t0 + lane < rows.rows ? adapter_of(rows, t0 + lane) : -1;
    const uint32_t same = __match_any_sync(0xffffffffu, id);
    const bool first = id >= 0 && (same & ((1u << lane) - 1u)) == 0;
    const uint32_t firsts = __ballot_sync(0xffffffffu, first);
    s.id[lane] = id;
    if (first) s.list[__popc(firsts & ((1u << lane) - 1u))] = id;
    if (lane == 0) s.count = __popc(firsts);
  }
  __syncthreads();
}

// Positions of the rows in the order of their adapters, rows without one last, each adapter's in their own order (the sums of gradients then have
// a fixed order too).  One block: every warp counts its share of the rows by adapter, the counts are added up adapter by adapter, and the
// warps go through their rows once more.  plan: [bins + 1] first positions, [rows] rows, [rows] ids; bins = n + 1.
constexpr int SORT_BYTES = 200 * 1024;
int sort_warps(int n) { return std::min(32, SORT_BYTES / 4 / (n + 1) - 1); }
__global__ void __launch_bounds__(1024) sort_kernel(LoraRows rows, int32_t* __restrict__ plan) {
  extern __shared__ int counts[];                    // [warps][bins], then the bins' own sums
  __shared__ int sums[32];
  const int warps = blockDim.x / 32, warp = threadIdx.x / 32, lane = threadIdx.x % 32, bins = rows.n + 1;
  int* mine = counts + warp * bins;
  const int64_t share = (rows.rows + blockDim.x - 1) / blockDim.x * 32, begin = warp * share, end = min(rows.rows, begin + share);
  int32_t *order = plan + bins + 1, *ids = order + rows.rows;
  for (int i = lane; i < bins; i += 32) mine[i] = 0;
  __syncwarp();
  auto walk = [&](auto&& step) {
    constexpr int AT_ONCE = 8;                       // loads on their way together
    for (int64_t t0 = begin; t0 < end; t0 += 32 * AT_ONCE) {
      int id[AT_ONCE];
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) id[i] = t0 + 32 * i + lane < end ? adapter_of(rows, t0 + 32 * i + lane) : -1;
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) {
        const int64_t row = t0 + 32 * i + lane;
        const bool in = row < end;
        const int bin = in ? (id[i] < 0 ? rows.n : id[i]) : -1;
        const uint32_t same = __match_any_sync(0xffffffffu, bin), before = same & ((1u << lane) - 1u);
        if (in) step(row, id[i], bin, __popc(before));
        __syncwarp();
        if (in && before == 0) mine[bin] += __popc(same);
        __syncwarp();
      }
    }
  };
  walk([](int64_t, int, int, int) {});
  __syncthreads();
  // exclusive sums, warp by warp within a bin, then bin by bin
  int* bases = counts + warps * bins;
  for (int i = warp; i < bins; i += warps) {
    const int n = lane < warps ? counts[lane * bins + i] : 0;
    int run = n;
#pragma unroll
    for (int off = 1; off < 32; off *= 2) {
      const int o = __shfl_up_sync(0xffffffffu, run, off);
      if (lane >= off) run += o;
    }
    if (lane < warps) counts[lane * bins + i] = run - n;
    if (lane == 31) bases[i] = run;
  }
  __syncthreads();
  const int each = (bins + blockDim.x - 1) / blockDim.x, first = threadIdx.x * each, last = min(bins, first + each);
  int total = 0;
  for (int i = first; i < last; ++i) total += bases[i];
  int run = total;
#pragma unroll
  for (int off = 1; off < 32; off *= 2) {
    const int o = __shfl_up_sync(0xffffffffu, run, off);
    if (lane >= off) run += o;
  }
  if (lane == 31) sums[warp] = run;
  __syncthreads();
  int base = run - total;
  for (int w = 0; w < warp; ++w) base += sums[w];
  for (int i = first; i < last; ++i) {
    const int n = bases[i];
    plan[i] = bases[i] = base;
    base += n;
  }
  if (threadIdx.x == 0) plan[bins] = (int)rows.rows;
  __syncthreads();
  walk([&](int64_t row, int id, int bin, int rank) {
    const int at = bases[bin] + mine[bin] + rank;
    order[at] = (int32_t)row;
    ids[at] = id;
  });
}

// h[t][j] = s_a sum over the columns of x[t][c] F_a(j, c).  A block: S_ROWS rows (four, or eight where there are enough of them); its warps share the
// columns, eight factors at a time, so that a thread's 16 loads feed 64 products.  Bound by the factors' way through the caches.
constexpr int S_WARPS = 8, S_FACTORS = 8;
template <typename T, int S_ROWS>
__global__ void __launch_bounds__(S_WARPS * 32) shrink_kernel(const T* __restrict__ x, int64_t stride, int cols, Factors<T> f, int rank, LoraRows rows,
                                                             float* __restrict__ h) {
  __shared__ Present here;
  __shared__ float part[S_WARPS][S_ROWS * S_FACTORS];
  const int64_t t0 = (int64_t)blockIdx.x * S_ROWS;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, j0 = blockIdx.y * S_FACTORS;
  const T* row[S_ROWS];
#pragma unroll
  for (int r = 0; r < S_ROWS; ++r) row[r] = x + row_at(rows, min(t0 + r, rows.rows - 1)) * stride;
  find_present(here, rows, t0, S_ROWS);
  for (int k = 0; k < here.count; ++k) {
    const int a = here.list[k];
    const T* fa = f.p + a * f.each + j0 * f.sj;
    float acc[S_ROWS][S_FACTORS];
#pragma unroll
    for (int r = 0; r < S_ROWS; ++r)
#pragma unroll
      for (int j = 0; j < S_FACTORS; ++j) acc[r][j] = 0.f;
#pragma unroll 2
    for (int c = threadIdx.x; c < cols; c += S_WARPS * 32) {
      float xv[S_ROWS], fv[S_FACTORS];
#pragma unroll
      for (int r = 0; r < S_ROWS; ++r) xv[r] = here.id[r] == a ? value(row[r] + c) : 0.f;
#pragma unroll
      for (int j = 0; j < S_FACTORS; ++j) fv[j] = j0 + j < rank ? value(fa + j * f.sj + (int64_t)c * f.sc) : 0.f;
#pragma unroll
      for (int r = 0; r < S_ROWS; ++r)
#pragma unroll
        for (int j = 0; j < S_FACTORS; ++j) acc[r][j] = fmaf(xv[r], fv[j], acc[r][j]);
    }
    // 32 sums over 32 lanes: lanes trade halves, and lane l ends with sum l
    __syncthreads();
#pragma unroll
    for (int k0 = 0; k0 < S_ROWS; k0 += 4) {
      float v[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = acc[k0 + i / S_FACTORS][i % S_FACTORS];
#pragma unroll
      for (int half = 16; half >= 1; half >>= 1) {
        const bool up = lane & half;
#pragma unroll
        for (int i = 0; i < half; ++i) v[i] = (up ? v[i + half] : v[i]) + __shfl_xor_sync(0xffffffffu, up ? v[i] : v[i + half], half);
      }
      part[warp][k0 * S_FACTORS + lane] = v[0];
    }
    __syncthreads();
    if (threadIdx.x < S_ROWS * S_FACTORS) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < S_WARPS; ++w) s += part[w][threadIdx.x];
      const int r = threadIdx.x / S_FACTORS, j = j0 + threadIdx.x % S_FACTORS;
      if (here.id[r] == a && j < rank) h[(t0 + r) * rank + j] = s * scaling_of(rows, a);
    }
  }
}

// y[t][c] = base[t][c] + bias[c] + sum over j of h[t][j] F_a(j, c), one rounding.  A block: 16 rows, 128 columns, one to a thread.
template <typename T>
__global__ void __launch_bounds__(COLS) expand_kernel(const float* base, const T* __restrict__ bias, const float* __restrict__ h, int rank, Factors<T> f,
                                                      LoraRows rows, int cols, T* y) {     // base may be y
  __shared__ Present here;
  __shared__ __align__(16) float hs[TILE][64];
  const int64_t t0 = (int64_t)blockIdx.x * TILE;
  const int c = blockIdx.y * COLS + threadIdx.x;
  __shared__ int64_t place[TILE];
  if (threadIdx.x < TILE && t0 + threadIdx.x < rows.rows) place[threadIdx.x] = row_at(rows, t0 + threadIdx.x) * cols;
  find_present(here, rows, t0, TILE);
  float sum[TILE];
#pragma unroll
  for (int r = 0; r < TILE; ++r) sum[r] = c < cols && t0 + r < rows.rows ? base[place[r] + c] : 0.f;
  float acc[TILE];
#pragma unroll
  for (int r = 0; r < TILE; ++r) acc[r] = 0.f;
  for (int j0 = 0; j0 < rank; j0 += 64) {
    const int jn = min(64, rank - j0);
    __syncthreads();
    for (int e = threadIdx.x; e < TILE * 64; e += COLS) {
      const int r = e / 64, j = e % 64;
      hs[r][j] = j < jn && here.id[r] >= 0 ? h[(t0 + r) * rank + j0 + j] : 0.f;
    }
    __syncthreads();
    if (c >= cols) continue;
    for (int k = 0; k < here.count; ++k) {
      const int a = here.list[k];
      const T* fa = f.p + a * f.each + j0 * f.sj + (int64_t)c * f.sc;
      uint32_t mine = 0, absent = 0;
#pragma unroll
      for (int r = 0; r < TILE; ++r) {
        mine |= (here.id[r] == a ? 1u : 0u) << r;
        absent |= (t0 + r >= rows.rows ? 1u : 0u) << r;
      }
      const bool vectors = sizeof(T) == 4 && f.sj == 1 && rank % 4 == 0 && (reinterpret_cast<uintptr_t>(fa) & 15) == 0;
      const bool whole = (mine | absent) == (1u << TILE) - 1u;
#pragma unroll 2
      for (int j = 0; j < jn; j += 4) {
        float v[4];
        if (vectors) {
          const float4 q = *reinterpret_cast<const float4*>(fa + j);
          v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = j + i < jn ? value(fa + (j + i) * f.sj) : 0.f;
        }
        if (whole) {
#pragma unroll
          for (int r = 0; r < TILE; ++r) {
            const float4 q = *reinterpret_cast<const float4*>(&hs[r][j]);
            acc[r] = fmaf(q.w, v[3], fmaf(q.z, v[2], fmaf(q.y, v[1], fmaf(q.x, v[0], acc[r]))));
          }
        } else {                                     // other rows' zeros must not meet what may not be finite
#pragma unroll
          for (int r = 0; r < TILE; ++r) {
            const float4 q = *reinterpret_cast<const float4*>(&hs[r][j]);
            const float s = fmaf(q.w, v[3], fmaf(q.z, v[2], fmaf(q.y, v[1], fmaf(q.x, v[0], acc[r]))));
            acc[r] = mine >> r & 1 ? s : acc[r];
          }
        }
      }
    }
  }
  if (c >= cols) return;
  const float b = bias ? value(bias + c) : 0.f;
#pragma unroll
  for (int r = 0; r < TILE; ++r)
    if (t0 + r < rows.rows) put(y + place[r] + c, sum[r] + b + acc[r]);
}

// part[z][a][j][c] = sum over a share of the rows t of adapter a of v[t][j] x[t][c].  A block: one adapter, 16 factors, 128 columns, of one of the
// two gradients (blockIdx.x: the blocks of columns of the first, then those of the second).
template <typename T> struct Side { const T* x; int64_t stride; int cols; const float* v; float* part; int blocks, shares; };
template <typename T>
__global__ void __launch_bounds__(COLS) gather_kernel(Side<T> one, Side<T> two, int rank, LoraRows rows, int j_blocks) {
  const bool later = (int)blockIdx.x >= one.blocks;
  const Side<T> side = later ? two : one;
  const T* __restrict__ x = side.x;
  const float* __restrict__ v = side.v;
  const int64_t stride = side.stride;
  const int cols = side.cols;
  if ((int)blockIdx.z >= side.shares) return;
  __shared__ int ids[32];
  __shared__ int64_t place[32];
  __shared__ __align__(16) float vs[32][16];
  const int a = blockIdx.y / j_blocks, j0 = blockIdx.y % j_blocks * 16, jn = min(16, rank - j0), c = (blockIdx.x - (later ? one.blocks : 0)) * COLS + threadIdx.x;
  // sorted rows: a share of the adapter's own positions, otherwise of all
  const int64_t first = rows.starts ? rows.starts[a] : 0, last = rows.starts ? rows.starts[a + 1] : rows.rows;
  const int64_t share = ((last - first + side.shares - 1) / side.shares + 31) / 32 * 32, begin = first + blockIdx.z * share, end = min(last, begin + share);
  float acc[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) acc[j] = 0.f;
  for (int64_t t0 = begin; t0 < end; t0 += 32) {
    const int count = (int)min((int64_t)32, end - t0);
    __syncthreads();
    int mine = 0;
    if (threadIdx.x < 32) {
      ids[threadIdx.x] = mine = (int)threadIdx.x < count && adapter_of(rows, t0 + threadIdx.x) == a;
      place[threadIdx.x] = mine ? row_at(rows, t0 + threadIdx.x) * stride : 0;
    }
    if (!__syncthreads_or(mine)) continue;
    for (int e = threadIdx.x; e < 32 * 16; e += COLS) {
      const int r = e / 16, j = e % 16;
      vs[r][j] = ids[r] && j < jn ? v[(t0 + r) * rank + j0 + j] : 0.f;
    }
    float xv[32];
#pragma unroll
    for (int r = 0; r < 32; ++r) xv[r] = ids[r] && c < cols ? value(x + place[r] + c) : 0.f;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 32; ++r)
#pragma unroll
      for (int j = 0; j < 16; j += 4) {
        const float4 q = *reinterpret_cast<const float4*>(&vs[r][j]);
        acc[j] = fmaf(q.x, xv[r], acc[j]); acc[j + 1] = fmaf(q.y, xv[r], acc[j + 1]);
        acc[j + 2] = fmaf(q.z, xv[r], acc[j + 2]); acc[j + 3] = fmaf(q.w, xv[r], acc[j + 3]);
      }
  }
  if (c >= cols) return;
  const int n = gridDim.y / j_blocks;
#pragma unroll
  for (int j = 0; j < 16; ++j)
    if (j < jn) side.part[(((int64_t)blockIdx.z * n + a) * rank + j0 + j) * cols + c] = acc[j];
}

// The shares' sums: of a's gradient as [a][j][c], of b's turned by pieces of 8 x 32 to [a][c][j].
template <typename T> struct Sum { const float* part; T* out; int shares, blocks, cols; };
template <typename T>
__global__ void __launch_bounds__(256) gather_sum_kernel(Sum<T> of_a, Sum<T> of_b, int n, int rank) {
  __shared__ float s[8][33];
  const bool turned = (int)blockIdx.x >= of_a.blocks;
  const Sum<T> sum = turned ? of_b : of_a;
  const int64_t total = (int64_t)n * rank * sum.cols;
  if (!turned) {
    const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (e >= total) return;
    float v = 0.f;
#pragma unroll 8
    for (int z = 0; z < sum.shares; ++z) v += sum.part[z * total + e];
    put(sum.out + e, v);
    return;
  }
  const int across = (sum.cols + 31) / 32, down = (rank + 7) / 8, block = blockIdx.x - of_a.blocks;
  const int64_t a = block / (across * down);
  const int c0 = block % across * 32, j0 = block / across % down * 8, tx = threadIdx.x % 32, ty = threadIdx.x / 32;
  float v = 0.f;
  if (j0 + ty < rank && c0 + tx < sum.cols)
#pragma unroll 8
    for (int z = 0; z < sum.shares; ++z) v += sum.part[z * total + (a * rank + j0 + ty) * sum.cols + c0 + tx];
  s[ty][tx] = v;
  __syncthreads();
  const int c = threadIdx.x / 8, j = threadIdx.x % 8;
  if (j0 + j < rank && c0 + c < sum.cols) put(sum.out + (a * sum.cols + c0 + c) * rank + j0 + j, s[j][c]);
}

template <typename T>
int shrink(const Lora& l, bool back, float* h, cudaStream_t s) {
  const int cols = back ? l.features : l.cols;
  const Factors<T> f = back ? Factors<T>{(const T*)l.b, (int64_t)l.features * l.rank, 1, l.rank} : Factors<T>{(const T*)l.a, (int64_t)l.cols * l.rank, l.cols, 1};
  int sms = 0;
  if (const int rc = device_sms(&sms)) return rc;
  const int js = (l.rank + S_FACTORS - 1) / S_FACTORS, each = (l.rows + 7) / 8 * js >= sms ? 8 : 4;
  const dim3 grid((unsigned)((l.rows + each - 1) / each), js);
  (each == 8 ? shrink_kernel<T, 8> : shrink_kernel<T, 4>)<<<grid, S_WARPS * 32, 0, s>>>((const T*)(back ? l.dy : l.x), back ? l.dy_stride : l.x_stride, cols, f, l.rank, lora_rows(l), h);
  return cuda_fail(cudaGetLastError(), "lora shrink launch");
}
template <typename T>
int expand(const Lora& l, bool back, const float* base, const float* h, void* y, cudaStream_t s) {
  const int cols = back ? l.cols : l.features;
  const Factors<T> f = back ? Factors<T>{(const T*)l.a, (int64_t)l.cols * l.rank, l.cols, 1} : Factors<T>{(const T*)l.b, (int64_t)l.features * l.rank, 1, l.rank};
  const dim3 grid((unsigned)((l.rows + TILE - 1) / TILE), (cols + COLS - 1) / COLS);
  expand_kernel<T><<<grid, COLS, 0, s>>>(base, back ? nullptr : (const T*)l.bias, h, l.rank, f, lora_rows(l), cols, (T*)y);
  return cuda_fail(cudaGetLastError(), "lora expand launch");
}
template <typename T>
int gather(const Lora& l, const LoraGradients& g, cudaStream_t s) {
  auto side = [&](const void* x, int64_t stride, int cols, const void* v, float* part, int shares) {
    return Side<T>{(const T*)x, stride, cols, (const float*)v, part, part ? (cols + COLS - 1) / COLS : 0, shares};
  };
  const int j_blocks = (l.rank + 15) / 16;
  const Side<T> a = side(l.x, l.x_stride, l.cols, g.u, g.part_a, g.shares_a), b = side(l.dy, l.dy_stride, l.features, g.h, g.part_b, g.shares_b);
  gather_kernel<T><<<dim3(a.blocks + b.blocks, l.n * j_blocks, std::max(a.shares, b.shares)), COLS, 0, s>>>(a, b, l.rank, lora_rows(l), j_blocks);
  return cuda_fail(cudaGetLastError(), "lora gather launch");
}
template <typename T>
int gather_sum(const Lora& l, const LoraGradients& g, cudaStream_t s) {
  const int64_t each = (int64_t)l.n * l.rank * l.cols, pieces = (int64_t)l.n * ((l.features + 31) / 32) * ((l.rank + 7) / 8);
  const Sum<T> a{g.part_a, (T*)g.da, g.shares_a, g.part_a ? (int)((each + 255) / 256) : 0, l.cols}, b{g.part_b, (T*)g.db, g.shares_b, g.part_b ? (int)pieces : 0, l.features};
  gather_sum_kernel<T><<<a.blocks + b.blocks, 256, 0, s>>>(a, b, l.n, l.rank);
  return cuda_fail(cudaGetLastError(), "lora gather sum launch");
}

}  // namespace
}  // namespace tdb

using namespace tdb;

extern "C" {

// Words of the plan that puts the rows in their adapters' order, 0 where there is none: with one adapter for all, and for few rows, where the launch
// costs more than it saves.  us of a pass 1024 -> 1024, rank 16, with the plan and without it, for 3 adapters in requests of 60 rows, 32 adapters in
// requests of 60, and every row with another of 32:
//   fp32, training             300 rows 102 and 96, 106 and 107, 115 and 179;  700 rows 146 and 148, 160 and 162, 160 and 323;  1000 rows 162 and 159, 171 and 178, 171 and 394
//   fp32, without gradients    300 rows 47 and 43, 49 and 43, 51 and 66;  700 rows 72 and 68, 76 and 68, 76 and 123;  1000 rows 78 and 72, 80 and 72, 81 and 145
//   tensor cores, training     300 rows 33 and 27, 44 and 48, 88 and 92;  768 rows 37 and 31, 47 and 59, 90 and 109;  2500 rows 55 and 53, 72 and 128, 145 and 232
// It costs some 5 us where requests are long and adapters few, and saves up to half where they are not; which of the two a call is only the device knows.
// Products on the tensor cores go by the rows as they come; their gradients want the plan, from more rows on.
int64_t tdb_lora_plan_words(const Lora* l, int tensor_cores) {
  return l->ids && l->n > 1 && l->rows >= (tensor_cores ? 768 : 256) && l->rows < (int64_t)1 << 30 ? l->n + 2 + 2 * l->rows : 0;
}
int tdb_lora_plan(const Lora* l, int32_t* plan, void* stream) {
  const int warps = sort_warps(l->n), smem = (warps + 1) * (l->n + 1) * 4;
  if (smem > 48 * 1024)
    if (const int rc = opt_in_smem(reinterpret_cast<const void*>(sort_kernel), SORT_BYTES)) return rc;
  Lora plain = *l;
  plain.plan = nullptr;
  sort_kernel<<<1, warps * 32, smem, (cudaStream_t)stream>>>(lora_rows(plain), plan);
  return cuda_fail(cudaGetLastError(), "lora sort launch");
}

// How many parts the rows of a gradient are shared out in, so that there are four blocks to an SM, down to 64 rows a part.  factors: to a block.
int tdb_lora_gather_shares(const Lora* l, int of_b, int factors) {
  int sms = 0;
  if (device_sms(&sms)) return 1;
  const int64_t blocks = (int64_t)l->n * ((l->rank + factors - 1) / factors) * (((of_b ? l->features : l->cols) + COLS - 1) / COLS);
  return (int)std::max<int64_t>(1, std::min<int64_t>({(l->rows + 63) / 64, 4 * sms / std::max<int64_t>(1, blocks), 32}));
}

int tdb_lora_shrink(const Lora* l, int back, float* h, void* stream) {
  return l->dtype == TDB_DTYPE_F32 ? shrink<float>(*l, back, h, (cudaStream_t)stream) : shrink<__nv_bfloat16>(*l, back, h, (cudaStream_t)stream);
}
int tdb_lora_expand(const Lora* l, int back, const float* base, const float* h, void* y, void* stream) {
  return l->dtype == TDB_DTYPE_F32 ? expand<float>(*l, back, base, h, y, (cudaStream_t)stream) : expand<__nv_bfloat16>(*l, back, base, h, y, (cudaStream_t)stream);
}
int tdb_lora_gather(const Lora* l, const LoraGradients* g, void* stream) {
  return l->dtype == TDB_DTYPE_F32 ? gather<float>(*l, *g, (cudaStream_t)stream) : gather<__nv_bfloat16>(*l, *g, (cudaStream_t)stream);
}
int tdb_lora_gather_sum(const Lora* l, const LoraGradients* g, void* stream) {
  return l->dtype == TDB_DTYPE_F32 ? gather_sum<float>(*l, *g, (cudaStream_t)stream) : gather_sum<__nv_bfloat16>(*l, *g, (cudaStream_t)stream);
}

}  // extern "C"

// Projections with adapters in bf16 on the tensor cores (lora.cu has the formulas, and the kernels for other types and odd sizes).
//
// Going forward: `shrink` makes the inner values h = s x A^T of every row, then one tcgen05 product makes y, bias and adapters included.
// The adapters' part is a few more columns of the product's inner dimension: behind the tiles of x and W come tiles of h and B_a, and the
// accumulator never leaves tensor memory in between.  A tile whose rows belong to D adapters takes D such steps, each with zeros in place
// of the other adapters' rows.  Coming back the same kernel makes dx = dy W + u A, with W read along its other axis, and `gather` the
// adapters' gradients.
//
// Inner values are held as the sum of two bf16 numbers (hi and lo, 2^-16 of the value or less away from it): rounding them to one would add an
// error as large as the output's own rounding, and the second costs `rank` more columns.
#include "attn_common.cuh"
#include "attn_warp_mma.cuh"
#include "lora.cuh"
#include <algorithm>

namespace tdb {
using namespace ptx;

namespace {

using bf16 = __nv_bfloat16;

// Goes through the adapters of 32 N rows, each once, in the order of their first rows; a whole warp holds the ids, lane l those of
// rows l, l + 32, ...
template <int N>
struct Adapters {
  int id[N];
  uint32_t left[N];
  __device__ __forceinline__ Adapters(const LoraRows& rows, int64_t t0, int lane) {
#pragma unroll
    for (int i = 0; i < N; ++i) id[i] = t0 + 32 * i + lane < rows.rows ? adapter_of(rows, t0 + 32 * i + lane) : -1;
#pragma unroll
    for (int i = 0; i < N; ++i) left[i] = __ballot_sync(0xffffffffu, id[i] >= 0);
  }
  // The next adapter, or -1.
  __device__ __forceinline__ int next() {
    int a = -1;
#pragma unroll
    for (int i = N - 1; i >= 0; --i)
      if (left[i]) a = __shfl_sync(0xffffffffu, id[i], __ffs(left[i]) - 1);
    if (a >= 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) left[i] &= ~__ballot_sync(0xffffffffu, id[i] == a);
    }
    return a;
  }
  __device__ __forceinline__ int count() {              // goes through them
    int n = 0;
    while (next() >= 0) ++n;
    return n;
  }
};

// ------------------------------------------------------------------------------------------------------------------- shrink
// hx[t] = the inner values of row t: r16 high parts, r16 low parts.  A block: 16 MT rows and 8 NJ factors; its eight warps share the columns,
// blocks of 32 in turn, and add up through shared memory.  Bound by reading x, and the factors from L2 once for every block.  As in the skinny
// projections a thread's fragments of two k16 steps are one 16-byte load, since the order of the columns inside a product is free.
// blockIdx.z takes every gridDim.z-th adapter of the rows.
constexpr int SHRINK_WARPS = 8;

template <int MT, int NJ>
__global__ void __launch_bounds__(SHRINK_WARPS * 32) shrink_mma_kernel(const bf16* __restrict__ x, int64_t stride, int cols, const bf16* __restrict__ f, int rank,
                                                                       int r16, LoraRows rows, bf16* __restrict__ hx) {
  extern __shared__ float part[];                      // [warps][16 MT][8 NJ]
  __shared__ int ids[16 * MT];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4, j0 = blockIdx.y * 8 * NJ;
  const int64_t t0 = (int64_t)blockIdx.x * 16 * MT;
  let_next_start();
  if (threadIdx.x < 16 * MT) ids[threadIdx.x] = t0 + threadIdx.x < rows.rows ? adapter_of(rows, t0 + threadIdx.x) : -1;
  __syncthreads();
  constexpr int N = (16 * MT + 31) / 32;
  Adapters<N> adapters(rows, t0, lane);
  if (MT == 1) adapters.left[0] &= 0xffffu;            // half a warp's rows
  const int blocks = (cols + 31) / 32;
  for (int d = 0;; ++d) {
    const int a = adapters.next();
    if (a < 0) break;
    if (d % gridDim.z != blockIdx.z) continue;
    float acc[MT][NJ][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[m][j][e] = 0.f;
    const bf16* fa = f + ((int64_t)a * rank + j0) * cols;
#pragma unroll 2
    for (int b = warp; b < blocks; b += SHRINK_WARPS) {
      const int c = b * 32 + t * 8;
      const bool in = c < cols;
      uint4 fr[NJ], xa[MT][2];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int64_t row = t0 + 16 * m + g + 8 * r;
          xa[m][r] = in && row < rows.rows ? __ldg(reinterpret_cast<const uint4*>(x + row * stride + c)) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
      for (int j = 0; j < NJ; ++j)
        fr[j] = in && j0 + 8 * j + g < rank ? __ldg(reinterpret_cast<const uint4*>(fa + (int64_t)(8 * j + g) * cols + c)) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const uint32_t lo[4] = {xa[m][0].x, xa[m][1].x, xa[m][0].y, xa[m][1].y}, hi[4] = {xa[m][0].z, xa[m][1].z, xa[m][0].w, xa[m][1].w};
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          mma(acc[m][j], lo, fr[j].x, fr[j].y);
          mma(acc[m][j], hi, fr[j].z, fr[j].w);
        }
      }
    }
    __syncthreads();                                   // the sums of the adapter before have been read
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int r = 0; r < 2; ++r)
          *reinterpret_cast<float2*>(part + (warp * 16 * MT + 16 * m + g + 8 * r) * 8 * NJ + 8 * j + 2 * t) = make_float2(acc[m][j][2 * r], acc[m][j][2 * r + 1]);
    __syncthreads();
    const float scale = scaling_of(rows, a);
    for (int e = threadIdx.x; e < 16 * MT * 8 * NJ; e += SHRINK_WARPS * 32) {
      const int row = e / (8 * NJ), j = e % (8 * NJ);
      if (ids[row] != a || j0 + j >= r16) continue;
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < SHRINK_WARPS; ++w) s += part[w * 16 * MT * 8 * NJ + e];
      s *= scale;
      const bf16 high = __float2bfloat16_rn(s);
      const float rest = s - __bfloat162float(high);
      bf16* out = hx + (t0 + row) * 2 * r16 + j0 + j;
      out[0] = high;
      out[r16] = __float2bfloat16_rn(isfinite(rest) ? rest : 0.f);
    }
  }
}

// ------------------------------------------------------------------------------------------------------------------ product
// Persistent, one CTA to an SM, tiles of 128 rows and BN columns, two accumulators.  Warp 0 fetches tiles of x and W by TMA into a ring of
// stages, warps 2..5 fill the stages of the adapters' steps by hand, warp 1 issues the products, warps 6..9 drain one accumulator (tensor
// memory, bias, bf16, shared memory, whole 128-byte lines) while the other one fills.  All of them walk the same list of steps, and
// each finds a tile's adapters for itself from the rows' ids.
//
// 0 x NaN is NaN, so what an adapter holds must not meet other rows' zeros: numbers that are not finite are left out of the B tile, and the
// rows of that adapter get their products from the slow loop at the end of the tile.
constexpr int BM = 128, THREADS = 320;
constexpr uint32_t A_BYTES = BM * 128;
constexpr uint64_t WAIT_NS = 1000ull * 1000ull * 1000ull;
__host__ __device__ constexpr int stages_of(int bn) { return bn == 256 ? 4 : bn == 128 ? 6 : 8; }
__host__ __device__ constexpr uint32_t ring_bytes(int bn) { return (uint32_t)stages_of(bn) * (A_BYTES + (uint32_t)bn * 128); }
constexpr uint32_t OUT_BYTES = 4 * 32 * 128, BAR_BYTES = 512;
__host__ __device__ constexpr uint32_t smem_of(int bn) { return ring_bytes(bn) + OUT_BYTES + BAR_BYTES + 1024; }

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* m, uint32_t bar, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
               ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(c0), "r"(c1) : "memory");
}
// W along its other axis: groups of 64 columns, each 64 rows of 128 bytes (rows run along the inner dimension).
__device__ __forceinline__ uint64_t smem_desc_columns(uint32_t saddr) { return (smem_desc_sw128(saddr) & ~(0x3FFFull << 16)) | ((uint64_t)(8192 >> 4) << 16); }

// Eight factors of one output column from j on; what is not finite is left out and reported.
template <bool VEC>
__device__ __forceinline__ uint4 factors8(const bf16* row, int j, int rank, uint32_t& bad) {
  uint32_t w[4];
  if (VEC) {
    const uint4 v = j < rank ? __ldg(reinterpret_cast<const uint4*>(row + j)) : make_uint4(0, 0, 0, 0);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = j + 2 * i < rank ? __bfloat16_as_ushort(row[j + 2 * i]) : 0, hi = j + 2 * i + 1 < rank ? __bfloat16_as_ushort(row[j + 2 * i + 1]) : 0;
      w[i] = lo | hi << 16;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t not_finite = __vcmpeq2(w[i] & 0x7f807f80u, 0x7f807f80u);
    bad |= not_finite;
    w[i] &= ~not_finite;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

struct ProductParams {
  LoraRows rows;
  const bf16 *hx, *f, *bias;                           // f: [n][N][rank]
  int K, N, rank, r16;
  bf16* y;                                             // [rows][N]
  int32_t* status;
};

template <int BN, bool BACK, bool VEC>
__global__ void __launch_bounds__(THREADS, 1) lora_product_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w, const ProductParams p) {
  constexpr int S = stages_of(BN);
  constexpr uint32_t STAGE = A_BYTES + BN * 128;
  extern __shared__ uint8_t smem_raw[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - smem_u32(smem_raw));
  constexpr uint32_t BARS = ring_bytes(BN) + OUT_BYTES;
  // full[s], empty[s], granted[s], then for both accumulators: filled, drained, and the loaders' report
  auto bar = [&](int i) { return base + BARS + 8u * (uint32_t)i; };
  constexpr int EMPTY = S, GRANTED = 2 * S, FILLED = 3 * S, DRAINED = 3 * S + 2, REPORT = 3 * S + 4;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gbase + BARS + 256);
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gbase + BARS + 260);
  volatile uint32_t* reports = reinterpret_cast<volatile uint32_t*>(gbase + BARS + 264);        // [2][4]
  auto wait = [&](int i, int phase) { return mbar_wait(bar(i), (uint32_t)(phase & 1), abort_flag, p.status, 200 + i, WAIT_NS); };

  if (tid == 0) {
    *abort_flag = 0;
    for (int i = 0; i < 3 * S; ++i) mbar_init(bar(i), 1u);
    for (int i = 0; i < 2; ++i) { mbar_init(bar(FILLED + i), 1u); mbar_init(bar(DRAINED + i), 4u); mbar_init(bar(REPORT + i), 4u); }
    fence_mbar_init();
    prefetch_tmap(&tm_x);
    prefetch_tmap(&tm_w);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), 2 * BN);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int n_tiles = (p.N + BN - 1) / BN, tiles = (int)((p.rows.rows + BM - 1) / BM) * n_tiles;
  const int nk = (p.K + 63) / 64, inner = 2 * p.r16, chunks = (inner + 63) / 64;
  int step = 0, it = 0;

  if (warp == 0) {
    // ---- tiles of x and W
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
      const int m0 = tile / n_tiles * BM, n0 = tile % n_tiles * BN;
      const int more = Adapters<4>(p.rows, m0, lane).count() * chunks;
      if (lane == 0) {
        for (int k = 0; k < nk + more; ++k) {
          const int s = (step + k) % S, round = (step + k) / S;
          // This lane alone waits for stages, in the order of the steps, and grants those of the adapters' steps to the warps that fill them: a
          // barrier tells two neighbouring phases apart and no more, so nobody may wait for one that others can go past.
          if (round > 0) wait(EMPTY + s, round - 1);
          if (k >= nk) mbar_arrive(bar(GRANTED + s));
          if (k >= nk || *abort_flag) continue;
          const uint32_t a = base + s * STAGE, b = a + A_BYTES;
          mbar_expect_tx(bar(s), STAGE);
          tma_load_2d(a, &tm_x, bar(s), k * 64, m0);
          if (!BACK) {
            tma_load_2d(b, &tm_w, bar(s), k * 64, n0);
          } else {
#pragma unroll
            for (int c = 0; c < BN / 64; ++c) tma_load_2d(b + c * 8192, &tm_w, bar(s), n0 + c * 64, k * 64);
          }
        }
      }
      step += nk + more;
      __syncwarp();
    }
  } else if (warp == 1) {
    // ---- products
    constexpr uint32_t ID = make_idesc_bf16(BM, BN, BACK), ID_ADAPTERS = make_idesc_bf16(BM, BN, 0);
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++it) {
      const int m0 = tile / n_tiles * BM;
      const int more = Adapters<4>(p.rows, m0, lane).count() * chunks;
      const uint32_t acc = tmem + (it & 1) * BN;
      if (lane == 0) {
        if (it >= 2) wait(DRAINED + (it & 1), it / 2 - 1);
        tc_fence_after();
        for (int k = 0; k < nk + more; ++k) {
          const int s = (step + k) % S;
          wait(s, (step + k) / S);
          tc_fence_after();
          const uint32_t a = base + s * STAGE, b = a + A_BYTES;
          const uint64_t da = smem_desc_sw128(a), db = BACK && k < nk ? smem_desc_columns(b) : smem_desc_sw128(b);
          const int left = inner - (k - nk) % chunks * 64, k16 = k < nk || left >= 64 ? 4 : left / 16;
          const uint64_t along = BACK && k < nk ? 128 : 2;
          for (int i = 0; i < k16; ++i) mma_ss(acc, da + 2 * i, db + along * i, k < nk ? ID : ID_ADAPTERS, k > 0 || i > 0 ? 1u : 0u);
          tc_commit(bar(EMPTY + s));
        }
        tc_commit(bar(FILLED + (it & 1)));
      }
      step += nk + more;
      __syncwarp();
    }
  } else if (warp < 6) {
    // ---- the adapters' steps: h as the A tile, with zeros in the rows of other adapters, and B_a as the B tile
    const int w = warp - 2, me = w * 32 + lane;
    uint32_t grants = 0;                               // of each stage: the phase to wait for
    wait_for_stream();                                 // hx is made by the kernel in front
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++it) {
      const int m0 = tile / n_tiles * BM, n0 = tile % n_tiles * BN;
      Adapters<4> adapters(p.rows, m0, lane);
      const int mine = w == 0 ? adapters.id[0] : w == 1 ? adapters.id[1] : w == 2 ? adapters.id[2] : adapters.id[3];
      step += nk;
      uint32_t bad = 0;
      for (int a = adapters.next(); a >= 0; a = adapters.next()) {
        for (int c = 0; c < chunks; ++c, ++step) {
          const int pieces = min(8, (inner - c * 64) / 8);
          const uint4* h = reinterpret_cast<const uint4*>(p.hx + (int64_t)(m0 + me) * inner + c * 64);
          uint4 av[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) av[i] = i < pieces && mine == a ? *(h + i) : make_uint4(0, 0, 0, 0);
          const int s = step % S;
          if (lane == 0) wait(GRANTED + s, (int)(grants >> s));
          __syncwarp();
          grants ^= 1u << s;
          const uint32_t at = base + s * STAGE;
          for (int r = me; r < BN; r += 128) {
            const bool real = n0 + r < p.N;
            const bf16* row = p.f + ((int64_t)a * p.N + (real ? n0 + r : 0)) * p.rank;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              if (i >= pieces) break;
              const int q = c * 64 + 8 * i, j = q >= p.r16 ? q - p.r16 : q;
              const uint4 v = factors8<VEC>(row, j, real ? p.rank : 0, bad);
              sts_128(at + A_BYTES + r * 128 + ((i ^ (r & 7)) << 4), v.x, v.y, v.z, v.w);
            }
          }
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (i < pieces) sts_128(at + me * 128 + ((i ^ (me & 7)) << 4), av[i].x, av[i].y, av[i].z, av[i].w);
          fence_proxy_async_smem();
          asm volatile("bar.sync 1, 128;" ::: "memory");
          if (me == 0) mbar_arrive(bar(s));
        }
      }
      bad = __any_sync(0xffffffffu, bad != 0);
      if (lane == 0) {
        if (it >= 2) wait(DRAINED + (it & 1), it / 2 - 1);
        reports[(it & 1) * 4 + w] = bad;
        mbar_arrive(bar(REPORT + (it & 1)));
      }
      __syncwarp();
    }
  } else {
    // ---- results: warp w may read tensor-memory lanes 32 (w % 4) ..., a row to a thread
    const int q = warp & 3;
    const uint32_t out = base + ring_bytes(BN) + q * 4096;
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++it) {
      const int64_t m0 = (int64_t)(tile / n_tiles) * BM + q * 32;
      const int n0 = tile % n_tiles * BN;
      wait(REPORT + (it & 1), it / 2);                 // read before DRAINED, which lets the loaders write the next one here
      const volatile uint32_t* r = reports + (it & 1) * 4;
      const bool bad = r[0] | r[1] | r[2] | r[3];
      wait(FILLED + (it & 1), it / 2);
      tc_fence_after();
      const uint32_t acc = tmem + (it & 1) * BN + ((uint32_t)(q * 32) << 16);
#pragma unroll 1
      for (int c = 0; c < BN / 64; ++c) {
        uint32_t v[64];
        tmem_ld32(acc + c * 64, v);
        tmem_ld32(acc + c * 64 + 32, v + 32);
        tmem_ld_wait32(v);
        tmem_ld_wait32(v + 32);
        if (c == BN / 64 - 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(DRAINED + (it & 1)));
        }
        const int n = n0 + c * 64;
        if (n >= p.N) continue;
        if (p.bias) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (n + 8 * i >= p.N) break;
            const uint4 b = __ldg(reinterpret_cast<const uint4*>(p.bias + n) + i);
            const uint32_t bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              v[8 * i + 2 * e] = __float_as_uint(__uint_as_float(v[8 * i + 2 * e]) + __uint_as_float(bw[e] << 16));
              v[8 * i + 2 * e + 1] = __float_as_uint(__uint_as_float(v[8 * i + 2 * e + 1]) + __uint_as_float(bw[e] & 0xffff0000u));
            }
          }
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          uint32_t o[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = pack_bf16x2(__uint_as_float(v[8 * i + 2 * e]), __uint_as_float(v[8 * i + 2 * e + 1]));
          sts_128(out + lane * 128 + ((i ^ (lane & 7)) << 4), o[0], o[1], o[2], o[3]);
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int row = i * 4 + lane / 8, piece = lane % 8;
          const uint4 o = lds_128(out + row * 128 + ((piece ^ (row & 7)) << 4));
          if (m0 + row < p.rows.rows && n + 8 * piece < p.N) *reinterpret_cast<uint4*>(p.y + (m0 + row) * p.N + n + 8 * piece) = o;
        }
      }
      if (bad && !*abort_flag) {
        __syncwarp();
        const int64_t t = m0 + lane;
        const int a = t < p.rows.rows ? adapter_of(p.rows, t) : -1;
        if (a >= 0)
          for (int n = n0; n < min(n0 + BN, p.N); ++n) {
            float s = 0.f;
            bool any = false;
            for (int j = 0; j < p.rank; ++j) {
              const float v = __bfloat162float(p.f[((int64_t)a * p.N + n) * p.rank + j]);
              if (isfinite(v)) continue;
              any = true;
              s += (__bfloat162float(p.hx[t * inner + j]) + __bfloat162float(p.hx[t * inner + p.r16 + j])) * v;
            }
            if (any) p.y[t * p.N + n] = __float2bfloat16_rn(__bfloat162float(p.y[t * p.N + n]) + s);
          }
      }
    }
  }
  if (*abort_flag) {                                   // copies that may still be in flight get time to land
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, 2 * BN);
}

// ------------------------------------------------------------------------------------------------------------------- gather
// part[z][a][j][c] = sum over this share of the rows t of adapter a of v[t][j] x[t][c], v being the sum of two bf16 numbers.  A block: one
// adapter, 16 MT factors, 128 columns; a warp: 16 columns.  Rows come in tiles of 64 through shared memory, two at a time; tiles without
// a row of the adapter are passed over, and other rows of a tile are zeros in both operands.  Bound by reading x.
constexpr int GC = 128, GP = GC + 8, G_BATCH = 256;
__host__ __device__ constexpr int gather_pitch(int mt) { return 32 * mt + 8; }
__host__ __device__ constexpr int gather_smem(int mt) { return 2 * 64 * (GP + gather_pitch(mt)) * 2; }

template <int MT>
__global__ void __launch_bounds__(256) gather_mma_kernel(const bf16* __restrict__ x, int64_t stride, int cols, const bf16* __restrict__ v, int r16, int rank,
                                                         LoraRows rows, int64_t share, int j_blocks, float* __restrict__ part) {
  constexpr int VP = gather_pitch(MT);
  extern __shared__ __align__(16) bf16 tiles[];
  __shared__ uint64_t masks[G_BATCH];
  bf16 *xs[2] = {tiles, tiles + 64 * GP}, *vs[2] = {tiles + 2 * 64 * GP, tiles + 2 * 64 * GP + 64 * VP};
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int a = blockIdx.y / j_blocks, j0 = blockIdx.y % j_blocks * 16 * MT, c0 = blockIdx.x * GC;
  const int64_t begin = blockIdx.z * share, end = min(rows.rows, begin + share);
  float acc[MT][2][4];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[m][n][e] = 0.f;

  auto copy = [](bf16* dst, const bf16* src, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(saddr(dst)), "l"(src), "r"(real ? 16 : 0) : "memory");
  };
  for (int64_t batch = begin; batch < end; batch += 64 * G_BATCH) {
    const int n = (int)min((int64_t)G_BATCH, (end - batch + 63) / 64);
    __syncthreads();
#pragma unroll 4
    for (int i = warp; i < n; i += 8) {
      const int64_t t = batch + 64 * i + lane;
      const uint32_t lo = __ballot_sync(0xffffffffu, t < end && adapter_of(rows, t) == a);
      const uint32_t hi = __ballot_sync(0xffffffffu, t + 32 < end && adapter_of(rows, t + 32) == a);
      if (lane == 0) masks[i] = (uint64_t)hi << 32 | lo;
    }
    __syncthreads();
    auto next = [&](int i) {
      do ++i;
      while (i < n && masks[i] == 0);
      return i;
    };
    auto load = [&](int i, int buf) {
      const uint64_t m = masks[i];
      const int64_t t0 = batch + 64 * i;
#pragma unroll
      for (int k = 0; k < 64 * GC / 8 / 256; ++k) {
        const int e = tid + 256 * k, r = e / (GC / 8), c = e % (GC / 8) * 8;
        const bool real = m >> r & 1 && c0 + c < cols;
        copy(xs[buf] + r * GP + c, x + (real ? (t0 + r) * stride + c0 + c : 0), real);
      }
#pragma unroll
      for (int k = 0; k < 64 * 4 * MT / 256; ++k) {    // 2 MT pieces of high parts, 2 MT of low ones
        const int e = tid + 256 * k, r = e / (4 * MT), q = e % (4 * MT), low = q / (2 * MT), j = j0 + q % (2 * MT) * 8;
        const bool real = m >> r & 1 && j < r16;
        copy(vs[buf] + r * VP + q * 8, v + (real ? (t0 + r) * 2 * r16 + low * r16 + j : 0), real);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int i = next(-1), buf = 0;
    if (i < n) load(i, 0);
    while (i < n) {
      const int then = next(i);
      if (then < n) load(then, buf ^ 1);
      if (then < n) asm volatile("cp.async.wait_group 1;" ::: "memory");
      else asm volatile("cp.async.wait_group 0;" ::: "memory");
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t xf[4];                                // both operands lie with the rows along the inner dimension: read transposed
        ldsm4t(xf, xs[buf] + (16 * k + (lane & 15)) * GP + warp * 16 + (lane >> 4) * 8);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int low = 0; low < 2; ++low) {
            uint32_t vf[4];
            ldsm4t(vf, vs[buf] + (16 * k + (lane & 7) + (lane >> 4) * 8) * VP + low * 16 * MT + 16 * m + (lane >> 3 & 1) * 8);
            mma(acc[m][0], vf, xf[0], xf[1]);
            mma(acc[m][1], vf, xf[2], xf[3]);
          }
      }
      __syncthreads();
      i = then;
      buf ^= 1;
    }
  }
  const int n = gridDim.y / j_blocks, g = lane / 4, t = lane % 4;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int j = j0 + 16 * m + g + 8 * r;
      if (j >= rank) continue;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int c = c0 + warp * 16 + 8 * e + 2 * t;
        if (c < cols)
          *reinterpret_cast<float2*>(part + (((int64_t)blockIdx.z * n + a) * rank + j) * cols + c) = make_float2(acc[m][e][2 * r], acc[m][e][2 * r + 1]);
      }
    }
}

// in [n][rows][cols] -> out [n][cols][rows], by squares of 32
__global__ void __launch_bounds__(256) turn_kernel(const bf16* __restrict__ in, int rows, int cols, bf16* __restrict__ out) {
  __shared__ bf16 s[32][33];
  const int64_t at = (int64_t)blockIdx.z * rows * cols;
  const int c0 = blockIdx.x * 32, r0 = blockIdx.y * 32, tx = threadIdx.x % 32, ty = threadIdx.x / 32;
  for (int i = ty; i < 32; i += 8)
    if (r0 + i < rows && c0 + tx < cols) s[i][tx] = in[at + (int64_t)(r0 + i) * cols + c0 + tx];
  __syncthreads();
  for (int i = ty; i < 32; i += 8)
    if (c0 + i < cols && r0 + tx < rows) out[at + (int64_t)(c0 + i) * rows + r0 + tx] = s[tx][i];
}

LoraRows rows_of(const Lora& l) { return LoraRows{l.ids, l.id_bytes, l.rows_per_id, l.rows, l.n, l.scaling, l.scaling_value}; }
int r16_of(const Lora& l) { return (l.rank + 15) / 16 * 16; }

template <int MT, int NJ>
int launch_shrink(const Lora& l, const bf16* x, int64_t stride, int cols, const bf16* f, bf16* hx, int sms, cudaStream_t s) {
  constexpr int smem = SHRINK_WARPS * 16 * MT * 8 * NJ * 4;
  if (smem > 48 * 1024)
    if (const int rc = opt_in_smem(reinterpret_cast<const void*>(shrink_mma_kernel<MT, NJ>), smem)) return rc;
  const int64_t tiles = (l.rows + 16 * MT - 1) / (16 * MT);
  const int js = (r16_of(l) + 8 * NJ - 1) / (8 * NJ);
  // where there are SMs to spare, a tile's adapters are shared out too
  const int z = (int)std::max<int64_t>(1, std::min<int64_t>({l.n, 16 * MT, l.rows, 2 * sms / std::max<int64_t>(1, tiles * js)}));
  shrink_mma_kernel<MT, NJ><<<dim3((unsigned)tiles, js, z), SHRINK_WARPS * 32, smem, s>>>(x, stride, cols, f, l.rank, r16_of(l), rows_of(l), hx);
  return cuda_fail(cudaGetLastError(), "lora shrink launch");
}

template <int BN, bool BACK>
int launch_product(const CUtensorMap& tx, const CUtensorMap& tw, const ProductParams& p, int sms, cudaStream_t s) {
  const bool vec = p.rank % 8 == 0 && (reinterpret_cast<uintptr_t>(p.f) & 15) == 0;
  auto kernel = vec ? lora_product_kernel<BN, BACK, true> : lora_product_kernel<BN, BACK, false>;
  if (const int rc = opt_in_smem(reinterpret_cast<const void*>(kernel), (int)smem_of(BN))) return rc;
  const int64_t tiles = (p.rows.rows + BM - 1) / BM * ((p.N + BN - 1) / BN);
  return cuda_fail(launch_early(kernel, dim3((unsigned)std::min<int64_t>(tiles, sms)), THREADS, smem_of(BN), s, tx, tw, p), "lora product launch");
}

// The width of the tiles: the one whose waves of tiles take least, 256 columns counting 256, 128 of them 136 (twice the steps for the same
// products) and 64 of them 96 (their operands come from shared memory slower than they are multiplied).
int columns_of(int64_t rows, int N, int sms) {
  const int64_t m = (rows + BM - 1) / BM;
  auto cost = [&](int bn, int each) { return (m * ((N + bn - 1) / bn) + sms - 1) / sms * each; };
  const int64_t c256 = cost(256, 256), c128 = cost(128, 136), c64 = cost(64, 96);
  return c256 <= c128 && c256 <= c64 ? 256 : c128 <= c64 ? 128 : 64;
}

}  // namespace
}  // namespace tdb

using namespace tdb;

extern "C" {

// bf16 whose rows TMA can address; the host sees to it that the tensors are aligned.
int tdb_lora_umma_applies(const Lora* l) {
  return l->dtype == TDB_DTYPE_BF16 && l->cols % 8 == 0 && l->features % 8 == 0 && l->rows < (int64_t)1 << 30;
}

int64_t tdb_lora_inner(const Lora* l) { return 2 * r16_of(*l); }

int tdb_lora_umma_shrink(const Lora* l, int back, const void* f, void* hx, void* stream) {
  int sms = 0;
  if (const int rc = device_sms(&sms)) return rc;
  const bf16* x = (const bf16*)(back ? l->dy : l->x);
  const int64_t stride = back ? l->dy_stride : l->x_stride;
  const int cols = back ? l->features : l->cols;
  auto run = [&](auto launch) { return launch(*l, x, stride, cols, (const bf16*)f, (bf16*)hx, sms, (cudaStream_t)stream); };
  const int mt = l->rows <= 16 * sms ? 1 : l->rows <= 64 * sms ? 2 : 4;
  if (l->rank <= 16) return run(mt == 1 ? launch_shrink<1, 2> : mt == 2 ? launch_shrink<2, 2> : launch_shrink<4, 2>);
  if (l->rank <= 32) return run(mt == 1 ? launch_shrink<1, 4> : mt == 2 ? launch_shrink<2, 4> : launch_shrink<4, 4>);
  return run(mt == 1 ? launch_shrink<1, 8> : launch_shrink<2, 8>);
}

int tdb_lora_umma_product(const Lora* l, int back, const void* f, const void* hx, void* y, int32_t* status, void* stream) {
  int sms = 0, rc;
  if ((rc = device_sms(&sms))) return rc;
  const int K = back ? l->features : l->cols, N = back ? l->cols : l->features;
  const ProductParams p{rows_of(*l), (const bf16*)hx, (const bf16*)f, back ? nullptr : (const bf16*)l->bias, K, N, l->rank, r16_of(*l), (bf16*)y, status};
  const int bn = columns_of(l->rows, N, sms);
  CUtensorMap tx, tw;
  if ((rc = bf16_map_2d(&tx, back ? l->dy : l->x, K, l->rows, back ? l->dy_stride : l->x_stride, BM, back ? "dy" : "x"))) return rc;
  if ((rc = bf16_map_2d(&tw, l->w, l->cols, l->features, l->cols, back ? 64 : bn, "weight"))) return rc;
  cudaStream_t s = (cudaStream_t)stream;
  if (back) return bn == 256 ? launch_product<256, true>(tx, tw, p, sms, s) : bn == 128 ? launch_product<128, true>(tx, tw, p, sms, s) : launch_product<64, true>(tx, tw, p, sms, s);
  return bn == 256 ? launch_product<256, false>(tx, tw, p, sms, s) : bn == 128 ? launch_product<128, false>(tx, tw, p, sms, s) : launch_product<64, false>(tx, tw, p, sms, s);
}

int tdb_lora_turn(const void* in, int n, int rows, int cols, void* out, void* stream) {
  turn_kernel<<<dim3((cols + 31) / 32, (rows + 31) / 32, n), 256, 0, (cudaStream_t)stream>>>((const bf16*)in, rows, cols, (bf16*)out);
  return cuda_fail(cudaGetLastError(), "lora turn launch");
}

int tdb_lora_umma_gather(const Lora* l, int of_b, const void* v, float* part, int shares, void* stream) {
  const int cols = of_b ? l->features : l->cols, r16 = r16_of(*l), mt = r16 <= 16 ? 1 : r16 <= 32 ? 2 : 4, j_blocks = (r16 + 16 * mt - 1) / (16 * mt);
  const int64_t share = ((l->rows + shares - 1) / shares + 63) / 64 * 64;
  auto run = [&](auto kernel) {
    if (const int rc = opt_in_smem(reinterpret_cast<const void*>(kernel), gather_smem(mt))) return rc;
    kernel<<<dim3((cols + GC - 1) / GC, l->n * j_blocks, shares), 256, gather_smem(mt), (cudaStream_t)stream>>>(
        (const bf16*)(of_b ? l->dy : l->x), of_b ? l->dy_stride : l->x_stride, cols, (const bf16*)v, r16, l->rank, rows_of(*l), share, j_blocks, part);
    return cuda_fail(cudaGetLastError(), "lora gather launch");
  };
  return mt == 1 ? run(gather_mma_kernel<1>) : mt == 2 ? run(gather_mma_kernel<2>) : run(gather_mma_kernel<4>);
}

}  // extern "C"

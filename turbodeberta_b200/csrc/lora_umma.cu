// Projections with adapters in bf16 on the tensor cores (lora.cu has the formulas, and the kernels for other types and odd sizes).
//
// Going forward: `shrink` makes the inner values h = s x A^T of every row, then one tcgen05 product makes y, bias and adapters included.
// The adapters' part is a few more columns of the product's inner dimension: behind the tiles of x and W come tiles of h and B_a, and the
// accumulator never leaves tensor memory in between.  A tile whose rows belong to several adapters takes the columns of each, one behind the other, with
// zeros in the rows of the others.  Coming back the same kernel makes dx = dy W + u A, with W read along its other axis, and `gather` the
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
  int id[N], high[N];
  uint32_t left[N];
  // ask() only starts the loads, so that their way from memory can pass beside other work; start() is the first to look at them.
  __device__ __forceinline__ void ask(const LoraRows& rows, int64_t t0, int lane) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      id[i] = high[i] = -1;
      const int64_t row = t0 + 32 * i + lane;
      if (row >= rows.rows) continue;
      const int64_t at = rows.rows_per_id == 1 ? row : row / rows.rows_per_id;
      if (!rows.ids) {
        id[i] = high[i] = 0;
      } else if (rows.id_bytes == 8) {
        const int2 v = static_cast<const int2*>(rows.ids)[at];
        id[i] = v.x; high[i] = v.y;
      } else {
        id[i] = static_cast<const int*>(rows.ids)[at];
        high[i] = 0;
      }
    }
  }
  __device__ __forceinline__ void start(int n) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      id[i] = high[i] == 0 && id[i] >= 0 && id[i] < n ? id[i] : -1;
      left[i] = __ballot_sync(0xffffffffu, id[i] >= 0);
    }
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
// hx[t] = the inner values of row t: r16 high parts, r16 low parts.  A block: 16 MT rows and 8 NJ factors; its warps share the columns, blocks of
// 64 in turn, and add up through shared memory.  Bound by reading x, and the factors from L2 once for every block: each warp has STAGES blocks
// of columns on their way into shared memory that is its own, so that nothing waits for the block's other warps.
// blockIdx.z takes every gridDim.z-th adapter of the rows.  Rows may come sorted by adapter (lora.cu); what is read and written then is the row at each position.
template <int MT, int NJ> __host__ __device__ constexpr int shrink_stage() { return (16 * MT + 8 * NJ) * 128; }

template <int MT, int NJ, int WARPS, int STAGES>
__global__ void __launch_bounds__(WARPS * 32) shrink_mma_kernel(const bf16* __restrict__ x, int64_t stride, int cols, const bf16* __restrict__ f, int rank,
                                                                int r16, LoraRows rows, bf16* __restrict__ hx) {
  extern __shared__ __align__(128) uint8_t ring[];     // [warps][stages][rows of x, then factors][64]; then the warps' sums
  __shared__ int ids[16 * MT], place[16 * MT];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4, j0 = blockIdx.y * 8 * NJ;
  const int64_t t0 = (int64_t)blockIdx.x * 16 * MT;
  let_next_start();
  if (threadIdx.x < 16 * MT) {
    const bool in = t0 + threadIdx.x < rows.rows;
    ids[threadIdx.x] = in ? adapter_of(rows, t0 + threadIdx.x) : -1;
    place[threadIdx.x] = in ? (int)row_at(rows, t0 + threadIdx.x) : 0;
  }
  __syncthreads();
  constexpr int N = (16 * MT + 31) / 32, STAGE = shrink_stage<MT, NJ>();
  Adapters<N> adapters;
#pragma unroll
  for (int i = 0; i < N; ++i) { adapters.id[i] = 32 * i + lane < 16 * MT ? ids[32 * i + lane] : -1; adapters.high[i] = 0; }
  adapters.start(rows.n);
  const uint32_t mine = smem_u32(ring) + warp * STAGES * STAGE;
  const int blocks = (cols + 63) / 64, n = blocks > warp ? (blocks - warp + WARPS - 1) / WARPS : 0;      // blocks of columns, and this warp's of them
  float* part = reinterpret_cast<float*>(ring);        // [warps][16 MT][8 NJ]
  for (int d = 0;; ++d) {
    const int a = adapters.next();
    if (a < 0) break;
    if (d % gridDim.z != blockIdx.z) continue;
    const bf16* fa = f + ((int64_t)a * rank + j0) * cols;
    auto ask = [&](int i) {                            // this warp's i-th block of columns
      if (i < n) {
        const int c = (warp + i * WARPS) * 64 + lane % 8 * 8;
        const uint32_t at = mine + i % STAGES * STAGE;
#pragma unroll
        for (int k = 0; k < (16 * MT + 8 * NJ) / 4; ++k) {
          const int r = 4 * k + lane / 8;
          const bool of_x = r < 16 * MT;
          const bool in = c < cols && (of_x ? t0 + r < rows.rows : j0 + r - 16 * MT < rank);
          const bf16* src = of_x ? x + place[r] * stride + c : fa + (int64_t)(r - 16 * MT) * cols + c;
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at + r * 128 + ((lane % 8 ^ (r & 7)) << 4)), "l"(in ? src : x), "r"(in ? 16 : 0) : "memory");
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    float acc[MT][NJ][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[m][j][e] = 0.f;
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) ask(i);
    for (int i = 0; i < n; ++i) {
      ask(i + STAGES - 1);
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
      __syncwarp();
      const uint8_t* at = ring + (mine - smem_u32(ring)) + i % STAGES * STAGE;
      auto piece = [&](int r, int c) { return reinterpret_cast<const bf16*>(at + r * 128 + ((c ^ (r & 7)) << 4)); };
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t xf[MT][4];
#pragma unroll
        for (int m = 0; m < MT; ++m) ldsm4(xf[m], piece(16 * m + lane % 16, 2 * k + lane / 16));
#pragma unroll
        for (int j = 0; j < NJ; j += 2) {
          uint32_t ff[4];
          ldsm4(ff, piece(16 * MT + 8 * j + lane % 8 + lane / 16 * 8, 2 * k + lane / 8 % 2));
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            mma(acc[m][j], xf[m], ff[0], ff[1]);
            mma(acc[m][j + 1], xf[m], ff[2], ff[3]);
          }
        }
      }
      __syncwarp();                                    // read by all lanes: may be filled again
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();                                   // the sums lie where the rings are
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int r = 0; r < 2; ++r)
          *reinterpret_cast<float2*>(part + (warp * 16 * MT + 16 * m + g + 8 * r) * 8 * NJ + 8 * j + 2 * t) = make_float2(acc[m][j][2 * r], acc[m][j][2 * r + 1]);
    __syncthreads();
    const float scale = scaling_of(rows, a);
    for (int e = threadIdx.x; e < 16 * MT * 8 * NJ; e += WARPS * 32) {
      const int row = e / (8 * NJ), j = e % (8 * NJ);
      if (ids[row] != a || j0 + j >= r16) continue;
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) s += part[w * 16 * MT * 8 * NJ + e];
      s = j0 + j < rank ? s * scale : 0.f;             // what pads the rank: x's infinities times its zeros would be NaN
      const bf16 high = __float2bfloat16_rn(s);
      const float rest = s - __bfloat162float(high);
      bf16* out = hx + (int64_t)place[row] * 2 * r16 + j0 + j;
      out[0] = high;
      out[r16] = __float2bfloat16_rn(isfinite(rest) ? rest : 0.f);
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------------------------------ product
// Persistent, tiles of 128 CTAS rows and BN columns, two accumulators.  With CTAS = 2 a pair of SMs works on one tile: each fetches its own
// 128 rows of x and half of the columns of W, and the tensor cores of both read the other half from the neighbour.  That halves what W takes of L2
// and of shared memory: 9216 rows 1024 -> 4096 without adapters take 74 us with a 128 x 256 tile to one SM and 52 with 256 x 256 to a pair, on
// rings of 192 KB (59 with the two stages that the adapters have of it; the library's product takes 57).
//
// Warp 0 fetches tiles of x and W by TMA into a ring of stages, warps 2..5 fill two stages of their own with the adapters' tiles, warp 1 (of
// the pair's first CTA) issues the products, warps 6..9 drain one accumulator (tensor memory, bias, bf16, shared memory, TMA) while the other one
// fills.  Warp 10 counts the adapters of the worker's tiles ahead of the others.  The adapters have stages apart because a load takes as long as
// all that TMA has asked for before it, 2500 cycles: filled a tile ahead they cost the product nothing, in the ring 4 us a tile (9216
// rows 1024 -> 4096, one adapter: 90 us, without 54).
//
// 0 x NaN is NaN, so what an adapter holds must not meet other rows' zeros: numbers that are not finite are left out of the B tile, and the
// rows of that adapter get their products from a loop at the end.
constexpr int BM = 128, THREADS = 352, MOST_TILES = 512;   // MOST_TILES: of one worker in a launch
constexpr uint32_t A_BYTES = BM * 128;
constexpr uint64_t WAIT_NS = 1000ull * 1000ull * 1000ull;
__host__ __device__ constexpr uint32_t stage_bytes(int bn, int ctas) { return A_BYTES + (uint32_t)(bn / ctas) * 128; }
constexpr int AHEAD = 2;                               // stages of the adapters
__host__ __device__ constexpr int stages_of(int bn, int ctas) { return 192 * 1024 / (int)stage_bytes(bn, ctas) - AHEAD; }
__host__ __device__ constexpr uint32_t ring_bytes(int bn, int ctas) { return (uint32_t)(stages_of(bn, ctas) + AHEAD) * stage_bytes(bn, ctas); }
constexpr uint32_t OUT_BYTES = 2 * 4 * 32 * 128, BAR_BYTES = 512 + 2 * MOST_TILES;
__host__ __device__ constexpr uint32_t smem_of(int bn, int ctas) { return ring_bytes(bn, ctas) + OUT_BYTES + BAR_BYTES + 1024; }

// The pair: addresses, barriers and tensor-core instructions that reach the neighbour.
__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
// RELEASE: what this thread wrote goes first; that waits for all its stores to global memory too, some 1500 cycles where there are any.
template <bool RELEASE>
__device__ __forceinline__ void arrive_in_cluster(uint32_t bar) {
  if (RELEASE) asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
  else asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
template <int CTAS>
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* m, uint32_t bar, int c0, int c1) {
  if (CTAS == 2)                                       // may signal the neighbour's barrier
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(c0), "r"(c1) : "memory");
  else
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(c0), "r"(c1) : "memory");
}
// For a converged warp: every lane computes the operands, so that they can stay in uniform registers, and one elected lane issues.
template <int CTAS>
__device__ __forceinline__ void mma_step(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
  if (CTAS == 2)
    asm volatile("{\n\t.reg .pred p, q;\n\telect.sync _|q, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t@q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accum) : "memory");
  else
    mma_ss_warp(d, a, b, idesc, accum);
}
// The barrier at this offset, in both CTAs of a pair, completes once the products so far have.
template <int CTAS>
__device__ __forceinline__ void commit_step(uint32_t bar) {
  if (CTAS == 2)
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\t"
                 "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(bar), "h"((uint16_t)3) : "memory");
  else
    tc_commit_warp(bar);
}
template <int CTAS>
__device__ __forceinline__ void alloc_columns(uint32_t dst, uint32_t n) {
  if (CTAS == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(n) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    tmem_alloc(dst, n);
    tmem_relinquish();
  }
}
template <int CTAS>
__device__ __forceinline__ void free_columns(uint32_t tmem, uint32_t n) {
  if (CTAS == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(n) : "memory");
  else tmem_dealloc(tmem, n);
}
// W along its other axis: groups of 64 columns, each 64 rows of 128 bytes (rows run along the inner dimension).
__device__ __forceinline__ uint64_t smem_desc_columns(uint32_t saddr) { return (smem_desc_sw128(saddr) & ~(0x3FFFull << 16)) | ((uint64_t)(8192 >> 4) << 16); }

// Eight factors of one output column from j on, where they are not vectors.
__device__ __forceinline__ uint4 factors8(const bf16* row, int j, int rank) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = j + 2 * i < rank ? __bfloat16_as_ushort(row[j + 2 * i]) : 0, hi = j + 2 * i + 1 < rank ? __bfloat16_as_ushort(row[j + 2 * i + 1]) : 0;
    w[i] = lo | hi << 16;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// What is not finite becomes zero, and is reported.
__device__ __forceinline__ uint4 finite8(uint4 v, uint32_t& bad) {
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
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

template <int BN, int CTAS, bool BACK, bool VEC>
__global__ void __launch_bounds__(THREADS, 1) lora_product_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_y,
                    const ProductParams p) {
  constexpr int S = stages_of(BN, CTAS), PART = BN / CTAS;        // PART: columns of W whose tile is in this CTA
  constexpr uint32_t STAGE = stage_bytes(BN, CTAS);
  extern __shared__ uint8_t smem_raw[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - smem_u32(smem_raw));
  constexpr uint32_t BARS = ring_bytes(BN, CTAS) + OUT_BYTES;
  // full[s] (the first CTA's counts for both CTAs) and empty[s], the adapters' stages behind the others; then for both accumulators: filled, drained
  auto bar = [&](int i) { return base + BARS + 8u * (uint32_t)i; };
  constexpr int EMPTY = S + AHEAD, FILLED = 2 * EMPTY, DRAINED = FILLED + 2;
  static_assert(8 * (DRAINED + 2) <= 256, "barriers");
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gbase + BARS + 256);
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gbase + BARS + 260);
  volatile int* counted = reinterpret_cast<volatile int*>(gbase + BARS + 268);                 // tiles whose adapters have been counted
  volatile uint16_t* counts = reinterpret_cast<volatile uint16_t*>(gbase + BARS + 512);
  volatile uint32_t* bad_factors = reinterpret_cast<volatile uint32_t*>(gbase + BARS + 264);
  auto wait = [&](int i, int phase) { return mbar_wait(bar(i), (uint32_t)(phase & 1), abort_flag, p.status, 200 + i, WAIT_NS); };
  const uint32_t rank = CTAS == 2 ? cta_rank() : 0;
  auto first_cta = [&](uint32_t addr) { return CTAS == 2 ? in_cta(addr, 0) : addr; };
  if (tid == 0) {
    *abort_flag = 0;
    *bad_factors = 0;
    *counted = 0;
    for (int i = 0; i < 2 * EMPTY; ++i) mbar_init(bar(i), i < EMPTY ? CTAS : 1u);
    for (int i = 0; i < 2; ++i) { mbar_init(bar(FILLED + i), 1u); mbar_init(bar(DRAINED + i), 4u * CTAS); }
    fence_mbar_init();
    prefetch_tmap(&tm_x);
    prefetch_tmap(&tm_w);
    prefetch_tmap(&tm_y);
  }
  if (warp == 1) alloc_columns<CTAS>(smem_u32(const_cast<uint32_t*>(tmem_slot)), 2 * BN);
  __syncwarp();
  tc_fence_before();
  if (CTAS == 2) cluster_sync();
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int n_tiles = (p.N + BN - 1) / BN, tiles = (int)((p.rows.rows + BM * CTAS - 1) / (BM * CTAS)) * n_tiles;
  const int workers = gridDim.x / CTAS, worker = blockIdx.x / CTAS;
  const int nk = (p.K + 63) / 64, inner = 2 * p.r16;      // inner: columns of an adapter; a tile's adapters lie one behind the other
  int it = 0;
  using Tile = Adapters<4 * CTAS>;
  auto count_of = [&](int i) {                         // of this worker's i-th tile
    if (*counted <= i) {
      const uint64_t t0 = globaltimer_ns();
      while (*counted <= i && !*abort_flag)
        if (globaltimer_ns() - t0 > WAIT_NS) {
          *abort_flag = 1;
          if (*reinterpret_cast<volatile int*>(p.status) == 0) *reinterpret_cast<volatile int*>(p.status) = 299;
        }
    }
    __threadfence_block();
    return *counted > i ? (int)counts[i] : 0;          // none where a wait has given up: whoever else knows of some finds its waits over at once
  };
  auto tile_row = [&](int tile) { return (int64_t)(tile / n_tiles) * BM * CTAS; };

  // Stages go round; `odd` is the parity of the round.  A fresh barrier counts as having completed the phase before its first.
  int s = 0, odd = 0, extra = 0, extra_odd = 0;
  auto advance = [&] { if (++s == S) { s = 0; odd ^= 1; } };
  auto advance_extra = [&] { if (++extra == AHEAD) { extra = 0; extra_odd ^= 1; } };

  if (warp == 0) {
    // ---- tiles of x and W
    for (int tile = worker; tile < tiles; tile += workers) {
      const int m0 = (int)tile_row(tile) + rank * BM, n0 = tile % n_tiles * BN + rank * PART;
      if (lane == 0) {
        bool go = true;
        for (int k = 0; k < nk; ++k, advance()) {
          go = wait(EMPTY + s, odd ^ 1) && go;
          if (!go) continue;
          const uint32_t a = base + s * STAGE, b = a + A_BYTES, full = first_cta(bar(s));
          if (rank == 0) mbar_expect_tx(bar(s), STAGE * CTAS);
          if (CTAS == 2 && rank == 0) mbar_arrive(bar(s));          // for the neighbour, whose bytes are counted here: an arrival from there would cost it a fence
          tma_load_2d<CTAS>(a, &tm_x, full, k * 64, m0);
          if (!BACK) {
            tma_load_2d<CTAS>(b, &tm_w, full, k * 64, n0);
          } else {
#pragma unroll
            for (int c = 0; c < PART / 64; ++c) tma_load_2d<CTAS>(b + c * 8192, &tm_w, full, n0 + c * 64, k * 64);
          }
        }
      }
      __syncwarp();
    }
  } else if (warp == 1 && rank == 0) {
    // ---- products
    constexpr uint32_t ID = make_idesc_bf16(BM * CTAS, BN, BACK), ID_ADAPTERS = make_idesc_bf16(BM * CTAS, BN, 0);
    const uint64_t a0 = smem_desc_sw128(base), b0 = smem_desc_sw128(base + A_BYTES), w0 = BACK ? smem_desc_columns(base + A_BYTES) : b0;
    constexpr uint64_t ALONG = BACK ? 128 : 2;         // 16 more of the inner dimension
    for (int tile = worker; tile < tiles; tile += workers, ++it) {
      const uint32_t acc = tmem + (it & 1) * BN;
      if (it >= 2) wait(DRAINED + (it & 1), it / 2 - 1);
      tc_fence_after();
      for (int k = 0; k < nk; ++k, advance()) {
        wait(s, odd);
        tc_fence_after();
        const uint64_t a = a0 + (uint32_t)s * (STAGE >> 4), b = w0 + (uint32_t)s * (STAGE >> 4);
        mma_step<CTAS>(acc, a, b, ID, k > 0 ? 1u : 0u);
#pragma unroll
        for (int i = 1; i < 4; ++i) mma_step<CTAS>(acc, a + 2 * i, b + ALONG * i, ID, 1u);
        commit_step<CTAS>(bar(EMPTY + s));
      }
      for (int left = count_of(it) * inner; left > 0; left -= 64, advance_extra()) {
        wait(S + extra, extra_odd);
        tc_fence_after();
        const uint64_t a = a0 + (uint32_t)(S + extra) * (STAGE >> 4), b = b0 + (uint32_t)(S + extra) * (STAGE >> 4);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (16 * i < left) mma_step<CTAS>(acc, a + 2 * i, b + 2 * i, ID_ADAPTERS, 1u);
        commit_step<CTAS>(bar(EMPTY + S + extra));
      }
      commit_step<CTAS>(bar(FILLED + (it & 1)));
    }
  } else if (warp >= 2 && warp < 6) {
    // ---- the adapters' steps: h as the A tile, with zeros in the rows of other adapters, and B_a as the B tile.  Two warps to each of the two
    // stages, so that one is on its way while the other is checked, handed over or waited for.
    static_assert(AHEAD == 2, "two pairs of warps");
    const int stage = S + (warp - 2) / 2, half = warp & 1;       // rows 32 half + lane, and those 64 further on, of both tiles
    constexpr int BR = PART / 64;
    uint32_t bad = 0;
    auto copy = [](uint32_t dst, const void* src, bool real) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
    };
    const int me = half * 32 + lane;
    const uint32_t at = base + stage * STAGE + me * 128;
    auto place = [&](int r, int piece) { return at + r * 64 * 128 + ((piece ^ (me & 7)) << 4); };
    Tile adapters;
    if (worker < tiles) adapters.ask(p.rows, tile_row(worker), lane);
    wait_for_stream();                                 // hx is made by the kernel in front
    for (int tile = worker; tile < tiles; tile += workers, ++it) {
      const bf16* h = p.hx + (tile_row(tile) + rank * BM + me) * inner;
      const int n0 = tile % n_tiles * BN + rank * PART;
      adapters.start(p.rows.n);
      int mine[2] = {-1, -1};
#pragma unroll
      for (int i = 0; i < 4 * CTAS; ++i)
        if (i / 4 == (int)rank && i % 2 == half) mine[i % 4 / 2] = adapters.id[i];
      int a = -1, q = inner;                           // the adapter, and the column of it, that comes next
      for (int left = count_of(it) * inner / 8; left > 0; left -= 8, advance_extra()) {        // left: pieces of eight columns
        const int pieces = min(8, left);
        const bool ours = S + extra == stage;
        if (ours) {
          if (lane == 0) wait(EMPTY + stage, extra_odd ^ 1);
          __syncwarp();
        }
#pragma unroll
        for (int four = 0; four < 8; four += 4) {      // an adapter has a multiple of four pieces
          if (four >= pieces) break;
          if (q == inner) { a = adapters.next(); q = 0; }
          if (ours) {
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
              for (int i = 0; i < 4; ++i) copy(place(r, four + i), mine[r] == a && a >= 0 ? h + (int64_t)r * 64 * inner + q + 8 * i : p.hx, mine[r] == a && a >= 0);
#pragma unroll
            for (int r = 0; r < BR; ++r) {
              const int n = n0 + me + 64 * r;
              const bf16* row = p.f + ((int64_t)max(a, 0) * p.N + min(n, p.N - 1)) * p.rank;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int j = q + 8 * i >= p.r16 ? q + 8 * i - p.r16 : q + 8 * i;
                const bool real = a >= 0 && n < p.N && j < p.rank;
                if (VEC) {
                  copy(place(r, four + i) + A_BYTES, real ? row + j : p.f, real);
                } else {
                  const uint4 v = factors8(row, j, real ? p.rank : 0);
                  sts_128(place(r, four + i) + A_BYTES, v.x, v.y, v.z, v.w);
                }
              }
            }
          }
          q += 32;
        }
        if (!ours) continue;
        asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
        for (int r = 0; r < BR; ++r)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (i >= pieces) break;
            uint32_t worse = 0;
            const uint4 v = finite8(lds_128(place(r, i) + A_BYTES), worse);
            if (worse) sts_128(place(r, i) + A_BYTES, v.x, v.y, v.z, v.w);
            bad |= worse;
          }
        fence_proxy_async_smem();
        asm volatile("bar.sync %0, 64;" ::"r"(stage - S + 1) : "memory");
        if (me == 0) {
          if (CTAS == 2) arrive_in_cluster<true>(in_cta(bar(stage), 0));
          else mbar_arrive(bar(stage));
        }
      }
      if (tile + workers < tiles) adapters.ask(p.rows, tile_row(tile + workers), lane);
    }
    if (bad) {                                         // for the loop at the end, in both CTAs
      const uint32_t at = smem_u32(const_cast<uint32_t*>(bad_factors));
      if (CTAS == 1) *bad_factors = 1;
      else
        for (int r = 0; r < CTAS; ++r) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(in_cta(at, r)), "r"(1u) : "memory");
    }
    __syncwarp();
  } else if (warp == 10) {
    // ---- how many adapters each tile has
    for (int tile = worker; tile < tiles; tile += workers, ++it) {
      Tile adapters;
      adapters.ask(p.rows, tile_row(tile), lane);
      adapters.start(p.rows.n);
      const int n = adapters.count();
      if (lane == 0) {
        counts[it] = (uint16_t)n;
        __threadfence_block();
        *counted = it + 1;
      }
    }
  } else if (warp >= 6) {
    // ---- results: warp w may read tensor-memory lanes 32 (w % 4) ..., a row to a thread; 32 rows and 64 columns at a time go out by TMA from one
    // of two buffers
    const int q = warp & 3;
    int turn = 0;
    for (int tile = worker; tile < tiles; tile += workers, ++it) {
      const int m0 = (int)tile_row(tile) + rank * BM + q * 32, n0 = tile % n_tiles * BN;
      wait(FILLED + (it & 1), it / 2);
      tc_fence_after();
      const uint32_t acc = tmem + (it & 1) * BN + ((uint32_t)(q * 32) << 16);
#pragma unroll 1
      for (int c = 0; c < BN / 64; ++c, turn ^= 1) {
        const int n = n0 + c * 64;
        uint32_t v[64];
        tmem_ld32(acc + c * 64, v);
        tmem_ld32(acc + c * 64 + 32, v + 32);
        uint4 b[8];
        if (p.bias) {
#pragma unroll
          for (int i = 0; i < 8; ++i) b[i] = n + 8 * i < p.N ? __ldg(reinterpret_cast<const uint4*>(p.bias + n) + i) : make_uint4(0, 0, 0, 0);
        }
        const uint32_t out = base + ring_bytes(BN, CTAS) + (q * 2 + turn) * 4096;
        asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");           // the store from this buffer has read it
        tmem_ld_wait32(v);
        tmem_ld_wait32(v + 32);
        __syncwarp();
        if (c == BN / 64 - 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (CTAS == 1) mbar_arrive(bar(DRAINED + (it & 1)));
            else arrive_in_cluster<false>(in_cta(bar(DRAINED + (it & 1)), 0));   // the first CTA issues the products
          }
        }
        if (p.bias) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint32_t bw[4] = {b[i].x, b[i].y, b[i].z, b[i].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              v[8 * i + 2 * e] = __float_as_uint(__uint_as_float(v[8 * i + 2 * e]) + __uint_as_float(bw[e] << 16));
              v[8 * i + 2 * e + 1] = __float_as_uint(__uint_as_float(v[8 * i + 2 * e + 1]) + __uint_as_float(bw[e] & 0xffff0000u));
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          uint32_t o[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = pack_bf16x2(__uint_as_float(v[8 * i + 2 * e]), __uint_as_float(v[8 * i + 2 * e + 1]));
          sts_128(out + lane * 128 + ((i ^ (lane & 7)) << 4), o[0], o[1], o[2], o[3]);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {                               // rows and columns behind the last are left out by the copy
          if (m0 < p.rows.rows && n < p.N && !*abort_flag)
            asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];"
                         ::"l"(reinterpret_cast<uint64_t>(&tm_y)), "r"(out), "r"(n), "r"(m0) : "memory");
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
      }
    }
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  if (*abort_flag) {                                   // copies that may still be in flight get time to land
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  __syncwarp();
  tc_fence_before();
  if (CTAS == 2) cluster_sync();                       // nobody leaves while the neighbour may still read or signal here
  else __syncthreads();
  tc_fence_after();
  if (warp == 1) free_columns<CTAS>(tmem, 2 * BN);
  if (!*bad_factors || *abort_flag) return;
  // Some factor is not finite: this CTA's tiles once more, for what was left out of them.
  for (int tile = worker; tile < tiles; tile += workers) {
    const int n0 = tile % n_tiles * BN;
    for (int e = tid; e < BM * BN; e += THREADS) {
      const int64_t t = tile_row(tile) + rank * BM + e / BN;
      const int n = n0 + e % BN, a = t < p.rows.rows ? adapter_of(p.rows, t) : -1;
      if (a < 0 || n >= p.N) continue;
      float sum = 0.f;
      bool any = false;
      for (int j = 0; j < p.rank; ++j) {
        const float v = __bfloat162float(p.f[((int64_t)a * p.N + n) * p.rank + j]);
        if (isfinite(v)) continue;
        any = true;
        sum += (__bfloat162float(p.hx[t * inner + j]) + __bfloat162float(p.hx[t * inner + p.r16 + j])) * v;
      }
      if (any) p.y[t * p.N + n] = __float2bfloat16_rn(__bfloat162float(p.y[t * p.N + n]) + sum);
    }
  }
}

// ------------------------------------------------------------------------------------------------------------------- gather
// part[z][a][j][c] = sum over a share of the rows t of adapter a of v[t][j] x[t][c], v being the sum of two bf16 numbers.  A block: one
// adapter, 16 MT factors, 128 columns; a warp: 16 columns.  The adapter's rows, which the plan lists, come in tiles of 64 through shared memory, two at
// a time; blockIdx.z takes every shares-th tile.  Without a plan (few rows) all rows do, zeros in the place of those that are not the adapter's.  Both
// gradients in one launch (blockIdx.x: the blocks of columns of the first, then those of the second).  Bound by reading x.
constexpr int GC = 128, GP = GC + 8, G_BATCH = 16;     // G_BATCH: tiles whose rows are looked up at once
__host__ __device__ constexpr int gather_pitch(int mt) { return 32 * mt + 8; }
__host__ __device__ constexpr int gather_smem(int mt) { return 2 * 64 * (GP + gather_pitch(mt)) * 2; }

struct GatherSide { const bf16* x; int64_t stride; int cols; const bf16* v; float* part; int blocks, shares; };

template <int MT>
__global__ void __launch_bounds__(256) gather_mma_kernel(const GatherSide one, const GatherSide two, int r16, int rank, const LoraRows rows, int j_blocks) {
  constexpr int VP = gather_pitch(MT);
  const bool later = (int)blockIdx.x >= one.blocks;
  const GatherSide side = later ? two : one;
  const bf16 *__restrict__ x = side.x, *__restrict__ v = side.v;
  const int64_t stride = side.stride;
  const int cols = side.cols, shares = side.shares;
  if ((int)blockIdx.z >= shares) return;
  extern __shared__ __align__(16) bf16 tiles[];
  __shared__ int place[G_BATCH * 64];                  // -1: not a row of the adapter
  bf16 *xs[2] = {tiles, tiles + 64 * GP}, *vs[2] = {tiles + 2 * 64 * GP, tiles + 2 * 64 * GP + 64 * VP};
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int a = blockIdx.y / j_blocks, j0 = blockIdx.y % j_blocks * 16 * MT, c0 = (blockIdx.x - (later ? one.blocks : 0)) * GC;
  const int first = rows.starts ? rows.starts[a] : 0, last = rows.starts ? rows.starts[a + 1] : (int)rows.rows, all = (last - first + 63) / 64;
  const int mine = all > (int)blockIdx.z ? (all - (int)blockIdx.z + shares - 1) / shares : 0;       // tiles of this block
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
  for (int batch = 0; batch < mine; batch += G_BATCH) {
    const int todo = min(G_BATCH, mine - batch);
    __syncthreads();
    for (int e = tid; e < todo * 64; e += 256) {
      const int at = first + ((batch + e / 64) * shares + (int)blockIdx.z) * 64 + e % 64;
      place[e] = at >= last || (!rows.starts && adapter_of(rows, at) != a) ? -1 : (int)row_at(rows, at);
    }
    __syncthreads();
    auto load = [&](int i, int buf) {
#pragma unroll
      for (int k = 0; k < 64 * GC / 8 / 256; ++k) {
        const int e = tid + 256 * k, r = e / (GC / 8), c = e % (GC / 8) * 8, row = place[i * 64 + r];
        const bool real = row >= 0 && c0 + c < cols;
        copy(xs[buf] + r * GP + c, x + (real ? row * stride + c0 + c : 0), real);
      }
#pragma unroll
      for (int k = 0; k < 64 * 4 * MT / 256; ++k) {    // 2 MT pieces of high parts, 2 MT of low ones
        const int e = tid + 256 * k, r = e / (4 * MT), q = e % (4 * MT), low = q / (2 * MT), j = j0 + q % (2 * MT) * 8, row = place[i * 64 + r];
        const bool real = row >= 0 && j < r16;
        copy(vs[buf] + r * VP + q * 8, v + (real ? (int64_t)row * 2 * r16 + low * r16 + j : 0), real);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    load(0, 0);
    for (int i = 0, buf = 0; i < todo; ++i, buf ^= 1) {
      if (i + 1 < todo) {
        load(i + 1, buf ^ 1);
        asm volatile("cp.async.wait_group 1;" ::: "memory");
      } else {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
      }
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
    }
  }
  const int g = lane / 4, t = lane % 4;
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
          *reinterpret_cast<float2*>(side.part + (((int64_t)blockIdx.z * rows.n + a) * rank + j) * cols + c) = make_float2(acc[m][e][2 * r], acc[m][e][2 * r + 1]);
      }
    }
}

// [n][rows][cols] -> [n][cols][rows] by squares of 32, for two lists of matrices at once.
struct Turn { const bf16* in; bf16* out; int rows, cols, blocks; };       // blocks: of one matrix
__global__ void __launch_bounds__(256) turn_kernel(Turn first, Turn second) {
  __shared__ bf16 s[32][33];
  const bool later = (int)blockIdx.x >= first.blocks;
  const Turn& t = later ? second : first;
  const int64_t at = (int64_t)blockIdx.y * t.rows * t.cols;
  const int block = blockIdx.x - (later ? first.blocks : 0), across = (t.cols + 31) / 32;
  const int c0 = block % across * 32, r0 = block / across * 32, tx = threadIdx.x % 32, ty = threadIdx.x / 32;
#pragma unroll
  for (int i = ty; i < 32; i += 8)
    if (r0 + i < t.rows && c0 + tx < t.cols) s[i][tx] = t.in[at + (int64_t)(r0 + i) * t.cols + c0 + tx];
  __syncthreads();
  const int wide = min(32, t.rows - r0);
  for (int e = threadIdx.x; e < 32 * wide; e += 256) {
    const int c = e / wide, r = e % wide;
    if (c0 + c < t.cols) t.out[at + (int64_t)(c0 + c) * t.rows + r0 + r] = s[r][c];
  }
}

int r16_of(const Lora& l) { return (l.rank + 15) / 16 * 16; }

template <int MT, int NJ, int WARPS, int STAGES>
int launch_shrink(const Lora& l, const bf16* x, int64_t stride, int cols, const bf16* f, bf16* hx, int sms, cudaStream_t s) {
  constexpr int smem = WARPS * STAGES * shrink_stage<MT, NJ>();
  static_assert(WARPS * 16 * MT * 8 * NJ * 4 <= smem, "the warps' sums");
  auto kernel = shrink_mma_kernel<MT, NJ, WARPS, STAGES>;
  if (const int rc = opt_in_smem(reinterpret_cast<const void*>(kernel), smem)) return rc;
  const int64_t tiles = (l.rows + 16 * MT - 1) / (16 * MT);
  const int js = (r16_of(l) + 8 * NJ - 1) / (8 * NJ);
  // where there are SMs to spare, a tile's adapters are shared out too
  const int z = (int)std::max<int64_t>(1, std::min<int64_t>({l.n, 16 * MT, l.rows, 2 * sms / std::max<int64_t>(1, tiles * js)}));
  kernel<<<dim3((unsigned)tiles, js, z), WARPS * 32, smem, s>>>(x, stride, cols, f, l.rank, r16_of(l), lora_rows(l), hx);
  return cuda_fail(cudaGetLastError(), "lora shrink launch");
}

template <int BN, int CTAS, bool BACK>
int launch_product(const CUtensorMap& tx, const CUtensorMap& tw, const CUtensorMap& ty, const ProductParams& p, int sms, cudaStream_t s) {
  const bool vec = p.rank % 8 == 0 && (reinterpret_cast<uintptr_t>(p.f) & 15) == 0;
  auto kernel = vec ? lora_product_kernel<BN, CTAS, BACK, true> : lora_product_kernel<BN, CTAS, BACK, false>;
  if (const int rc = opt_in_smem(reinterpret_cast<const void*>(kernel), (int)smem_of(BN, CTAS))) return rc;
  const int64_t tiles = (p.rows.rows + BM * CTAS - 1) / (BM * CTAS) * ((p.N + BN - 1) / BN);
  cudaLaunchAttribute attr[2]{};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {CTAS, 1, 1};
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)std::min<int64_t>(tiles, sms / CTAS) * CTAS); cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = smem_of(BN, CTAS); cfg.stream = s;
  cfg.attrs = attr; cfg.numAttrs = CTAS == 2 ? 2 : 1;
  return cuda_fail(cudaLaunchKernelEx(&cfg, kernel, tx, tw, ty, p), "lora product launch");
}

// Columns of a tile, and whether a pair of SMs shares it: the form whose waves of tiles take least.  us of a launch by waves, inner dimension 4096:
// 256 x 256 to a pair 25..27, 49..56, 83 (one, two, three); 128 x 128 to one SM 19..25, 43, 64..78 (three, four); 128 x 64 19, 37..39, 72 (four).
// Per wave that is 256 to 195 to 175.  1024 rows 4096 -> 4096: pair 33, 43 and 69 with one SM to a tile; 512 rows 27, 25, 37; 200 rows 25, 21, 20.
struct Shape { int columns, ctas; };
Shape shape_of(int64_t rows, int N, int sms) {
  auto waves = [&](int m, int n, int workers) { return ((rows + m - 1) / m * ((N + n - 1) / n) + workers - 1) / workers; };
  const int64_t pair = waves(256, 256, sms / 2) * 256, wide = waves(128, 128, sms) * 195, narrow = waves(128, 64, sms) * 175;
  return pair <= wide && pair <= narrow ? Shape{256, 2} : wide <= narrow ? Shape{128, 1} : Shape{64, 1};
}

}  // namespace
}  // namespace tdb

using namespace tdb;

extern "C" {

// bf16 whose rows TMA can address; the host sees to it that the tensors are aligned.
int tdb_lora_umma_applies(const Lora* l) {
  int sms = 0;
  if (l->dtype != TDB_DTYPE_BF16 || l->cols % 8 || l->features % 8 || l->rows >= (int64_t)1 << 30 || device_sms(&sms)) return 0;
  for (const int N : {l->features, l->cols}) {
    const Shape s = shape_of(l->rows, N, sms);
    if ((l->rows + BM * s.ctas - 1) / (BM * s.ctas) * ((N + s.columns - 1) / s.columns) > (int64_t)MOST_TILES * (sms / s.ctas)) return 0;     // outputs of some 5 GB
  }
  return 1;
}

int tdb_lora_umma_form(int64_t rows, int columns, int* tile_columns, int* ctas) {
  int sms = 0;
  if (const int rc = device_sms(&sms)) return rc;
  const Shape s = shape_of(rows, columns, sms);
  *tile_columns = s.columns;
  *ctas = s.ctas;
  return TDB_OK;
}

int64_t tdb_lora_inner(const Lora* l) { return 2 * r16_of(*l); }

int tdb_lora_umma_shrink(const Lora* l, int back, const void* f, void* hx, void* stream) {
  int sms = 0;
  if (const int rc = device_sms(&sms)) return rc;
  const bf16* x = (const bf16*)(back ? l->dy : l->x);
  const int64_t stride = back ? l->dy_stride : l->x_stride;
  const int cols = back ? l->features : l->cols;
  auto run = [&](auto launch) { return launch(*l, x, stride, cols, (const bf16*)f, (bf16*)hx, sms, (cudaStream_t)stream); };
  const bool few = l->rows <= 16 * sms;
  if (l->rank <= 16) return run(few ? launch_shrink<1, 2, 8, 2> : launch_shrink<2, 2, 4, 4>);
  if (l->rank <= 32) return run(few ? launch_shrink<1, 4, 8, 2> : launch_shrink<2, 4, 4, 3>);
  return run(few ? launch_shrink<1, 8, 8, 2> : launch_shrink<2, 8, 4, 2>);
}

int tdb_lora_umma_product(const Lora* l, int back, const void* f, const void* hx, void* y, int32_t* status, void* stream) {
  int sms = 0, rc;
  if ((rc = device_sms(&sms))) return rc;
  const int K = back ? l->features : l->cols, N = back ? l->cols : l->features;
  const ProductParams p{lora_rows_as_they_come(*l), (const bf16*)hx, (const bf16*)f, back ? nullptr : (const bf16*)l->bias, K, N, l->rank, r16_of(*l), (bf16*)y, status};
  const Shape shape = shape_of(l->rows, N, sms);
  CUtensorMap tx, tw, ty;
  if ((rc = bf16_map_2d(&tx, back ? l->dy : l->x, K, l->rows, back ? l->dy_stride : l->x_stride, BM, back ? "dy" : "x"))) return rc;
  if ((rc = bf16_map_2d(&tw, l->w, l->cols, l->features, l->cols, back ? 64 : shape.columns / shape.ctas, "weight"))) return rc;
  if ((rc = bf16_map_2d(&ty, y, N, l->rows, N, 32, "y"))) return rc;
  cudaStream_t s = (cudaStream_t)stream;
  auto run = [&](auto launch) { return launch(tx, tw, ty, p, sms, s); };
  if (back) return run(shape.columns == 256 ? launch_product<256, 2, true> : shape.columns == 128 ? launch_product<128, 1, true> : launch_product<64, 1, true>);
  return run(shape.columns == 256 ? launch_product<256, 2, false> : shape.columns == 128 ? launch_product<128, 1, false> : launch_product<64, 1, false>);
}

int tdb_lora_turn(const Lora* l, void* a_turned, void* b_turned, void* stream) {
  auto list = [](const void* in, void* out, int rows, int cols) {
    return Turn{(const bf16*)in, (bf16*)out, rows, cols, out ? (cols + 31) / 32 * ((rows + 31) / 32) : 0};
  };
  const Turn a = list(l->a, a_turned, l->rank, l->cols), b = list(l->b, b_turned, l->features, l->rank);
  turn_kernel<<<dim3(a.blocks + b.blocks, l->n), 256, 0, (cudaStream_t)stream>>>(a, b);
  return cuda_fail(cudaGetLastError(), "lora turn launch");
}

int tdb_lora_umma_gather_factors(const Lora* l) { return l->rank <= 16 ? 16 : l->rank <= 32 ? 32 : 64; }

int tdb_lora_umma_gather(const Lora* l, const LoraGradients* g, void* stream) {
  auto side = [](const void* x, int64_t stride, int cols, const void* v, float* part, int shares) {
    return GatherSide{(const bf16*)x, stride, cols, (const bf16*)v, part, part ? (cols + GC - 1) / GC : 0, shares};
  };
  const GatherSide a = side(l->x, l->x_stride, l->cols, g->u, g->part_a, g->shares_a), b = side(l->dy, l->dy_stride, l->features, g->h, g->part_b, g->shares_b);
  const int r16 = r16_of(*l), mt = tdb_lora_umma_gather_factors(l) / 16, j_blocks = (r16 + 16 * mt - 1) / (16 * mt);
  auto run = [&](auto kernel) {
    if (const int rc = opt_in_smem(reinterpret_cast<const void*>(kernel), gather_smem(mt))) return rc;
    kernel<<<dim3(a.blocks + b.blocks, l->n * j_blocks, std::max(a.shares, b.shares)), 256, gather_smem(mt), (cudaStream_t)stream>>>(
        a, b, r16, l->rank, lora_rows(*l), j_blocks);
    return cuda_fail(cudaGetLastError(), "lora gather launch");
  };
  return mt == 1 ? run(gather_mma_kernel<1>) : mt == 2 ? run(gather_mma_kernel<2>) : run(gather_mma_kernel<4>);
}

}  // extern "C"

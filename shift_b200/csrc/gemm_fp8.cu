// Products of 8-bit matrices with a power-of-two scale per block of 128.
//
//   D[m, n] (+)= sum_b 2^(ea[m, b] + eb[n, b]) sum_{k in block b} A[m, k] B[n, k]
//
// Both operands have the contraction inside (K-major), see fp8.cuh for their
// layout.  Row groups: A and D rows are cut into segments by offs[0..G], group
// g multiplies with B rows [g N, (g + 1) N).  K groups: the contraction is cut
// into segments on block boundaries, group g writes D rows [g M, (g + 1) M).
//
// The block-scaled form of tcgen05.mma multiplies each product by both scales
// itself, for runs of 32 along K: a block of 128 is four of them with the same
// exponent.  So sums stay in one fp32 accumulator in tensor memory over the
// whole contraction and no partial sum is ever rescaled.  The exponents of 128
// rows and four blocks are 128 words; the scale plane is stored so that they
// are contiguous, and tcgen05.cp spreads them over tensor memory in the order
// the instruction wants (row r in lane r % 32, column r / 32).
//
// Two CTAs on neighbouring SMs work on one tile of 256 rows (cta_group::2): each
// loads half of A's and half of B's rows, so an operand byte feeds twice as
// many products as in a CTA of its own; the first one issues the instructions
// for both.  Rows that fit one CTA's 128 take the single form.
//
// Warp roles (384 threads):
//   warp 0      TMA loads of the operand tiles (one lane)
//   warp 1      MMA issue (one lane)
//   warp 2      scale words: global -> shared memory
//   warp 3      tensor memory allocation; in a pair, word of the scales' arrival
//   warps 4..11 epilogue: a lane quarter of tensor memory (warp % 4) is read by
//               two warps, which take alternate columns
// All waits are bounded (common.cuh).
//
// Bound: operations where the contraction is long (8192^3: 0.374 ms, 2943
// TFLOP/s, 512 of every 590 clocks a block are products; 0.466 ms under the
// power cap), the way from L2 where it is short (16384 x 1536 x 1024: 27 us
// from a warm L2, 34 us from DRAM): a pair's tile of 256 x 256 brings 32 KB
// into each SM per block, which takes 64 bytes a clock for the 512 clocks that
// its products take.
#include <cuda.h>
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <atomic>
#include <mutex>

#include "fp8.cuh"

namespace sb {
namespace fp8 {

enum Mode : int { kRowGroups = 0, kKGroups = 1 };

constexpr int kThreads = 384;
constexpr int kEpiWarps = 8;
constexpr int BM = 128;
constexpr int BK = 128;            // one scale block, one 128-byte swizzled row
constexpr int kMaxGroups = 512;
constexpr int kBand = 8;           // row tiles whose column tiles are walked together

// CTAS: CTAs that share a tile of 128 * CTAS rows and BN columns.  Two
// accumulators alternate so that the epilogue of one tile runs under the next
// one's products.  256 columns twice would leave no room for the scales, so
// there the two share 32 columns, which the epilogue reads first.
template <int BN, int CTAS>
struct Cfg {
  static constexpr int kTileM = BM * CTAS;
  static constexpr int kABytes = BM * BK;
  static constexpr int kBRows = BN / CTAS;                       // rows of B that one CTA loads
  static constexpr int kBBytes = kBRows * BK;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kEpiBytes = kEpiWarps * 4096;             // per warp a buffer of 32 rows x 128 bytes
  static constexpr int kBParts = (BN + 127) / 128;               // 128-row parts of the B scales
  static constexpr int kScaleBytes = 512 * (1 + kBParts);
  static constexpr bool kShared = BN == 256;
  static constexpr int kAccCols = kShared ? 224 : BN;
  static constexpr int kScaleStages = kShared ? 2 : 4;
  static constexpr int kScaleCols = 4 * (1 + kBParts);
  static constexpr int kTmemCols = 512;
  static constexpr int kScaleCol0 = kAccCols + BN;
  static_assert(kScaleCol0 + kScaleStages * kScaleCols <= kTmemCols, "tensor memory budget");
  static constexpr int kFixed = kEpiBytes + kScaleStages * kScaleBytes + 1024 + 512 + 2 * (kMaxGroups + 1) * 4;
  static constexpr int kStages = (232448 - kFixed) / kStageBytes < 8 ? (232448 - kFixed) / kStageBytes : 8;
  static constexpr int kSmemBytes = kStages * kStageBytes + kFixed;
  static_assert(kStages >= 3 && kStageBytes % 1024 == 0, "shared memory budget");
};

// Division of a number below 2^31 by a fixed one: high half of a product, and
// a shift.  With s = ceil(log2 d) and m = ceil(2^(31 + s) / d) the quotient is
// exact, since m d - 2^(31 + s) < 2^s.
struct Divisor {
  unsigned m, s, d;
  void set(unsigned by) {
    d = by;
    for (s = 0; (1u << s) < by; ++s) {}
    m = static_cast<unsigned>(((1ull << (31 + s)) + by - 1) / by);
  }
  SB_DEVICE int operator()(int x) const {
    return static_cast<int>((static_cast<unsigned long long>(static_cast<unsigned>(x)) * m) >> (31 + s));
  }
};

struct Args {
  const uint32_t *sa, *sb;
  int rows_a, rows_b;      // rows of the scale planes
  int M, N, K, G, mode;
  int split;               // row mode, one group: K ranges, partial sums into D [split][M][N] fp32
  int tiles_n;
  Divisor by_band, by_tiles;   // kBand * tiles_n; tiles of one group (K groups, split)
  const int* offs;
  void* D;
  long ldd;
  bool f32, acc, d_vec;    // d_vec: D takes 16-byte stores
  uint32_t idesc;
  int* status;
};

struct Tile {
  int n0;                  // first column of D
  int a_row, b_row;        // rows of the operands
  long d_row;              // first output row
  int m_valid;             // rows of this CTA that are wanted (none: 0 or less)
  int kb0, kb;             // first block of 128, number of blocks
};

// True in one lane of a converged warp.  A role that only issues instructions
// for the tensor cores or TMA runs under this: the compiler then knows that one
// lane runs it and keeps descriptors and barriers in uniform registers, where
// those instructions take them from (under `lane == 0` the four products of a
// block took 290 clocks to issue, more than they take to run).
SB_DEVICE bool elect_one() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}
// D[tmem] (+)= A[smem] B[smem]^T with the scales in tensor memory.
template <int CTAS>
SB_DEVICE void umma_scaled(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                           uint32_t accumulate) {
  if constexpr (CTAS == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}
// 32 rows of 16 bytes to 32 lanes x 4 columns, repeated in the four lane
// quarters; in both CTAs of a pair, each from its own shared memory.
template <int CTAS>
SB_DEVICE void tmem_copy_scales(uint32_t taddr, uint32_t smem_addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>(128 >> 4) << 32;      // eight rows of 16 bytes apart
  d |= 1ull << 46;
  if constexpr (CTAS == 1)
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(d) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(d) : "memory");
}
// Arrive on this barrier (of both CTAs of a pair) when the products issued so far are done.
template <int CTAS>
SB_DEVICE void commit(uint64_t* bar) {
  if constexpr (CTAS == 1) {
    umma_commit(bar);
  } else {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"(static_cast<uint16_t>(3))
        : "memory");
  }
}
// The same on this CTA's barrier alone.
template <int CTAS>
SB_DEVICE void commit_here(uint64_t* bar) {
  if constexpr (CTAS == 1) umma_commit(bar);
  else
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
// The first CTA's barrier at the same place, as a cluster address.
SB_DEVICE uint32_t leader_addr(const void* p) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_u32(p)));
  return a;
}
template <int CTAS>
SB_DEVICE void arrive_leader(uint64_t* bar) {
  if constexpr (CTAS == 1) {
    mbar_arrive(bar);
  } else {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(leader_addr(bar)) : "memory");
  }
}
// Wait (bounded) for a barrier that the other CTA's threads arrive on too.
template <int CTAS>
SB_DEVICE bool wait_both(uint64_t* bar, uint32_t phase, int* status) {
  if constexpr (CTAS == 1) {
    return mbar_wait(bar, phase, status);
  } else {
    uint64_t start = 0;
    while (true) {
      uint32_t ok;
      asm volatile(
          "{\n\t.reg .pred p;\n\t"
          "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, 1000000;\n\t"
          "selp.u32 %0, 1, 0, p;\n\t}"
          : "=r"(ok)
          : "r"(smem_u32(bar)), "r"(phase)
          : "memory");
      if (ok) return true;
      const uint64_t now = globaltimer_ns();
      if (start == 0) start = now;
      if (now - start > kPipelineTimeoutNs) {
        record_status(status, kTimeoutPipeline);
        return false;
      }
    }
  }
}
// A tile of this GPU's memory into this CTA's shared memory; completes on the first CTA's barrier.
template <int CTAS>
SB_DEVICE void load_tile(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y) {
  if constexpr (CTAS == 1) {
    tma_load_2d(dst, map, bar, x, y);
  } else {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(leader_addr(bar)), "r"(x), "r"(y)
        : "memory");
  }
}
// Whether the phase is over already; does not wait.
SB_DEVICE bool mbar_test(uint64_t* bar, uint32_t phase) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(phase)
      : "memory");
  return ok != 0;
}
// The same without ordering this thread's memory accesses before it: for an
// accumulator that has been read.  What orders it is tcgen05.wait::ld: after it
// the columns are in registers, so nothing of the reads is left that the next
// products could overtake, and nothing else is handed over.  (The releasing
// form waits for the global stores before it, 600 clocks.)
template <int CTAS>
SB_DEVICE void arrive_leader_relaxed(uint64_t* bar) {
  if constexpr (CTAS == 1) {
    mbar_arrive(bar);
  } else {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(leader_addr(bar)) : "memory");
  }
}
template <int CTAS>
SB_DEVICE void tmem_take(uint32_t* slot, uint32_t cols) {
  if constexpr (CTAS == 1) {
    tmem_alloc(slot, cols);
    tmem_relinquish();
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
}
template <int CTAS>
SB_DEVICE void tmem_give(uint32_t taddr, uint32_t cols) {
  if constexpr (CTAS == 1) tmem_dealloc(taddr, cols);
  else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}
template <int CTAS>
SB_DEVICE void sync_pair() {
  if constexpr (CTAS == 1) {
    __syncthreads();
  } else {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  }
}

// 16 staged bytes to D: sums (fp32, to be added or not) or finished bf16 values.
// `here` values of them, at `at` elements from `out`.
SB_DEVICE void store_some(const Args& p, const uint8_t* staged, uint8_t* out, long at, int here) {
  if (p.f32 || p.acc) {
    const float4 w = *reinterpret_cast<const float4*>(staged);
    float f[4] = {w.x, w.y, w.z, w.w};
    if (p.f32) {
      float* d = reinterpret_cast<float*>(out) + at;
      if (p.d_vec && here == 4) {
        float4 o = p.acc ? *reinterpret_cast<const float4*>(d) : make_float4(0.f, 0.f, 0.f, 0.f);
        *reinterpret_cast<float4*>(d) = make_float4(f[0] + o.x, f[1] + o.y, f[2] + o.z, f[3] + o.w);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < here) d[i] = p.acc ? d[i] + f[i] : f[i];
      }
    } else {
      __nv_bfloat16* d = reinterpret_cast<__nv_bfloat16*>(out) + at;
      if (p.d_vec && here == 4) {
        const uint2 o = *reinterpret_cast<const uint2*>(d);
        const float2 a = unpack_bf16x2(o.x), b = unpack_bf16x2(o.y);
        *reinterpret_cast<uint2*>(d) = make_uint2(pack_bf16x2(f[0] + a.x, f[1] + a.y), pack_bf16x2(f[2] + b.x, f[3] + b.y));
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < here) d[i] = __float2bfloat16(__bfloat162float(d[i]) + f[i]);
      }
    }
  } else {
    const uint4 w = *reinterpret_cast<const uint4*>(staged);
    const uint32_t e[4] = {w.x, w.y, w.z, w.w};
    uint16_t* d = reinterpret_cast<uint16_t*>(out) + at;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < here) d[i] = static_cast<uint16_t>(e[i / 2] >> (16 * (i % 2)));
  }
}

// Row and column tile of number `local` among tiles_m x tiles_n: bands of
// kBand row tiles, rows first, so that the tiles in flight at one time share
// few rows of both operands.
SB_DEVICE void walk(const Args& p, int local, int tiles_m, int& tm, int& tn) {
  const int band = p.by_band(local);
  const int height = min(kBand, tiles_m - band * kBand);
  const int in = local - band * kBand * p.tiles_n;
  tn = height == kBand ? in / kBand : static_cast<int>(static_cast<unsigned>(in) / static_cast<unsigned>(height));
  tm = band * kBand + in - tn * height;
}

// The blocks that a tile contracts, all that the issuer has to know.
SB_DEVICE void tile_blocks(const Args& p, const int* s_prefix, const int* s_offs, int tile, int& kb0, int& kb) {
  if (p.mode == kKGroups) {
    const int g = p.by_tiles(tile);
    kb0 = s_offs[g] / BK;
    kb = (s_offs[g + 1] - s_offs[g] + BK - 1) / BK;
    return;
  }
  kb0 = 0;
  kb = (p.K + BK - 1) / BK;
  if (p.split > 1) {                               // 2^24 blocks by 148 ranges at most: 32 bits hold it
    const unsigned s = p.by_tiles(tile), blocks = kb;
    kb0 = blocks * s / p.split;
    kb = blocks * (s + 1) / p.split - kb0;
  }
}

// `rank`: the CTA's place in its pair.
template <int BN, int CTAS>
__device__ __forceinline__ Tile decode_tile(const Args& p, const int* s_prefix, const int* s_offs, int tile, int rank) {
  using C = Cfg<BN, CTAS>;
  Tile t;
  int tm, tn;
  tile_blocks(p, s_prefix, s_offs, tile, t.kb0, t.kb);
  if (p.mode == kRowGroups) {
    int lo = 0, hi = p.G - 1;                      // last group whose first tile is at most `tile`
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (s_prefix[mid] <= tile) lo = mid;
      else hi = mid - 1;
    }
    int local = tile - s_prefix[lo], s = 0;
    const int rows = s_offs[lo + 1] - s_offs[lo], tiles_m = (rows + C::kTileM - 1) / C::kTileM;
    if (p.split > 1) {
      s = p.by_tiles(local);
      local -= s * p.by_tiles.d;
    }
    walk(p, local, tiles_m, tm, tn);
    const int m = tm * C::kTileM + rank * BM;
    t.n0 = tn * BN;
    t.a_row = s_offs[lo] + m;
    t.b_row = lo * p.N + t.n0;
    t.d_row = t.a_row + static_cast<long>(s) * p.M;
    t.m_valid = min(BM, rows - m);
  } else {
    const int g = p.by_tiles(tile);
    walk(p, tile - g * p.by_tiles.d, (p.M + C::kTileM - 1) / C::kTileM, tm, tn);
    const int m = tm * C::kTileM + rank * BM;
    t.n0 = tn * BN;
    t.a_row = m;
    t.b_row = t.n0;
    t.d_row = static_cast<long>(g) * p.M + m;
    t.m_valid = min(BM, p.M - m);
  }
  return t;
}

template <int BN, int CTAS>
__global__ void __launch_bounds__(kThreads, 1) __cluster_dims__(CTAS, 1, 1)
matmul_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
              const Args p) {
  using C = Cfg<BN, CTAS>;
  constexpr int kScaleStages = C::kScaleStages;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* tiles = smem_raw + (((raw_addr + 1023) & ~1023u) - raw_addr);
  uint8_t* epi = tiles + C::kStages * C::kStageBytes;
  uint8_t* scales = epi + C::kEpiBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(scales + kScaleStages * C::kScaleBytes);
  uint64_t* empty = full + C::kStages;
  uint64_t* sf_full = empty + C::kStages;
  uint64_t* sf_empty = sf_full + kScaleStages;
  uint64_t* sf_here = sf_empty + kScaleStages;
  uint64_t* acc_full = sf_here + kScaleStages;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* drain = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  int* s_total = reinterpret_cast<int*>(tmem_slot + 1);
  int* s_offs = s_total + 1;
  int* s_prefix = s_offs + kMaxGroups + 1;

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = CTAS == 1 ? 0 : blockIdx.x % CTAS;

  for (int g = threadIdx.x; g <= p.G; g += kThreads) {
    const int lim = p.mode == kRowGroups ? p.M : p.K;
    s_offs[g] = p.offs != nullptr ? min(max(p.offs[g], 0), lim) : (g == 0 ? 0 : lim);
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < kScaleStages; ++s) {
      mbar_init(&sf_full[s], CTAS);
      mbar_init(&sf_empty[s], 1);
      mbar_init(&sf_here[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], kEpiWarps * CTAS);
    }
    mbar_init(drain, 1);
    fence_barrier_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  if (warp == 3) tmem_take<CTAS>(tmem_slot, C::kTmemCols);
  __syncthreads();
  if (threadIdx.x == 0) {
    int total = 0;
    if (p.mode == kRowGroups) {
      for (int g = 0; g < p.G; ++g) {
        s_prefix[g] = total;
        s_offs[g + 1] = max(s_offs[g + 1], s_offs[g]);
        total += (s_offs[g + 1] - s_offs[g] + C::kTileM - 1) / C::kTileM * p.tiles_n * p.split;
      }
      s_prefix[p.G] = total;
    } else {
      bool ok = true;
      for (int g = 0; g < p.G; ++g) {
        s_offs[g + 1] = max(s_offs[g + 1], s_offs[g]);
        // a segment that starts or ends inside a block would take its neighbour's columns along
        ok &= s_offs[g + 1] == s_offs[g] ||
              (s_offs[g] % BK == 0 && (s_offs[g + 1] % BK == 0 || s_offs[g + 1] == p.K));
      }
      total = ok ? p.G * p.by_tiles.d : 0;
      if (!ok && blockIdx.x == 0) record_status(p.status, kBadShape);
    }
    *s_total = total;
  }
  tc_fence_before();
  sync_pair<CTAS>();          // the other CTA's barriers exist before anything arrives on them
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int first_tile = blockIdx.x / CTAS, tile_step = gridDim.x / CTAS, total = *s_total;

  if (warp == 0) {
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = first_tile; tile < total && ok; tile += tile_step) {
        const Tile t = decode_tile<BN, CTAS>(p, s_prefix, s_offs, tile, rank);
        for (int i = 0; i < t.kb; ++i) {
          if (!mbar_wait(&empty[stage], phase ^ 1, p.status)) { ok = false; break; }
          uint8_t* s = tiles + stage * C::kStageBytes;
          if (rank == 0) mbar_arrive_expect_tx(&full[stage], C::kStageBytes * CTAS);
          load_tile<CTAS>(s, &tmA, &full[stage], (t.kb0 + i) * BK, t.a_row);
          load_tile<CTAS>(s + C::kABytes, &tmB, &full[stage], (t.kb0 + i) * BK, t.b_row + rank * C::kBRows);
          if (++stage == C::kStages) { stage = 0; phase ^= 1; }
        }
      }
      // every stage's products have signalled here before this CTA may go: the other one's signals are remote
      for (int s = 0; s < C::kStages && ok; ++s) {
        ok = mbar_wait(&empty[stage], phase ^ 1, p.status);
        if (++stage == C::kStages) { stage = 0; phase ^= 1; }
      }
      // an early end: wait (briefly) for the loads in flight, which must not land after the CTA has gone
      // (the second CTA's complete on the first one's barriers; the pair leaves together)
      if (!ok && rank == 0)
        for (int s = 0; s < C::kStages; ++s) mbar_wait(&full[s], phase ^ (s < stage ? 0 : 1), nullptr, 200000000ull);
    }
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      const uint64_t desc0 = make_sw128_desc(smem_u32(tiles), 16, 1024);
      int stage = 0, acc = 0, sf = 0;
      uint32_t phase = 0, acc_phase = 0, sf_phase = 0;
      uint32_t sfa = 0;
      bool ok = true, ready = false;
      for (int tile = first_tile; tile < total && ok; tile += tile_step) {
        int kb0, kb;
        tile_blocks(p, s_prefix, s_offs, tile, kb0, kb);
        // its accumulator has been read; one that shares columns with the other also waits until the tile before
        // has read those, which it does first, and the epilogue takes tiles in order
        if (C::kShared) {
          if (tile != first_tile && !wait_both<CTAS>(&acc_empty[acc ^ 1], acc == 0 ? acc_phase ^ 1 : acc_phase, p.status)) {
            ok = false;
            break;
          }
        } else if (!wait_both<CTAS>(&acc_empty[acc], acc_phase ^ 1, p.status)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem + acc * C::kAccCols;
        for (int i = 0; i < kb; ++i) {
          const uint32_t part = (kb0 + i) % 4;         // the byte of the scale words
          if (i == 0 || part == 0) {
            if (!wait_both<CTAS>(&sf_full[sf], sf_phase, p.status)) { ok = false; break; }
            tc_fence_after();
            // step sf of the words has its own columns, free since sf_empty[sf] was signalled
            sfa = tmem + C::kScaleCol0 + sf * C::kScaleCols;
            const uint32_t src = smem_u32(scales + sf * C::kScaleBytes);
#pragma unroll
            for (int q = 0; q < 1 + C::kBParts; ++q) tmem_copy_scales<CTAS>(sfa + 4 * q, src + 512 * q);
          }
          if (!ready && !mbar_wait(&full[stage], phase, p.status)) { ok = false; break; }
          tc_fence_after();
          // all lies below 256 KB: adding to the address field never carries out of its 14 bits
          const uint64_t ad = desc0 + stage * (C::kStageBytes >> 4), bd = ad + (C::kABytes >> 4);
          const uint32_t idesc = p.idesc | (part << 29) | (part << 4);
#pragma unroll
          for (int kk = 0; kk < BK / 32; ++kk)
            umma_scaled<CTAS>(d, ad + 2 * kk, bd + 2 * kk, idesc, sfa, sfa + 4, (i | kk) != 0 ? 1u : 0u);
          commit<CTAS>(&empty[stage]);
          if (++stage == C::kStages) { stage = 0; phase ^= 1; }
          ready = mbar_test(&full[stage], phase);      // asked early: the answer takes 100 clocks
          if (part == 3 || i == kb - 1) {
            commit<CTAS>(&sf_empty[sf]);
            if (++sf == kScaleStages) { sf = 0; sf_phase ^= 1; }
          }
        }
        if (!ok) break;
        commit<CTAS>(&acc_full[acc]);
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
      }
      // whatever was issued is done before tensor memory is given back, after an early end too
      commit_here<CTAS>(drain);
      mbar_wait(drain, 0, p.status);
    }
  } else if (warp == 2) {
    // Words of kAhead steps are in flight in registers: one step feeds four blocks of products, less than a load takes.
    constexpr int kAhead = 4, kWords = 4 * (1 + C::kBParts);
    int sf = 0, tile = first_tile - tile_step, w = 0, w_end = -1;
    uint32_t sf_phase = 0;
    bool ok = true;
    Tile t = {};
    uint32_t v[kAhead][kWords];
    auto fetch = [&](uint32_t (&to)[kWords]) -> bool {
      if (++w > w_end) {
        do {
          tile += tile_step;
          if (tile >= total) return false;
          t = decode_tile<BN, CTAS>(p, s_prefix, s_offs, tile, rank);
        } while (t.kb == 0);
        w = t.kb0 / 4;
        w_end = (t.kb0 + t.kb - 1) / 4;
      }
      const uint32_t* wa = p.sa + static_cast<long>(w) * p.rows_a;
      const uint32_t* wb = p.sb + static_cast<long>(w) * p.rows_b;
#pragma unroll
      for (int q = 0; q < kWords; ++q) {
        const int row = q < 4 ? t.a_row + q * 32 + lane : t.b_row + (q - 4) * 32 + lane;
        to[q] = row < (q < 4 ? p.rows_a : p.rows_b) ? __ldg((q < 4 ? wa : wb) + row) : 0u;
      }
      return true;
    };
    auto hand_over = [&](const uint32_t (&from)[kWords]) {
      ok = mbar_wait(&sf_empty[sf], sf_phase ^ 1, p.status);
      if (!ok) return;
      uint8_t* dst = scales + sf * C::kScaleBytes + lane * 16;
#pragma unroll
      for (int q = 0; q < 1 + C::kBParts; ++q)
        *reinterpret_cast<uint4*>(dst + 512 * q) =
            make_uint4(from[4 * q], from[4 * q + 1], from[4 * q + 2], from[4 * q + 3]);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(CTAS == 1 ? &sf_full[sf] : &sf_here[sf]);
      if (++sf == kScaleStages) { sf = 0; sf_phase ^= 1; }
    };
    // the first step goes out alone, before time is spent on the next ones
    bool have[kAhead];
    have[0] = fetch(v[0]);
    if (have[0]) {
      hand_over(v[0]);
#pragma unroll
      for (int j = 0; j < kAhead; ++j) have[j] = (j == 0 || have[j - 1]) && fetch(v[j]);
    }
    while (ok && have[0]) {
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        if (!ok || !have[j]) continue;
        hand_over(v[j]);
        have[j] = tile < total && fetch(v[j]);
      }
    }
    for (int s = 0; s < kScaleStages && ok; ++s) {
      ok = mbar_wait(&sf_empty[sf], sf_phase ^ 1, p.status);
      if (++sf == kScaleStages) { sf = 0; sf_phase ^= 1; }
    }
  } else if (warp == 3) {
    // Tells the first CTA that words have come.  A lane of warp 2 cannot: arriving at another CTA's barrier
    // releases, which waits for all loads of the lane, also those of the words to come.
    if (CTAS == 2 && elect_one()) {
      int sf = 0;
      uint32_t sf_phase = 0;
      bool ok = true;
      for (int tile = first_tile; tile < total && ok; tile += tile_step) {
        int kb0, kb;
        tile_blocks(p, s_prefix, s_offs, tile, kb0, kb);
        for (int w = kb0 / 4; kb > 0 && w <= (kb0 + kb - 1) / 4; ++w) {
          if (!mbar_wait(&sf_here[sf], sf_phase, p.status)) { ok = false; break; }
          arrive_leader<CTAS>(&sf_full[sf]);
          if (++sf == kScaleStages) { sf = 0; sf_phase ^= 1; }
        }
      }
    }
  } else if (warp >= 4) {
    const int quarter = warp % 4, half = (warp - 4) / 4;
    const int r = quarter * 32 + lane;
    uint8_t* buf = epi + (warp - 4) * 4096;
    int acc = 0;
    uint32_t acc_phase = 0;
    // piece j of a staged row, turned so that neither a column of pieces nor a row meets a bank twice
    auto staged_at = [](int row, int j) { return (row * 8 + (j ^ (row % 8))) * 16; };
    for (int tile = first_tile; tile < total; tile += tile_step) {
      const Tile t = decode_tile<BN, CTAS>(p, s_prefix, s_offs, tile, rank);
      if (!mbar_wait(&acc_full[acc], acc_phase, p.status)) break;
      tc_fence_after();
      const uint32_t src = tmem + acc * C::kAccCols + ((quarter * 32) << 16);
      const int cols = min(BN, p.N - t.n0);
      // A warp's 32 rows of 128 bytes go through shared memory, so that each global store covers whole runs of
      // rows: 64 columns that leave as bf16, or 32 that leave as fp32 or are added to what D holds.
      const bool wide = p.f32 || p.acc;
      const int step = wide ? 32 : 64;
      const int n = (cols + step - 1) / step;
      if (half >= n && lane == 0) arrive_leader_relaxed<CTAS>(&acc_empty[acc]);    // nothing for this warp to read
      const int rows_here = min(32, t.m_valid - quarter * 32);
      uint8_t* const out = static_cast<uint8_t*>(p.D) + ((t.d_row + quarter * 32) * p.ldd + t.n0) * (p.f32 ? 4 : 2);
#pragma unroll 1
      for (int i = half; i < n; i += 2) {
        // shared columns first: the last of the first accumulator, the first of the second
        const int s = C::kShared && acc == 0 ? n - 1 - i : i;
        uint32_t v[64];
        __syncwarp();                                  // the buffer has been read, the warp is whole
        tmem_ld_32x32b_x32(src + s * step, v);
        if (!wide) tmem_ld_32x32b_x32(src + s * step + 32, v + 32);
        tmem_wait_ld();
        if (C::kShared ? i < 2 : i + 2 >= n) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_leader_relaxed<CTAS>(&acc_empty[acc]);
        }
        if (rows_here <= 0) continue;
        if (t.kb == 0) {
#pragma unroll
          for (int j = 0; j < 64; ++j) v[j] = 0u;      // nothing was contracted: zeros
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint4 w = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          if (!wide) {
            const bf16x8 h = float_to_bf16x8(reinterpret_cast<const float*>(v) + 8 * j);
            w = make_uint4(h.w[0], h.w[1], h.w[2], h.w[3]);
          }
          *reinterpret_cast<uint4*>(buf + staged_at(lane, j)) = w;
        }
        __syncwarp();
        const int r0 = lane / 8, j = lane % 8, per = wide ? 4 : 8, c = s * step + j * per;
        const int here = min(per, cols - c);           // of this lane's 16 bytes
        if (p.d_vec && here == per && !p.acc) {
          uint8_t* d = out + (r0 * p.ldd + c) * (p.f32 ? 4 : 2);
          const long jump = 4 * p.ldd * (p.f32 ? 4 : 2);
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const int row = q * 4 + r0;
            const uint4 w = *reinterpret_cast<const uint4*>(buf + staged_at(row, j));
            if (row < rows_here) *reinterpret_cast<uint4*>(d) = w;
            d += jump;
          }
        } else if (here > 0) {
#pragma unroll 1
          for (int row = r0; row < rows_here; row += 4)
            store_some(p, buf + staged_at(row, j), out, row * p.ldd + c, here);
        }
      }
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
    }
  }

  tc_fence_before();
  sync_pair<CTAS>();
  tc_fence_after();
  if (warp == 3) tmem_give<CTAS>(tmem, C::kTmemCols);
}

// Sum of the partial products of a split contraction, in the order of the
// ranges, into D with the requested type and accumulation; four columns a
// thread (ranges of ws are rows of N rounded up to 4).
__global__ void split_sum_kernel(const float* __restrict__ ws, int S, int M, int N, Divisor by_quads, bool f32, bool acc,
                                 bool vec, void* D, long ldd) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  const int m = by_quads(i), c = (i - m * static_cast<int>(by_quads.d)) * 4;
  if (m >= M) return;
  const long range = static_cast<long>(M) * by_quads.d;
  const float4* src = reinterpret_cast<const float4*>(ws) + i;
  float4 v = src[0];
#pragma unroll 4
  for (int s = 1; s < S; ++s) {
    const float4 w = src[s * range];
    v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
  }
  const float f[4] = {v.x, v.y, v.z, v.w};
  const long at = m * ldd + c;
  if (f32) {
    float* d = static_cast<float*>(D) + at;
    if (vec) {
      const float4 o = acc ? *reinterpret_cast<const float4*>(d) : make_float4(0.f, 0.f, 0.f, 0.f);
      *reinterpret_cast<float4*>(d) = make_float4(f[0] + o.x, f[1] + o.y, f[2] + o.z, f[3] + o.w);
      return;
    }
    for (int j = 0; j < 4 && c + j < N; ++j) d[j] = acc ? d[j] + f[j] : f[j];
  } else {
    __nv_bfloat16* d = static_cast<__nv_bfloat16*>(D) + at;
    for (int j = 0; j < 4 && c + j < N; ++j)
      d[j] = __float2bfloat16(acc ? __bfloat162float(d[j]) + f[j] : f[j]);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeFn encode_fn() {
  static EncodeFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q);
    TORCH_CHECK(e == cudaSuccess && q == cudaDriverEntryPointSuccess && ptr != nullptr,
                "shift_b200: cannot resolve cuTensorMapEncodeTiled");
    fn = reinterpret_cast<EncodeFn>(ptr);
  });
  return fn;
}

// Row-major bytes [rows, cols] with row stride `bytes`, boxes of 128 bytes x box_rows, 128-byte swizzle.
static CUtensorMap make_map(const void* base, long rows, long cols, long bytes, int box_rows) {
  CUtensorMap m;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(bytes)};
  cuuint32_t box[2] = {128, static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = encode_fn()(&m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed with code ", static_cast<int>(r));
  return m;
}

static int num_sms(int device) {
  static int n[64] = {};
  int& v = n[device & 63];
  if (v == 0) cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, device);
  return v;
}

template <int BN, int CTAS>
static void launch(const CUtensorMap& ta, const CUtensorMap& tb, const Args& p, long tiles,
                   int device, cudaStream_t st) {
  using C = Cfg<BN, CTAS>;
  auto kern = matmul_kernel<BN, CTAS>;
  static std::atomic<uint64_t> ready{0};          // devices that know the kernel's shared memory size
  const uint64_t bit = 1ull << (device & 63);
  if ((ready.load(std::memory_order_relaxed) & bit) == 0) {
    C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes));
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  const int grid = static_cast<int>(std::min<long>(num_sms(device) / CTAS, std::max<long>(1, tiles))) * CTAS;
  kern<<<grid, kThreads, C::kSmemBytes, st>>>(ta, tb, p);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

struct Plan {
  int ctas, bn, split;
  long tiles;            // upper bound for the grid
};

// Up to 128 rows take one CTA per tile (a pair would compute 128 rows of
// nothing: 1 x 32768 x 1024 in 13 us against 20), more a pair.  The width is
// the one with the least columns walked by the busiest CTA or pair, with 64
// added per tile for what a tile costs whatever its width.  128 columns count
// as 176: per block they bring 24 KB into an SM for 256 clocks of products,
// where 64 bytes a clock arrive.  Measured, 192 against 256 columns: 16384 x
// 1536 x 1024 27.6 and 29.1 us, 16384 x 1024 x 1024 23.4 and 21.9 us.  The split
// is looked at after the width: 1536 x 1024 x 16384 takes 48 tiles of 128
// columns on 74 pairs and is not split (50 us).
static Plan make_plan(long M, long N, long K, long G, int64_t mode, bool offs, int sms) {
  Plan p;
  const long blocks = (K + BK - 1) / BK;
  p.ctas = M > BM ? 2 : 1;
  const long slots = sms / p.ctas, tm = (M + BM * p.ctas - 1) / (BM * p.ctas);
  long best = -1;
  for (int bn : {256, 224, 192, 128}) {
    if (bn == 256 && p.ctas == 1) continue;
    const long tn = (N + bn - 1) / bn, tiles = mode == kRowGroups ? tm * tn : G * tm * tn;
    const long cost = (tiles + slots - 1) / slots * ((bn == 128 ? 176 : bn) + 64);
    if (best >= 0 && cost >= best) continue;
    best = cost;
    p.bn = bn;
    p.tiles = mode == kRowGroups ? (tm + (offs ? G : 0)) * tn : tiles;
  }
  // few tiles over a long contraction: ranges of at least four blocks to the CTAs that would have none
  p.split = 1;
  if (!offs && p.tiles * 2 <= slots && blocks >= 8) {
    p.split = static_cast<int>(std::min<long>(slots / p.tiles, blocks / 4));
    p.tiles *= p.split;
  }
  return p;
}

static void check_operand(const at::Tensor& q, const at::Tensor& scale, int64_t cols) {
  const auto t = q.scalar_type();
  TORCH_CHECK_VALUE(q.dim() == 2 && (t == at::kFloat8_e4m3fn || t == at::kFloat8_e5m2),
                    "fp8 product: codes are a matrix of float8_e4m3fn or float8_e5m2, got ", t);
  TORCH_CHECK_VALUE(cols >= 0 && q.size(1) >= cols, "fp8 product: ", q.size(1), " columns of codes, ", cols, " are said");
  TORCH_CHECK_VALUE(scale.scalar_type() == at::kFloat8_e8m0fnu && scale.is_contiguous() && scale.dim() == 3 &&
                        scale.size(0) == (cols + 511) / 512 && scale.size(1) == q.size(0) && scale.size(2) == 4,
                    "fp8 product: scales [", (cols + 511) / 512, ", ", q.size(0),
                    ", 4] of float8_e8m0fnu, contiguous, got ", scale.sizes(), " of ", scale.scalar_type());
  // four scales are read as one word; a view of bytes can start anywhere
  TORCH_CHECK_VALUE((reinterpret_cast<uintptr_t>(scale.data_ptr()) & 3) == 0, "fp8 product: scales start on 4 bytes");
  TORCH_CHECK_VALUE(scale.device() == q.device() && q.is_cuda(), "fp8 product: codes and scales on one CUDA device");
}

// a, b: codes [rows, ld] with scales [words, rows, 4] and `K` columns each.
// Without offs: out [a.rows, b.rows].  With offs [G + 1]: mode 0 (row groups)
// out [a.rows, b.rows / G], mode 1 (K groups) out [G, a.rows, b.rows].  An out
// that is not given is made, in fp32 or bf16.
at::Tensor matmul(const at::Tensor& a, const at::Tensor& sa, int64_t K, const at::Tensor& b, const at::Tensor& sb,
                  int64_t Kb, const c10::optional<at::Tensor>& out, const c10::optional<at::Tensor>& offs, int64_t mode,
                  bool accumulate, bool make_f32, const at::Tensor& status) {
  // a contraction by segments is never cut into ranges: without segments it has no form
  TORCH_CHECK_VALUE(mode == kRowGroups || (mode == kKGroups && offs.has_value()), "fp8 product: groups of the contraction need offs");
  check_operand(a, sa, K);
  check_operand(b, sb, Kb);
  TORCH_CHECK_VALUE(K == Kb, "fp8 product: the operands contract ", K, " and ", Kb, " values");
  TORCH_CHECK_VALUE(a.device() == b.device(), "fp8 product: operands on ", a.device(), " and ", b.device());
  int64_t G = 1;
  if (offs.has_value()) {
    TORCH_CHECK_VALUE(offs->dim() == 1 && offs->numel() >= 2 && offs->scalar_type() == at::kInt && offs->is_contiguous() &&
                          offs->device() == a.device(),
                      "fp8 product: offs are int32 [groups + 1] on the operands' device");
    G = offs->numel() - 1;
    TORCH_CHECK_VALUE(mode == kKGroups || b.size(0) % G == 0, "fp8 product: ", b.size(0), " rows of b for ", G, " groups");
  }
  const int64_t M = a.size(0), N = mode == kRowGroups ? b.size(0) / G : b.size(0);
  TORCH_CHECK_VALUE(out.has_value() || !accumulate, "fp8 product: accumulate needs out");
  const at::cuda::CUDAGuard guard(a.device());
  at::Tensor result = out.has_value() ? *out : at::empty({M, N}, a.options().dtype(make_f32 ? at::kFloat : at::kBFloat16));
  if (mode == kKGroups) {
    TORCH_CHECK_VALUE(result.dim() == 3 && result.size(0) == G && result.size(1) == M && result.size(2) == N &&
                          result.is_contiguous(),
                      "fp8 product: out ", result.sizes(), ", expected [", G, ", ", M, ", ", N, "], contiguous");
  } else {
    TORCH_CHECK_VALUE(result.dim() == 2 && result.size(0) == M && result.size(1) == N && (N <= 1 || result.stride(1) == 1),
                      "fp8 product: out ", result.sizes(), ", expected [", M, ", ", N, "] with inner stride 1");
    TORCH_CHECK_VALUE(M <= 1 || N == 0 || result.stride(0) >= N, "fp8 product: rows of out overlap");
  }
  TORCH_CHECK_VALUE(result.scalar_type() == at::kFloat || result.scalar_type() == at::kBFloat16,
                    "fp8 product: out in bf16 or fp32, got ", result.scalar_type());
  TORCH_CHECK_VALUE(result.device() == a.device(), "fp8 product: out on ", result.device(), ", operands on ", a.device());
  const at::Tensor D = mode == kKGroups ? result.view({G * M, N}) : result;
  TORCH_CHECK(M < (1l << 31) - 256 && N < (1l << 31) - 256 && K < (1l << 31) - 256 && G * M < (1l << 31) - 256 &&
                  b.size(0) < (1l << 31) - 256,
              "fp8 matmul: a side is too long");
  TORCH_CHECK(G >= 1 && G <= kMaxGroups, "fp8 matmul: 1 to ", kMaxGroups, " groups");
  if (M == 0 || N == 0) return result;
  if (K == 0) {                                    // nothing to contract: zeros, by group in the rows of the segments
    if (accumulate) return result;
    if (mode == kKGroups || !offs.has_value()) {
      D.zero_();
    } else {
      const at::Tensor row = at::arange(M, offs->options());
      D.masked_fill_(row.ge(offs->narrow(0, 0, 1)).__and__(row.lt(offs->max())).unsqueeze(1), 0);
    }
    return result;
  }
  for (const auto* t : {&a, &b})                   // a tensor map's strides are whole: no row repeats another
    TORCH_CHECK_VALUE(t->size(0) <= 1 || t->stride(0) >= K, "fp8 product: rows of codes overlap");
  for (const auto* t : {&a, &b})
    TORCH_CHECK(t->stride(1) == 1 && aligned16(t->data_ptr()) && (t->size(0) == 1 || t->stride(0) % 16 == 0),
                "fp8 matmul: codes start on 16 bytes, rows a multiple of 16 bytes apart");
  const auto st = at::cuda::getCurrentCUDAStream();
  const int sms = num_sms(a.device().index());
  Args p;
  p.sa = static_cast<const uint32_t*>(sa.data_ptr());
  p.sb = static_cast<const uint32_t*>(sb.data_ptr());
  p.rows_a = static_cast<int>(a.size(0));
  p.rows_b = static_cast<int>(b.size(0));
  p.M = static_cast<int>(M);
  p.N = static_cast<int>(N);
  p.K = static_cast<int>(K);
  p.G = static_cast<int>(G);
  p.mode = static_cast<int>(mode);
  p.offs = offs.has_value() ? offs->data_ptr<int>() : nullptr;
  p.status = status.data_ptr<int>();

  const Plan plan = make_plan(M, N, K, G, mode, p.offs != nullptr, sms);
  const int bn = plan.bn;
  const long tiles = plan.tiles;
  p.split = plan.split;
  p.tiles_n = static_cast<int>((N + bn - 1) / bn);
  p.by_band.set(kBand * p.tiles_n);
  p.by_tiles.set(static_cast<unsigned>((M + BM * plan.ctas - 1) / (BM * plan.ctas) * p.tiles_n));

  at::Tensor ws;
  const long quads = (N + 3) / 4;
  const bool f32 = D.scalar_type() == at::kFloat;
  p.f32 = f32;
  p.acc = accumulate;
  p.D = D.data_ptr();
  p.ldd = D.size(0) > 1 ? D.stride(0) : N;
  if (p.split > 1) {
    ws = at::empty({p.split * M, quads * 4}, a.options().dtype(at::kFloat));
    p.f32 = true;
    p.acc = false;
    p.D = ws.data_ptr();
    p.ldd = quads * 4;
  }
  const int es = p.f32 ? 4 : 2;
  p.d_vec = aligned16(p.D) && (p.ldd * es) % 16 == 0;
  // fp32 accumulator, both operands K-major, UE8M0 scales; the byte of the scale words is added per block
  p.idesc = (static_cast<uint32_t>(a.scalar_type() == at::kFloat8_e5m2) << 7) |
            (static_cast<uint32_t>(b.scalar_type() == at::kFloat8_e5m2) << 10) |
            (static_cast<uint32_t>(bn >> 3) << 17) | (1u << 23) | (static_cast<uint32_t>((BM * plan.ctas) >> 4) << 24);

  const long lda = a.size(0) > 1 ? a.stride(0) : (K + 15) / 16 * 16, ldb = b.size(0) > 1 ? b.stride(0) : (K + 15) / 16 * 16;
  const CUtensorMap ta = make_map(a.data_ptr(), a.size(0), K, lda, BM);
  const CUtensorMap tb = make_map(b.data_ptr(), b.size(0), K, ldb, bn / plan.ctas);
  const int dev = a.device().index();
  if (plan.ctas == 2) {
    if (bn == 256) launch<256, 2>(ta, tb, p, tiles, dev, st);
    else if (bn == 224) launch<224, 2>(ta, tb, p, tiles, dev, st);
    else if (bn == 192) launch<192, 2>(ta, tb, p, tiles, dev, st);
    else launch<128, 2>(ta, tb, p, tiles, dev, st);
  } else {
    if (bn == 224) launch<224, 1>(ta, tb, p, tiles, dev, st);
    else if (bn == 192) launch<192, 1>(ta, tb, p, tiles, dev, st);
    else launch<128, 1>(ta, tb, p, tiles, dev, st);
  }
  if (p.split > 1) {
    const long n = M * quads, ldd = D.size(0) > 1 ? D.stride(0) : N;
    TORCH_CHECK(n < (1l << 31) - 256, "fp8 matmul: too large to split");
    Divisor by_quads;
    by_quads.set(static_cast<unsigned>(quads));
    const bool vec = N % 4 == 0 && aligned16(D.data_ptr()) && ldd % 4 == 0;
    split_sum_kernel<<<static_cast<unsigned>((n + 127) / 128), 128, 0, st>>>(
        ws.data_ptr<float>(), p.split, p.M, p.N, by_quads, f32, accumulate, vec, D.data_ptr(), ldd);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
  return result;
}

}  // namespace fp8
}  // namespace sb

// Backward kernels of causal attention over packed sequences (attention_packed.cuh has the design).
//
// Two passes, each with the products it needs, so that every sum stays in one tensor memory accumulator and no order hangs
// on timing: dK / dV by tiles of 128 keys (S^T = K Q^T, dP^T = V dO^T, dV += P^T dO, dK += dS^T Q), dQ by tiles of 128
// queries (S = Q K^T, dP = dO V^T, dQ += dS K).  Seven products instead of five; one pass would add dQ across CTAs in the
// order in which they get there.
//
// The other side comes in blocks of 128, of which each group of softmax warps has 64 columns; S and dP have columns of their
// own in tensor memory and P and dS have too, so that S and dP of the next block are computed while the groups are still at
// this one (blocks of 64 that the groups took in turn: 412 us where this took 335, 8 x 2048 rows, 16 / 4 heads of 64).  The
// dK / dV pass of heads of 128 has no columns left for that: its blocks are of 64, the groups take them in turn, and P and dS
// lie over S and dP.
//
// At those sizes (heads of 64) the products take 1024 of the 2290 clocks that a 128 x 128 block of the dK / dV pass takes,
// and 768 of 2180 of the dQ pass; the rest is the chain scores - exponentials - operands of one block.  Four groups of warps
// instead of two, with 32 columns a thread, take as long.
#include "attention_packed.cuh"

namespace sb {
namespace pa {

constexpr int kOnFma = 2;          // of 8 exponentials, those computed on the FMA pipe (of 64, 8 x 2048: 343 us, 1: 345)

// kUpP - lse log2(e) and -delta of every query, [Hq][2 tiles][2][64]; zeros for rows of no sequence.  Eight or sixteen lanes
// have a row of a head.
template <int D, typename T>
__global__ void __launch_bounds__(256) rows_kernel(const __grid_constant__ Args a, float* __restrict__ out) {
  constexpr int L = D / 8;
  const long i = static_cast<long>(blockIdx.x) * (256 / L) + threadIdx.x / L;
  const int sub = threadIdx.x % L, h = static_cast<int>(i % a.Hq);
  const long row = i / a.Hq;
  const bool there = row < static_cast<long>(a.tiles) * 128;   // the same in all L lanes of a group
  const unsigned lanes = (L == 8 ? 0xffu : 0xffffu) << (threadIdx.x % 32 / L * L);
  float s = 0.f, nl = 0.f, top = 0.f;
  if (there && row < a.T && a.start[row] <= row) {
    const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.o) + row * a.o_ld + static_cast<long>(h) * D + sub * 8);
    const uint4 g = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.dout) + row * a.do_ld + static_cast<long>(h) * D + sub * 8);
    const T *x = reinterpret_cast<const T*>(&u), *y = reinterpret_cast<const T*>(&g);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      s += to_float(x[k]) * to_float(y[k]);
      top = fmaxf(top, fabsf(to_float(y[k])));
    }
    nl = fmaf(-a.lse[static_cast<long>(h) * a.T + row], kLog2e, static_cast<float>(kUpP<T>));
  }
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) s += __shfl_xor_sync(lanes, s, o);
  if (a.tops != nullptr) {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(lanes, top, o));
    if (there && sub == 0) a.tops[static_cast<long>(h) * (a.tiles * 128) + row] = top;
  }
  if (there && sub == 0) {
    float* p = out + (static_cast<long>(h) * (a.tiles * 2) + row / 64) * 128 + row % 64;
    p[0] = nl;
    p[64] = -s;
  }
}

// fp16: every key's shift, from the largest |do| of the rows that see it.  A CTA has 1024 rows of a key head: maxima from a row
// to its sequence's end within a warp, then over the warps behind it, then over what the sequence has behind the CTA's rows,
// which it reads itself (for one sequence of n rows that is n^2 / 2048 values in all, beside n^2 / 2 products).
__global__ void __launch_bounds__(1024) shift_kernel(const __grid_constant__ Args a) {
  __shared__ float first[32], behind[32];
  const long pad = static_cast<long>(a.tiles) * 128;
  const float* tops = a.tops + static_cast<long>(blockIdx.y) * a.group * pad;
  const int c0 = blockIdx.x * 1024, row = c0 + threadIdx.x, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  auto top_of = [&](int r) {
    float m = 0.f;
    for (int h = 0; h < a.group; ++h) m = fmaxf(m, tops[h * pad + r]);
    return m;
  };
  const int stop = row < a.T ? a.stop[row] : row;      // of a row of no sequence: the row itself
  float m = row < a.T ? top_of(row) : 0.f;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const float other = __shfl_down_sync(0xffffffffu, m, o);
    if (lane + o < 32 && row + o < stop) m = fmaxf(m, other);
  }
  if (lane == 0) first[warp] = m;
  const int c1 = min(c0 + 1024, a.T), end = a.stop[c1 - 1];
  float far = 0.f;
#pragma unroll 4
  for (int r = c1 + threadIdx.x; r < end; r += 1024) far = fmaxf(far, top_of(r));
  far = warp_max(far);
  if (lane == 0) behind[warp] = far;
  __syncthreads();
  for (int w = warp + 1; w < 32 && c0 + w * 32 < stop; ++w) m = fmaxf(m, first[w]);
  if (stop > c1)
    for (int w = 0; w < 32; ++w) m = fmaxf(m, behind[w]);
  if (row < pad) a.shifts[blockIdx.y * pad + row] = shift_for(m);
}

// ============================ dK, dV ============================
template <int D>
struct Dkv {
  static constexpr bool kWide = D == 64;
  static constexpr int kW = kWide ? 128 : 64;                                      // queries of a block
  static constexpr int kHalves = D / 64, kTile = kHalves * kChunk, kNext = kW * 128, kBlock = kHalves * kNext;
  static constexpr int kStages = 4, kStage = 2 * kBlock + kW * 8;                  // Q, dO, -lse and -delta of the queries
  // columns: S, dP (wide: one buffer of 2 x 128, else two of 2 x 64) | dV | dK | P, dS (else over S, dP)
  static constexpr int kDp = kW, kP = kWide ? 384 : 0, kDs = 64;
  static constexpr int kSmem = 1024 + 2 * kTile + kStages * kStage + 512;
  static SB_DEVICE int buffer(int g) { return kWide ? 0 : g & 1; }
  static SB_DEVICE int phase(int g) { return (kWide ? g : g >> 1) & 1; }
};

struct DkvItem {
  int kvh, part, k0, first_h, heads, blocks, subs;      // `blocks` of w queries a head
  SB_DEVICE DkvItem(const Args& a, int idx, int w) {
    const int per = a.Hkv * a.split, r = idx % per;
    kvh = r / a.split;
    part = r % a.split;
    heads = a.group / a.split;
    first_h = kvh * a.group + part * heads;
    k0 = a.order[idx / per] * 128;
    const int end = a.stop[min(k0 + 127, a.T - 1)];
    blocks = k0 < a.ends[1] && k0 + 128 > a.ends[0] ? (end - k0 + w - 1) / w : 0;
    subs = blocks * heads;
  }
};

template <int D, typename T>
__global__ void __launch_bounds__(kThreads, 1)
dkv_kernel(const __grid_constant__ CUtensorMap tm128, const __grid_constant__ CUtensorMap tmw,
           const __grid_constant__ CUtensorMap tmo, const __grid_constant__ Args a) {
  using F = Dkv<D>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* sK = smem_raw + (((raw + 1023) & ~1023u) - raw);
  uint8_t* sV = sK + F::kTile;
  uint8_t* sQ = sV + F::kTile;                                  // [stages][Q | dO]
  float* sR = reinterpret_cast<float*>(sQ + F::kStages * 2 * F::kBlock);          // [stages][blocks of 64][2][64]
  uint4* answer = reinterpret_cast<uint4*>(sR + F::kStages * 2 * F::kW);
  uint64_t* bar = reinterpret_cast<uint64_t*>(answer + 2);
  uint64_t *kv_full = bar, *kv_empty = bar + 1, *land = bar + 2, *acc_full = bar + 3, *acc_free = bar + 4, *drain = bar + 5;
  uint64_t *in_full = bar + 6, *in_empty = in_full + F::kStages, *s_full = in_empty + F::kStages, *p_full = s_full + 2;
  uint64_t *s_empty = p_full + 2, *p_free = s_empty + 2;
  const Sched sched{answer, p_free + 2, p_free + 4};
  uint32_t* tslot = reinterpret_cast<uint32_t*>(p_free + 6);
  int* lists = reinterpret_cast<int*>(tslot + 1);      // [8]
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  if (threadIdx.x == 0) {
    mbar_init(kv_full, 1);
    mbar_init(kv_empty, 1);
    mbar_init(land, 1);
    mbar_init(acc_full, 1);
    mbar_init(acc_free, 8);
    mbar_init(drain, 1);
    for (int i = 0; i < F::kStages; ++i) {
      mbar_init(&in_full[i], 1);
      mbar_init(&in_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], F::kWide ? 8 : 4);
      mbar_init(&s_empty[i], 8);
      mbar_init(&p_free[i], 1);
      mbar_init(&sched.full[i], 1);
      mbar_init(&sched.empty[i], kReaders);
    }
    fence_barrier_init();
  }
  if (warp == kIssuer) {
    tmem_alloc(tslot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = *tslot, tdV = tbase + 256, tdK = tbase + 256 + D;

  if (warp >= 8) {
    regs_down<kOtherRegs>();
    if (warp == kLoader) {
      const int first = a.ends[0], last = min(a.ends[1], a.T);
      int g = 0, nkv = 0, nl = 0, asked = 0;
      bool ok = true;
      for (int n = 0, idx = blockIdx.x; idx >= 0 && ok; ++n) {
        if (lane == 0) ok = sched_request(sched, n, a.status);
        ok = __all_sync(0xffffffffu, ok);
        const DkvItem it(a, idx, F::kW);
        if (ok && it.subs > 0) {
          if (lane == 0) {
            ok = mbar_wait(kv_empty, (nkv & 1) ^ 1, a.status);
            if (ok) {
              mbar_arrive_expect_tx(kv_full, 2 * F::kTile);
              for (int c = 0; c < F::kHalves; ++c) {
                tma_load_2d(sK + c * kChunk, &tm128, kv_full, (a.Hq + it.kvh) * D + c * 64, it.k0);
                tma_load_2d(sV + c * kChunk, &tm128, kv_full, (a.Hq + a.Hkv + it.kvh) * D + c * 64, it.k0);
              }
            }
          }
          ++nkv;
          ok = __all_sync(0xffffffffu, ok);
          for (int s = 0; s < it.subs && ok; ++s, ++g) {
            const int st = g % F::kStages, h = it.first_h + s / it.blocks, row = it.k0 + s % it.blocks * F::kW;
            const bool clear = row < first || min(row + F::kW, a.T) > last;
            uint8_t* in = sQ + st * 2 * F::kBlock;
            if (lane == 0) {
              ok = mbar_wait(&in_empty[st], ((g / F::kStages) & 1) ^ 1, a.status);
              if (ok) {
                uint64_t* to = clear ? land : &in_full[st];
                mbar_arrive_expect_tx(to, F::kStage);
                for (int c = 0; c < F::kHalves; ++c) {
                  tma_load_2d(in + c * F::kNext, &tmw, to, h * D + c * 64, row);
                  tma_load_2d(in + F::kBlock + c * F::kNext, &tmo, to, h * D + c * 64, row);
                }
                bulk_load(sR + st * 2 * F::kW, row_block(a, h, row), F::kW * 8, to);
              }
            }
            ok = __all_sync(0xffffffffu, ok);
            if (clear && ok) {
              ok = __all_sync(0xffffffffu, mbar_wait(land, nl & 1, a.status));
              ++nl;
              if (ok) {
                clear_rows(in, F::kW, F::kHalves, F::kNext, row, first, last);
                clear_rows(in + F::kBlock, F::kW, F::kHalves, F::kNext, row, first, last);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&in_full[st]);
              }
            }
          }
        }
        asked = n + 1;
        if (ok) idx = sched_next(sched, n, a.status);
      }
      if (lane == 0) {
        landed(kv_full, 1, nkv);
        landed(in_full, F::kStages, g);
        landed(sched.full, 2, asked);
      }
    } else if (warp == kIssuer) {
      constexpr uint32_t idS = idesc<T>(128, F::kW, 0), idG = idesc<T>(128, D, 1);
      // all of shared memory lies below 256 KB: adding to a descriptor's address field (16-byte units) never carries out
      const uint64_t dk = kdesc(smem_u32(sK)), dv = kdesc(smem_u32(sV)), din = kdesc(smem_u32(sQ));
      const uint64_t din_mn = mndesc(smem_u32(sQ), F::kNext);
      auto scores = [&](int g) -> bool {               // S^T and dP^T of block g to its buffer
        const int st = g % F::kStages;
        if (!mbar_wait(&in_full[st], (g / F::kStages) & 1, a.status)) return false;
        if (F::kWide && g >= 1 && !mbar_wait(&s_empty[0], (g - 1) & 1, a.status)) return false;
        tc_fence_after();
        const uint64_t q = din + st * (2 * F::kBlock >> 4), o = q + (F::kBlock >> 4);
        const uint32_t ts = tbase + F::buffer(g) * 128;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const int off = ((kk >> 2) * kChunk + (kk & 3) * 32) >> 4, sub = ((kk >> 2) * F::kNext + (kk & 3) * 32) >> 4;
          umma_f16(ts, dk + off, q + sub, idS, kk > 0);
        }
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const int off = ((kk >> 2) * kChunk + (kk & 3) * 32) >> 4, sub = ((kk >> 2) * F::kNext + (kk & 3) * 32) >> 4;
          umma_f16(ts + F::kDp, dv + off, o + sub, idS, kk > 0);
        }
        umma_commit(&s_full[F::buffer(g)]);
        return true;
      };
      if (elect_one()) {
      int g = 0, nkv = 0;
      bool ok = true;
      DkvItem it(a, blockIdx.x, F::kW);
      for (int n = 0, idx = blockIdx.x; idx >= 0 && ok; ++n) {
        DkvItem following = it;
        auto look_ahead = [&]() {                      // before the last wait of an item: its loads take a microsecond
          idx = sched_next<false>(sched, n, a.status);
          if (idx >= 0) following = DkvItem(a, idx, F::kW);
        };
        if (it.subs == 0) {
          look_ahead();
        } else {
          ok = mbar_wait(kv_full, nkv & 1, a.status);
          if (ok) ok = scores(g);
          for (int s = 0; s < it.subs && ok; ++s, ++g) {
            if (s + 1 < it.subs) ok = scores(g + 1);
            if (ok && s == max(0, it.subs - 2)) umma_commit(kv_empty);                    // the last scores were issued
            if (ok && s + 1 == it.subs) look_ahead();
            if (ok) ok = mbar_wait(&p_full[F::buffer(g)], F::phase(g), a.status);
            if (ok && s == 0 && nkv > 0) ok = mbar_wait(acc_free, (nkv - 1) & 1, a.status);
            if (!ok) break;
            tc_fence_after();
            const int st = g % F::kStages;
            const uint64_t q = din_mn + st * (2 * F::kBlock >> 4), o = q + (F::kBlock >> 4);
            const uint32_t tp = tbase + F::kP + F::buffer(g) * 128;
#pragma unroll
            for (int kk = 0; kk < F::kW / 16; ++kk) umma_f16_ts(tdV, tp + kk * 8, o + kk * (2048 >> 4), idG, s > 0 || kk > 0);
#pragma unroll
            for (int kk = 0; kk < F::kW / 16; ++kk)
              umma_f16_ts(tdK, tp + F::kDs + kk * 8, q + kk * (2048 >> 4), idG, s > 0 || kk > 0);
            umma_commit(&in_empty[st]);
            if (F::kWide) umma_commit(p_free);
          }
          if (ok) umma_commit(acc_full);
          ++nkv;
        }
        it = following;
      }
      umma_commit(drain);
      mbar_wait(drain, 0, a.status);
      }
      __syncwarp();
    }
  } else {
    regs_up<kSoftRegs>();
    const int w = warp / 4;                            // this group's half of the columns or its buffer; 0 stores dV, 1 dK
    const int b = F::buffer(w);
    const uint32_t lane_off = static_cast<uint32_t>((warp % 4) * 32) << 16;
    const uint32_t ts = tbase + w * (F::kWide ? 64 : 128) + lane_off;
    const uint32_t tp = tbase + F::kP + w * (F::kWide ? 32 : 128) + lane_off;
    const float2 sc2 = make_float2(a.scale_log2, a.scale_log2);
    int g = 0, nkv = 0;
    bool ok = true, in_ready = false, s_ready = false;
    DkvItem it(a, blockIdx.x, F::kW);
    Later later{a.later, -1};
    for (int n = 0, idx = blockIdx.x; idx >= 0 && ok; ++n) {
      const int row = it.k0 + (warp % 4) * 32 + lane;
      const int end = row < a.T ? a.stop[row] : row;
      const int least = a.stop[it.k0];                 // the tile's earliest end
      const int shift = key_shift<T>(a, it.kvh, row);
      const float2 up = make_float2(ldexpf(1.f, shift - kUpP<T>), ldexpf(1.f, shift - kUpP<T>));
      for (int s = 0; s < it.subs; ++s, ++g) {
        if (!F::kWide && (g & 1) != w) continue;
        const int st = g % F::kStages, q0 = it.k0 + s % it.blocks * F::kW + (F::kWide ? w * 64 : 0);
        // -lse and -delta came with Q and dO; S cannot be there before them
        if (!warp_wait(&in_full[st], (g / F::kStages) & 1, a.status, in_ready) ||
            !warp_wait(&s_full[b], F::phase(g), a.status, s_ready)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const bool p_ready = F::kWide && g >= 1 && mbar_test(p_free, (g - 1) & 1);
        const float4* nl4 = reinterpret_cast<const float4*>(sR + st * 2 * F::kW + (F::kWide ? w * 128 : 0));
        const bool masked = q0 < it.k0 + 127 || q0 + 64 > least;
        uint32_t ws[64], wd[64];
        tmem_ld_32x32b_x32(ts, ws);
        tmem_ld_32x32b_x32(ts + F::kDp, wd);
        tmem_ld_32x32b_x32(ts + 32, ws + 32);
        tmem_ld_32x32b_x32(ts + F::kDp + 32, wd + 32);
        tmem_wait_ld();
        if (F::kWide) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(s_empty);
        }
#pragma unroll
        for (int c = 0; c < 64; c += 32) {
          const uint32_t *vs = ws + c, *vd = wd + c;
          uint32_t pp[16], pd[16];
#pragma unroll
          for (int k = 0; k < 32; k += 4) {
            const float4 nl = nl4[(c + k) / 4], nd = nl4[16 + (c + k) / 4];
            float2 z[2], e[2];
            z[0] = fma2(make_float2(__uint_as_float(vs[k]), __uint_as_float(vs[k + 1])), sc2, make_float2(nl.x, nl.y));
            z[1] = fma2(make_float2(__uint_as_float(vs[k + 2]), __uint_as_float(vs[k + 3])), sc2, make_float2(nl.z, nl.w));
            e[0] = add2(make_float2(__uint_as_float(vd[k]), __uint_as_float(vd[k + 1])), make_float2(nd.x, nd.y));
            e[1] = add2(make_float2(__uint_as_float(vd[k + 2]), __uint_as_float(vd[k + 3])), make_float2(nd.z, nd.w));
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              z[u] = (k / 2 + u) % 8 < kOnFma ? ex2_fma(z[u]) : make_float2(ex2(z[u].x), ex2(z[u].y));
              e[u] = mul2(e[u], z[u]);
              pp[k / 2 + u] = Half<T>::pack(z[u].x, z[u].y);
              if constexpr (Half<T>::kFormat == 0) e[u] = mul2(e[u], up);
              pd[k / 2 + u] = Half<T>::pack(e[u].x, e[u].y);
            }
          }
          if (masked) {                                // two packed values at a time
            const uint32_t bits = seen(row - q0 - c, end - 1 - q0 - c);
            if (!__all_sync(0xffffffffu, bits == 0xffffffffu))
#pragma unroll
              for (int k = 0; k < 16; ++k) {
                const uint32_t keep = (bits >> (2 * k) & 1 ? 0xffffu : 0u) | (bits >> (2 * k + 1) & 1 ? 0xffff0000u : 0u);
                pp[k] &= keep;
                pd[k] &= keep;
              }
          }
          if (F::kWide && c == 0 && g >= 1) {          // the products of the block before have read P and dS
            if (!warp_wait(p_free, (g - 1) & 1, a.status, p_ready)) ok = false;
            tc_fence_after();
          }
          tmem_st_32x32b_x16(tp + c / 2, pp);
          tmem_st_32x32b_x16(tp + F::kDs + c / 2, pd);
        }
        if (!ok) break;
        const int next = g + (F::kWide ? 1 : 2);       // this group's; what came before it on these barriers is over
        in_ready = mbar_test(&in_full[next % F::kStages], (next / F::kStages) & 1);
        s_ready = mbar_test(&s_full[b], F::phase(next));
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[b]);
      }
      if (!ok) break;
      const bool covered = row < a.T && end > row;
      const bool dk = w == 1;
      const DkvItem at = it;
      const int item = idx;
      idx = sched_next(sched, n, a.status);            // its tile is looked up while the last products run
      if (idx >= 0) it = DkvItem(a, idx, F::kW);
      const long col = static_cast<long>(a.Hq + (dk ? 0 : a.Hkv) + at.kvh) * D;
      T* out = static_cast<T*>(a.dqkv) + row * a.dqkv_ld + col;
      float* partial = nullptr;
      if (a.split > 1)
        partial = a.partial + ((static_cast<long>(at.part) * a.Hkv + at.kvh) * a.T + row) * (2 * D) + (dk ? 0 : D);
      bool bad = false;
      if (at.subs > 0) {
        if (!__all_sync(0xffffffffu, mbar_wait(acc_full, nkv & 1, a.status))) {
          ok = false;
          break;
        }
        ++nkv;
        tc_fence_after();
        const float f = dk ? ldexpf(a.scale, -shift) : ldexpf(1.f, -kUpP<T>);
        float chk = 0.f;
#pragma unroll
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
          tmem_ld_32x32b_x32((dk ? tdK : tdV) + lane_off + c, o);
          tmem_wait_ld();
          if (c + 32 == D) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_free);
          }
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            const float y = __uint_as_float(o[k]) * f;
            chk = fmaf(y, 0.f, chk);
            o[k] = __float_as_uint(y);
          }
          if (covered && partial != nullptr) {
#pragma unroll
            for (int k = 0; k < 32; k += 4)
              *reinterpret_cast<uint4*>(partial + c + k) = make_uint4(o[k], o[k + 1], o[k + 2], o[k + 3]);
          } else if (covered) {
#pragma unroll
            for (int k = 0; k < 32; k += 8) {
              uint32_t y[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                y[e] = Half<T>::pack(__uint_as_float(o[k + 2 * e]), __uint_as_float(o[k + 2 * e + 1]));
              *reinterpret_cast<uint4*>(out + c + k) = make_uint4(y[0], y[1], y[2], y[3]);
            }
          }
        }
        bad = covered && chk != 0.f;
      }
      if (row < a.T && !covered && a.fill && at.part == 0)
#pragma unroll
        for (int c = 0; c < D; c += 8) *reinterpret_cast<uint4*>(out + c) = make_uint4(0, 0, 0, 0);
      later.add(__ballot_sync(0xffffffffu, bad), item);
    }
    later.run(lists, [&](int item, int finder, int who) {
      const DkvItem at(a, item, F::kW);
      const int row = at.k0 + finder % 4 * 32 + who;
      const bool dk = finder / 4 == 1;
      float* partial = nullptr;
      if (a.split > 1)
        partial = a.partial + ((static_cast<long>(at.part) * a.Hkv + at.kvh) * a.T + row) * (2 * D) + (dk ? 0 : D);
      slow_dkv<D, T>(a, row, at.kvh, at.first_h, at.first_h + at.heads, dk, partial);
    });
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kIssuer) tmem_dealloc(tbase, 512);
}

// Sums of a split, in order: one thread has 8 values of a row's [dK | dV].
template <int D, typename T>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ Args a) {
  const long i = static_cast<long>(blockIdx.x) * 256 + threadIdx.x;
  const int c = static_cast<int>(i % (2 * D / 8)) * 8;
  const long r = i / (2 * D / 8);
  const int row = static_cast<int>(r % a.T), kvh = static_cast<int>(r / a.T);
  if (kvh >= a.Hkv || a.stop[row] <= row) return;
  float s[8] = {};
  for (int p = 0; p < a.split; ++p) {
    const float4* x = reinterpret_cast<const float4*>(a.partial + ((static_cast<long>(p) * a.Hkv + kvh) * a.T + row) * (2 * D) + c);
    const float4 u = x[0], v = x[1];
    s[0] += u.x; s[1] += u.y; s[2] += u.z; s[3] += u.w;
    s[4] += v.x; s[5] += v.y; s[6] += v.z; s[7] += v.w;
  }
  const long col = static_cast<long>(a.Hq + kvh + (c < D ? 0 : a.Hkv)) * D + c % D;
  *reinterpret_cast<uint4*>(static_cast<T*>(a.dqkv) + row * a.dqkv_ld + col) =
      make_uint4(Half<T>::pack(s[0], s[1]), Half<T>::pack(s[2], s[3]), Half<T>::pack(s[4], s[5]), Half<T>::pack(s[6], s[7]));
}

// ============================ dQ ============================
template <int D>
struct Dq {
  static constexpr int kHalves = D / 64, kTile = kHalves * kChunk;
  // tiles of 128 keys: V is done with after the scores, K after dQ
  static constexpr int kK = D == 64 ? 4 : 3, kV = D == 64 ? 4 : 2;
  static constexpr int kP = 256 + D;                                               // S | dP | dQ | dS
  static constexpr int kSmem = 1024 + (2 + kK + kV) * kTile + 512;
};

struct DqItem {
  int h, kvh, q0, lo, hi;                              // blocks of 128 keys
  SB_DEVICE DqItem(const Args& a, int idx) {
    h = idx % a.Hq;
    kvh = h / a.group;
    q0 = a.order[idx / a.Hq] * 128;
    lo = hi = 0;
    if (q0 < a.ends[1] && q0 + 128 > a.ends[0]) {
      lo = a.start[q0] / 128;
      hi = q0 / 128 + 1;
    }
  }
};

template <int D, typename T>
__global__ void __launch_bounds__(kThreads, 1)
dq_kernel(const __grid_constant__ CUtensorMap tm, const __grid_constant__ CUtensorMap tmo, const __grid_constant__ Args a) {
  using F = Dq<D>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* sQ = smem_raw + (((raw + 1023) & ~1023u) - raw);
  uint8_t* sO = sQ + F::kTile;
  uint8_t* sK = sO + F::kTile;
  uint8_t* sV = sK + F::kK * F::kTile;
  uint4* answer = reinterpret_cast<uint4*>(sV + F::kV * F::kTile);
  uint64_t* bar = reinterpret_cast<uint64_t*>(answer + 2);
  uint64_t *q_full = bar, *q_empty = bar + 1, *land = bar + 2, *acc_full = bar + 3, *acc_free = bar + 4, *drain = bar + 5;
  uint64_t *k_full = bar + 6, *k_empty = k_full + F::kK, *v_full = k_empty + F::kK, *v_empty = v_full + F::kV;
  uint64_t *s_full = v_empty + F::kV, *p_full = s_full + 2, *s_empty = p_full + 2, *p_free = s_empty + 2;
  const Sched sched{answer, p_free + 2, p_free + 4};
  uint32_t* tslot = reinterpret_cast<uint32_t*>(p_free + 6);
  int* lists = reinterpret_cast<int*>(tslot + 1);      // [8]
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    mbar_init(land, 1);
    mbar_init(acc_full, 1);
    mbar_init(acc_free, 8);
    mbar_init(drain, 1);
    for (int i = 0; i < F::kK; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < F::kV; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 8);
      mbar_init(&s_empty[i], 8);
      mbar_init(&p_free[i], 1);
      mbar_init(&sched.full[i], 1);
      mbar_init(&sched.empty[i], kReaders);
    }
    fence_barrier_init();
  }
  if (warp == kIssuer) {
    tmem_alloc(tslot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = *tslot, tdQ = tbase + 256;

  if (warp >= 8) {
    regs_down<kOtherRegs>();
    if (warp == kLoader) {
      const int first = a.ends[0], last = min(a.ends[1], a.T);
      int g = 0, nq = 0, nl = 0, asked = 0;
      bool ok = true;
      for (int n = 0, idx = blockIdx.x; idx >= 0 && ok; ++n) {
        if (lane == 0) ok = sched_request(sched, n, a.status);
        ok = __all_sync(0xffffffffu, ok);
        const DqItem it(a, idx);
        if (ok && it.hi > it.lo) {
          if (lane == 0) {
            ok = mbar_wait(q_empty, (nq & 1) ^ 1, a.status);
            if (ok) {
              mbar_arrive_expect_tx(q_full, 2 * F::kTile);
              for (int c = 0; c < F::kHalves; ++c) {
                tma_load_2d(sQ + c * kChunk, &tm, q_full, it.h * D + c * 64, it.q0);
                tma_load_2d(sO + c * kChunk, &tmo, q_full, it.h * D + c * 64, it.q0);
              }
            }
          }
          ++nq;
          ok = __all_sync(0xffffffffu, ok);
          for (int j = it.lo; j < it.hi && ok; ++j, ++g) {
            const int sk = g % F::kK, sv = g % F::kV, row = j * 128;
            const bool clear = row < first || min(row + 128, a.T) > last;
            uint8_t* in = sK + sk * F::kTile;
            if (lane == 0) {
              ok = mbar_wait(&k_empty[sk], ((g / F::kK) & 1) ^ 1, a.status);
              if (ok) {
                uint64_t* to = clear ? land : &k_full[sk];
                mbar_arrive_expect_tx(to, F::kTile);
                for (int c = 0; c < F::kHalves; ++c)
                  tma_load_2d(in + c * kChunk, &tm, to, (a.Hq + it.kvh) * D + c * 64, row);
                ok = mbar_wait(&v_empty[sv], ((g / F::kV) & 1) ^ 1, a.status);
              }
              if (ok) {
                mbar_arrive_expect_tx(&v_full[sv], F::kTile);
                for (int c = 0; c < F::kHalves; ++c)
                  tma_load_2d(sV + sv * F::kTile + c * kChunk, &tm, &v_full[sv], (a.Hq + a.Hkv + it.kvh) * D + c * 64, row);
              }
            }
            ok = __all_sync(0xffffffffu, ok);
            if (clear && ok) {                         // K alone is multiplied by masked values
              ok = __all_sync(0xffffffffu, mbar_wait(land, nl & 1, a.status));
              ++nl;
              if (ok) {
                clear_rows(in, 128, F::kHalves, kChunk, row, first, last);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&k_full[sk]);
              }
            }
          }
        }
        asked = n + 1;
        if (ok) idx = sched_next(sched, n, a.status);
      }
      if (lane == 0) {
        landed(q_full, 1, nq);
        landed(k_full, F::kK, g);
        landed(v_full, F::kV, g);
        landed(sched.full, 2, asked);
      }
    } else if (warp == kIssuer) {
      constexpr uint32_t idS = idesc<T>(128, 128, 0), idG = idesc<T>(128, D, 1);
      const uint64_t dq = kdesc(smem_u32(sQ)), dob = kdesc(smem_u32(sO)), dk = kdesc(smem_u32(sK)), dv = kdesc(smem_u32(sV));
      const uint64_t dk_mn = mndesc(smem_u32(sK), kChunk);
      auto scores = [&](int g) -> bool {
        const int sk = g % F::kK, sv = g % F::kV;
        if (!mbar_wait(&k_full[sk], (g / F::kK) & 1, a.status)) return false;
        if (!mbar_wait(&v_full[sv], (g / F::kV) & 1, a.status)) return false;
        if (g >= 1 && !mbar_wait(s_empty, (g - 1) & 1, a.status)) return false;
        tc_fence_after();
        const uint64_t k = dk + sk * (F::kTile >> 4), v = dv + sv * (F::kTile >> 4);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const int off = ((kk >> 2) * kChunk + (kk & 3) * 32) >> 4, sub = ((kk >> 2) * kChunk + (kk & 3) * 32) >> 4;
          umma_f16(tbase, dq + off, k + sub, idS, kk > 0);
        }
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const int off = ((kk >> 2) * kChunk + (kk & 3) * 32) >> 4, sub = ((kk >> 2) * kChunk + (kk & 3) * 32) >> 4;
          umma_f16(tbase + 128, dob + off, v + sub, idS, kk > 0);
        }
        umma_commit(s_full);
        umma_commit(&v_empty[sv]);
        return true;
      };
      if (elect_one()) {
      int g = 0, nq = 0;
      bool ok = true;
      DqItem it(a, blockIdx.x);
      for (int n = 0, idx = blockIdx.x; idx >= 0 && ok; ++n) {
        DqItem following = it;
        const int subs = it.hi - it.lo;
        auto look_ahead = [&]() {                      // before the last wait of an item: its loads take a microsecond
          idx = sched_next<false>(sched, n, a.status);
          if (idx >= 0) following = DqItem(a, idx);
        };
        if (subs == 0) {
          look_ahead();
        } else {
          ok = mbar_wait(q_full, nq & 1, a.status);
          if (ok) ok = scores(g);
          for (int s = 0; s < subs && ok; ++s, ++g) {
            if (s + 1 < subs) ok = scores(g + 1);
            if (ok && s == max(0, subs - 2)) umma_commit(q_empty);              // the last scores were issued
            if (ok && s + 1 == subs) look_ahead();
            if (ok) ok = mbar_wait(p_full, g & 1, a.status);
            if (ok && s == 0 && nq > 0) ok = mbar_wait(acc_free, (nq - 1) & 1, a.status);
            if (!ok) break;
            tc_fence_after();
            const int sk = g % F::kK;
            const uint64_t k = dk_mn + sk * (F::kTile >> 4);
#pragma unroll
            for (int kk = 0; kk < 8; ++kk) umma_f16_ts(tdQ, tbase + F::kP + kk * 8, k + kk * (2048 >> 4), idG, s > 0 || kk > 0);
            umma_commit(&k_empty[sk]);
            umma_commit(p_free);
          }
          if (ok) umma_commit(acc_full);
          ++nq;
        }
        it = following;
      }
      umma_commit(drain);
      mbar_wait(drain, 0, a.status);
      }
      __syncwarp();
    }
  } else {
    regs_up<kSoftRegs>();
    const int w = warp / 4;                            // this group's half of the columns, also of dQ
    const uint32_t lane_off = static_cast<uint32_t>((warp % 4) * 32) << 16;
    const uint32_t ts = tbase + w * 64 + lane_off, tp = tbase + F::kP + w * 32 + lane_off;
    const float2 sc2 = make_float2(a.scale_log2, a.scale_log2);
    int g = 0, nq = 0;
    bool ok = true, s_ready = false;
    DqItem it(a, blockIdx.x);
    Later later{a.later, -1};
    for (int n = 0, idx = blockIdx.x; idx >= 0 && ok; ++n) {
      const int row = it.q0 + (warp % 4) * 32 + lane;
      const int st = row < a.T ? a.start[row] : row + 1;
      const int most = a.start[min(it.q0 + 127, a.T - 1)];
      const float* rb = row_block(a, it.h, row);       // there are rows up to a multiple of 128
      const int shift = query_shift<T>(a, it.h, row);  // of dS: in its exponential's argument
      const float out_scale = ldexpf(a.scale, -shift);
      const float2 nl = make_float2(rb[0] + (shift - kUpP<T>), rb[0] + (shift - kUpP<T>)), nd = make_float2(rb[64], rb[64]);
      for (int j = it.lo; j < it.hi; ++j, ++g) {
        if (!warp_wait(s_full, g & 1, a.status, s_ready)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const bool p_ready = g >= 1 && mbar_test(p_free, (g - 1) & 1);
        const int k0 = j * 128 + w * 64;
        const bool masked = k0 < most || k0 + 63 > it.q0;
        uint32_t ws[64], wd[64];
        tmem_ld_32x32b_x32(ts, ws);
        tmem_ld_32x32b_x32(ts + 128, wd);
        tmem_ld_32x32b_x32(ts + 32, ws + 32);
        tmem_ld_32x32b_x32(ts + 128 + 32, wd + 32);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(s_empty);
#pragma unroll
        for (int c = 0; c < 64; c += 32) {
          const uint32_t *vs = ws + c, *vd = wd + c;
          uint32_t pd[16];
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            float2 z = fma2(make_float2(__uint_as_float(vs[k]), __uint_as_float(vs[k + 1])), sc2, nl);
            float2 e = add2(make_float2(__uint_as_float(vd[k]), __uint_as_float(vd[k + 1])), nd);
            z = k / 2 % 8 < kOnFma ? ex2_fma(z) : make_float2(ex2(z.x), ex2(z.y));
            e = mul2(e, z);
            pd[k / 2] = Half<T>::pack(e.x, e.y);
          }
          if (masked) {
            const uint32_t bits = seen(st - k0 - c, row - k0 - c);
            if (!__all_sync(0xffffffffu, bits == 0xffffffffu))
#pragma unroll
              for (int k = 0; k < 16; ++k)
                pd[k] &= (bits >> (2 * k) & 1 ? 0xffffu : 0u) | (bits >> (2 * k + 1) & 1 ? 0xffff0000u : 0u);
          }
          if (c == 0 && g >= 1) {                      // the product of the block before has read dS
            if (!warp_wait(p_free, (g - 1) & 1, a.status, p_ready)) ok = false;
            tc_fence_after();
          }
          tmem_st_32x32b_x16(tp + c / 2, pd);
        }
        if (!ok) break;
        s_ready = mbar_test(s_full, (g + 1) & 1);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full);
      }
      if (!ok) break;
      const bool covered = row < a.T && st <= row;
      const DqItem at = it;
      const int item = idx;
      idx = sched_next(sched, n, a.status);            // its tile is looked up while the last products run
      if (idx >= 0) it = DqItem(a, idx);
      T* out = static_cast<T*>(a.dqkv) + row * a.dqkv_ld + static_cast<long>(at.h) * D;
      bool bad = false;
      if (at.hi > at.lo) {
        if (!__all_sync(0xffffffffu, mbar_wait(acc_full, nq & 1, a.status))) {
          ok = false;
          break;
        }
        ++nq;
        tc_fence_after();
        float chk = 0.f;
#pragma unroll
        for (int u = 0; u < D / 64; ++u) {
          const int c = w * (D / 2) + u * 32;
          uint32_t o[32];
          tmem_ld_32x32b_x32(tdQ + lane_off + c, o);
          tmem_wait_ld();
          if (u + 1 == D / 64) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_free);
          }
#pragma unroll
          for (int k = 0; k < 32; k += 8) {
            uint32_t y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float y0 = __uint_as_float(o[k + 2 * e]) * out_scale, y1 = __uint_as_float(o[k + 2 * e + 1]) * out_scale;
              chk = fmaf(y0, 0.f, fmaf(y1, 0.f, chk));
              y[e] = Half<T>::pack(y0, y1);
            }
            if (covered) *reinterpret_cast<uint4*>(out + c + k) = make_uint4(y[0], y[1], y[2], y[3]);
          }
        }
        bad = covered && chk != 0.f;
      }
      if (row < a.T && !covered && a.fill)
#pragma unroll
        for (int c = 0; c < D / 2; c += 8) *reinterpret_cast<uint4*>(out + w * (D / 2) + c) = make_uint4(0, 0, 0, 0);
      later.add(__ballot_sync(0xffffffffu, bad), item);
    }
    later.run(lists, [&](int item, int finder, int who) {
      const DqItem at(a, item);
      slow_dq<D, T>(a, at.q0 + finder % 4 * 32 + who, at.h, finder / 4 * (D / 2), (finder / 4 + 1) * (D / 2));
    });
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kIssuer) tmem_dealloc(tbase, 512);
}

template <int D, typename T>
static void launch(const CUtensorMap& tm128, const CUtensorMap& tm64, const CUtensorMap& do128, const CUtensorMap& do64,
                   Args a, const int* q_order, const int* k_order, float* rows, cudaStream_t stream) {
  const long work = static_cast<long>(a.tiles) * 128 * a.Hq;
  rows_kernel<D, T><<<static_cast<unsigned>((work + 256 / (D / 8) - 1) / (256 / (D / 8))), 256, 0, stream>>>(a, rows);
  a.rows = rows;
  if (a.tops != nullptr)
    shift_kernel<<<dim3((a.tiles * 128 + 1023) / 1024, a.Hkv), 1024, 0, stream>>>(a);
  cudaFuncSetAttribute(dkv_kernel<D, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, Dkv<D>::kSmem);
  cudaFuncSetAttribute(dq_kernel<D, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, Dq<D>::kSmem);
  a.order = k_order;
  dkv_kernel<D, T><<<static_cast<unsigned>(a.tiles * a.Hkv * a.split), kThreads, Dkv<D>::kSmem, stream>>>(
      tm128, Dkv<D>::kWide ? tm128 : tm64, Dkv<D>::kWide ? do128 : do64, a);
  if (a.split > 1) {
    const long n = static_cast<long>(a.Hkv) * a.T * (2 * D / 8);
    join_kernel<D, T><<<static_cast<unsigned>((n + 255) / 256), 256, 0, stream>>>(a);
  }
  a.order = q_order;
  dq_kernel<D, T><<<static_cast<unsigned>(a.tiles * a.Hq), kThreads, Dq<D>::kSmem, stream>>>(tm128, do128, a);
}

void launch_bwd(int D, bool half, const CUtensorMap& tm128, const CUtensorMap& tm64, const CUtensorMap& do128,
                const CUtensorMap& do64, const Args& a, const int* q_order, const int* k_order, float* rows,
                cudaStream_t stream) {
  if (D == 64) {
    if (half) launch<64, __half>(tm128, tm64, do128, do64, a, q_order, k_order, rows, stream);
    else launch<64, __nv_bfloat16>(tm128, tm64, do128, do64, a, q_order, k_order, rows, stream);
  } else {
    if (half) launch<128, __half>(tm128, tm64, do128, do64, a, q_order, k_order, rows, stream);
    else launch<128, __nv_bfloat16>(tm128, tm64, do128, do64, a, q_order, k_order, rows, stream);
  }
}

}  // namespace pa
}  // namespace sb

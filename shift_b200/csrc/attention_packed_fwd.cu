// Forward kernel of causal attention over packed sequences (attention_packed.cuh has the design).
#include "attention_packed.cuh"

namespace sb {
namespace pa {

// ============================ forward ============================
// An item is two tiles of 128 queries that share a loop over key blocks.  Group w of softmax warps has tile w.
//   issuer   S_w = Q_w K_j^T (128 x 128),  O_w += P_w V_j (128 x D), P_w read from tensor memory
//   softmax  a thread's whole row of S to registers, running maximum and sum, P back to tensor memory
// Heads of 64: S, P and O of both tiles have columns of their own (2 x (128 + 64 + 64)), so the next S is computed while a
// group is still at its exponentials.  Heads of 128: P lies over S (2 x (128 + 128)).
//
// SPLIT: with few tiles of heads of 64 (the rule stands in attention_packed_host.cpp) the two tiles are one: group w has every
// second key block of it, from the w-th, and the two partial results are joined at the end, half of the columns a group.  An
// item then takes half of its blocks' time, which is what counts when every SM has one or two.
template <int D, bool SPLIT>
struct Fwd {
  static constexpr int kHalves = D / 64, kTile = kHalves * kChunk;
  static constexpr int kK = D == 64 ? 4 : 3, kV = D == 64 ? 4 : 2;     // stages
  static constexpr bool kOver = D == 128;                              // P over S
  static constexpr int kQ = SPLIT ? 1 : 2;                             // tiles of Q
  static constexpr int kSmem = 1024 + (kQ + kK + kV) * kTile + 512 + (SPLIT ? 2 * 2 * 128 * 8 : 0);
  static constexpr int kP = kOver ? 0 : 256, kPStep = kOver ? 128 : 64, kO = kOver ? 256 : 384;
};

template <bool SPLIT>
struct FwdItem {
  int h[2], q0[2], lo[2], hi[2], all_lo, all_hi, kvh;
  SB_DEVICE FwdItem(const Args& a, int idx) {
    const bool pair = !SPLIT && a.pair_heads;
    const int per = pair ? a.Hq / 2 : a.Hq;
    const int t = a.order[idx / per], r = idx % per;
    const int first = a.ends[0], last = a.ends[1];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      h[i] = pair ? 2 * r + i : r;
      q0[i] = SPLIT || pair ? t * 128 : t * 256 + i * 128;
      lo[i] = hi[i] = 0;
      if (q0[i] < a.T && q0[i] < last && q0[i] + 128 > first) {
        lo[i] = a.start[q0[i]] / 128;
        hi[i] = q0[i] / 128 + 1;
      }
    }
    const bool one = hi[0] > lo[0], two = hi[1] > lo[1];
    all_lo = one && two ? min(lo[0], lo[1]) : one ? lo[0] : lo[1];
    all_hi = max(hi[0], hi[1]);
    kvh = h[0] / a.group;
  }
  SB_DEVICE bool has(int i, int j) const { return j >= lo[i] && j < hi[i] && (!SPLIT || ((j - lo[i]) & 1) == i); }
  SB_DEVICE bool first(int i, int j) const { return j == lo[i] + (SPLIT ? i : 0); }
  SB_DEVICE bool last(int i, int j) const { return j + (SPLIT ? 2 : 1) >= hi[i]; }
  SB_DEVICE bool any(int i) const { return hi[i] > lo[i] + (SPLIT ? i : 0); }
};

// Of 8 exponentials, those computed on the FMA pipe.  3 and 2, 16 / 4 heads: 8 x 2048 rows, heads of 64 122 and 122 us, of 128
// 144 and 141; 24 x 700, of 64 79 and 77.
constexpr int kOnFma = 2;

template <int D, typename T, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1) fwd_kernel(const __grid_constant__ CUtensorMap tm, const __grid_constant__ Args a) {
  using F = Fwd<D, SPLIT>;
  using FwdItem = FwdItem<SPLIT>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* sQ = smem_raw + (((raw + 1023) & ~1023u) - raw);
  uint8_t* sK = sQ + F::kQ * F::kTile;
  uint8_t* sV = sK + F::kK * F::kTile;
  float2* s_ml = reinterpret_cast<float2*>(sV + F::kV * F::kTile);           // SPLIT: [item parity][group][row] (m, l)
  uint4* answer = reinterpret_cast<uint4*>(s_ml + (SPLIT ? 2 * 2 * 128 : 0));
  uint64_t* bar = reinterpret_cast<uint64_t*>(answer + 2);
  uint64_t *q_full = bar, *q_empty = bar + 1, *land = bar + 2, *k_full = bar + 3, *k_empty = k_full + F::kK;
  uint64_t *v_full = k_empty + F::kK, *v_empty = v_full + F::kV, *s_full = v_empty + F::kV, *s_empty = s_full + 2;
  uint64_t *p_full = s_empty + 2, *o_full = p_full + 2, *o_free = o_full + 2, *drain = o_free + 2;
  const Sched sched{answer, drain + 1, drain + 3};
  uint64_t* ml_full = drain + 5;                       // SPLIT: a group's maxima and sums
  uint32_t* tslot = reinterpret_cast<uint32_t*>(drain + 7);
  int* lists = reinterpret_cast<int*>(tslot + 1);      // [8]
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const FwdItem first_item(a, blockIdx.x);             // its dependent loads run under the set-up

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    mbar_init(land, 1);
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
      mbar_init(&s_empty[i], 4);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_full[i], 1);
      mbar_init(&o_free[i], SPLIT ? 8 : 4);
      mbar_init(&ml_full[i], 4);
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
  const uint32_t tbase = *tslot;

  if (warp >= 8) {
    regs_down<kOtherRegs>();
    if (warp == kLoader) {
      const int first = a.ends[0], last = min(a.ends[1], a.T);
      int nk = 0, nv = 0, nq = 0, nl = 0, asked = 0;
      bool ok = true;
      if (lane == 0) tma_prefetch_desc(&tm);
      FwdItem it = first_item;
      for (int n = 0, idx = blockIdx.x; idx >= 0 && ok; ++n) {
        if (lane == 0) ok = sched_request(sched, n, a.status);
        ok = __all_sync(0xffffffffu, ok);
        if (n > 0) it = FwdItem(a, idx);
        if (ok && it.all_hi > it.all_lo) {
          if (lane == 0) {
            ok = mbar_wait(q_empty, (nq & 1) ^ 1, a.status);
            if (ok) {
              mbar_arrive_expect_tx(q_full, F::kQ * F::kTile);
              for (int i = 0; i < F::kQ; ++i)
                for (int c = 0; c < F::kHalves; ++c)
                  tma_load_2d(sQ + i * F::kTile + c * kChunk, &tm, q_full, it.h[i] * D + c * 64, it.q0[i]);
            }
          }
          ++nq;
          ok = __all_sync(0xffffffffu, ok);
          for (int j = it.all_lo; j < it.all_hi && ok; ++j, ++nk, ++nv) {
            const int sk = nk % F::kK, sv = nv % F::kV, row = j * 128;
            const bool clear = row < first || min(row + 128, a.T) > last;
            if (lane == 0) {
              ok = mbar_wait(&k_empty[sk], ((nk / F::kK) & 1) ^ 1, a.status);
              if (ok) {
                mbar_arrive_expect_tx(&k_full[sk], F::kTile);
                for (int c = 0; c < F::kHalves; ++c)
                  tma_load_2d(sK + sk * F::kTile + c * kChunk, &tm, &k_full[sk], (a.Hq + it.kvh) * D + c * 64, row);
                ok = mbar_wait(&v_empty[sv], ((nv / F::kV) & 1) ^ 1, a.status);
              }
              if (ok) {
                uint64_t* to = clear ? land : &v_full[sv];
                mbar_arrive_expect_tx(to, F::kTile);
                for (int c = 0; c < F::kHalves; ++c)
                  tma_load_2d(sV + sv * F::kTile + c * kChunk, &tm, to, (a.Hq + a.Hkv + it.kvh) * D + c * 64, row);
              }
            }
            ok = __all_sync(0xffffffffu, ok);
            if (clear && ok) {
              ok = __all_sync(0xffffffffu, mbar_wait(land, nl & 1, a.status));
              ++nl;
              if (ok) {
                clear_rows(sV + sv * F::kTile, 128, F::kHalves, kChunk, row, first, last);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&v_full[sv]);
              }
            }
          }
        }
        asked = n + 1;
        if (ok) idx = sched_next(sched, n, a.status);
      }
      if (lane == 0) {
        landed(q_full, 1, nq);
        landed(k_full, F::kK, nk);
        landed(v_full, F::kV, nv);
        landed(sched.full, 2, asked);
      }
    } else if (warp == kIssuer) {
      constexpr uint32_t idS = idesc<T>(128, 128, 0), idO = idesc<T>(128, D, 1);
      // all of shared memory lies below 256 KB: adding to a descriptor's address field (16-byte units) never carries out
      const uint64_t dq = kdesc(smem_u32(sQ)), dk = kdesc(smem_u32(sK)), dv = mndesc(smem_u32(sV), kChunk);
      auto issue_s = [&](int i, int sk) {              // S_i of the key block in stage sk
        const uint64_t q = dq + (SPLIT ? 0 : i) * (F::kTile >> 4), k = dk + sk * (F::kTile >> 4);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const int off = ((kk >> 2) * kChunk + (kk & 3) * 32) >> 4;
          umma_f16(tbase + i * 128, q + off, k + off, idS, kk > 0);
        }
        umma_commit(&s_full[i]);
      };
      auto issue_o = [&](int i, int sv, bool fresh, bool last) {
        const uint64_t v = dv + sv * (F::kTile >> 4);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          umma_f16_ts(tbase + F::kO + i * D, tbase + F::kP + i * F::kPStep + kk * 8, v + kk * (2048 >> 4), idO,
                      !(fresh && kk == 0));
        if (!F::kOver || last) umma_commit(&o_full[i]);
      };
      if (elect_one()) {
      int nk = 0, nv = 0, nq = 0, nb[2] = {0, 0}, no[2] = {0, 0};   // blocks and items of each tile so far
      bool ok = true;
      FwdItem it = first_item;
      for (int n = 0, idx = blockIdx.x; idx >= 0 && ok; ++n) {
        FwdItem following = it;
        auto look_ahead = [&]() {                      // before the last wait of an item: its loads take a microsecond
          idx = sched_next<false>(sched, n, a.status);
          if (idx >= 0) following = FwdItem(a, idx);
        };
        if (it.all_hi <= it.all_lo) {
          look_ahead();
        } else {
          ok = mbar_wait(q_full, nq & 1, a.status);
          ++nq;
          // S of block j: its stage is nk % kK
          auto scores = [&](int j, int i) -> bool {
            if (!F::kOver && nb[i] > 0 && !mbar_wait(&s_empty[i], (nb[i] - 1) & 1, a.status)) return false;
            tc_fence_after();
            issue_s(i, nk % F::kK);
            ++nb[i];
            return true;
          };
          auto keys = [&]() -> bool { return mbar_wait(&k_full[nk % F::kK], (nk / F::kK) & 1, a.status); };
          auto keys_done = [&](int j) {
            umma_commit(&k_empty[nk % F::kK]);
            ++nk;
            if (j == it.all_hi - 1) umma_commit(q_empty);
          };
          int np[2] = {nb[0], nb[1]};                  // blocks whose P was used
          // scores are issued one block ahead, SPLIT two (one for each group)
          constexpr int kAhead = SPLIT ? 2 : 1;
          for (int j = it.all_lo; j < min(it.all_lo + kAhead, it.all_hi) && ok; ++j) {
            ok = keys();
            for (int i = 0; i < 2 && ok; ++i)
              if (it.has(i, j)) ok = scores(j, i);
            if (ok) keys_done(j);
          }
          for (int j = it.all_lo; j < it.all_hi && ok; ++j) {
            const int next = j + kAhead;
            const bool more = next < it.all_hi;
            if (more) ok = keys();
            if (!F::kOver && more) {
              for (int i = 0; i < 2 && ok; ++i)
                if (it.has(i, next)) ok = scores(next, i);
              if (ok) keys_done(next);
            }
            const int sv = nv % F::kV;
            if (ok && j + 1 == it.all_hi) look_ahead();
            if (ok) ok = mbar_wait(&v_full[sv], (nv / F::kV) & 1, a.status);
            for (int i = 0; i < 2 && ok; ++i) {
              if (it.has(i, j)) {
                ok = mbar_wait(&p_full[i], np[i] & 1, a.status);
                ++np[i];
                if (ok && it.first(i, j) && no[i] > 0) ok = mbar_wait(&o_free[i], (no[i] - 1) & 1, a.status);
                if (!ok) break;
                tc_fence_after();
                issue_o(i, sv, it.first(i, j), it.last(i, j));
              }
              if (F::kOver && more && it.has(i, next)) ok = scores(next, i);
            }
            if (!ok) break;
            umma_commit(&v_empty[sv]);
            ++nv;
            if (F::kOver && more) keys_done(next);
          }
          for (int i = 0; i < 2; ++i) no[i] += it.any(i);
        }
        it = following;
      }
      umma_commit(drain);                              // nothing of this CTA is in flight when tensor memory is given back
      mbar_wait(drain, 0, a.status);
      }
      __syncwarp();
    }
  } else {
    regs_up<kSoftRegs>();
    const int w = warp / 4;                            // tile
    const uint32_t lane_off = static_cast<uint32_t>((warp % 4) * 32) << 16;
    const uint32_t ts = tbase + w * 128 + lane_off, tp = tbase + F::kP + w * F::kPStep + lane_off;
    const uint32_t to = tbase + F::kO + w * D + lane_off;
    const float2 sc2 = make_float2(a.scale_log2, a.scale_log2);
    int nb = 0, items = 0;
    int live = 0, other_nb = 0, other_items = 0;       // SPLIT: items with blocks; the other group's blocks and items
    bool ok = true, s_ready = false;
    constexpr int kStep = SPLIT ? 2 : 1;
    struct Mine {                                      // this group's tile: blocks lo, lo + kStep ... below hi
      int h, q0, lo, hi, row, st, most;
      SB_DEVICE Mine(const Args& a, const FwdItem& it, int w) {
        q0 = w ? it.q0[1] : it.q0[0];
        lo = w ? it.lo[1] + (SPLIT ? 1 : 0) : it.lo[0];
        hi = w ? it.hi[1] : it.hi[0];
        h = w ? it.h[1] : it.h[0];
        row = q0 + threadIdx.x % 128;
        st = row < a.T ? a.start[row] : row + 1;
        most = q0 < a.T ? a.start[min(q0 + 127, a.T - 1)] : 0;             // the tile's latest start
      }
    };
    Mine now(a, first_item, w);
    Later later{a.later, -1};
    for (int n = 0, idx = blockIdx.x; idx >= 0 && ok; ++n) {
      const int h = now.h, q0 = now.q0, lo = now.lo, hi = now.hi, row = now.row, st = now.st, most = now.most;
      float m = -INFINITY, l = 0.f;
      for (int j = lo; j < hi; j += kStep, ++nb) {
        if (!warp_wait(&s_full[w], nb & 1, a.status, s_ready)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t v[128];
#pragma unroll
        for (int c = 0; c < 128; c += 32) tmem_ld_32x32b_x32(ts + c, v + c);
        tmem_wait_ld();
        if (!F::kOver) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_empty[w]);
        }
        if (j * 128 < most || j * 128 + 127 > q0) {
#pragma unroll
          for (int c = 0; c < 128; c += 32) {
            const uint32_t bits = seen(st - j * 128 - c, row - j * 128 - c);
            if (!__all_sync(0xffffffffu, bits == 0xffffffffu))
#pragma unroll
              for (int k = 0; k < 32; ++k)
                if (!(bits >> k & 1)) v[c + k] = 0xff800000u;
          }
        }
        // P V of the block before must be done before P is written again or O rescaled: where P lies over S, this block's
        // S was issued behind it
        const bool o_ready = !F::kOver && j > lo && mbar_test(&o_full[w], (nb - 1) & 1);
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 128; c += 8)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            m4[k] = max3(m4[k], __uint_as_float(v[c + 2 * k]), __uint_as_float(v[c + 2 * k + 1]));
        const float mx = fmaxf(m, fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * a.scale_log2);
        if (!F::kOver && j > lo) {
          if (!warp_wait(&o_full[w], (nb - 1) & 1, a.status, o_ready)) {
            ok = false;
            break;
          }
          tc_fence_after();
        }
        if (__any_sync(0xffffffffu, mx > m + kRescale)) {
          if (j > lo) {
            const float f = mx == -INFINITY ? 1.f : ex2(m - mx);
#pragma unroll
            for (int c = 0; c < D; c += 16) {          // few at a time: S is still in registers
              uint32_t o[16];
              tmem_ld_32x32b_x16(to + c, o);
              tmem_wait_ld();
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
              tmem_st_32x32b_x16(to + c, o);
            }
            tmem_wait_st();
            l *= f;
          }
          m = mx;
        }
        const float nm = m == -INFINITY ? 0.f : -m;
        const float2 nm2 = make_float2(nm, nm);
        float2 l2[4] = {};
#pragma unroll
        for (int c = 0; c < 128; c += 32) {
          float2 z[16];
          uint32_t pk[16];
#pragma unroll
          for (int k = 0; k < 16; ++k)
            z[k] = fma2(make_float2(__uint_as_float(v[c + 2 * k]), __uint_as_float(v[c + 2 * k + 1])), sc2, nm2);
#pragma unroll
          for (int k = 0; k < 16; ++k) z[k] = k % 8 < kOnFma ? ex2_fma(z[k]) : make_float2(ex2(z[k].x), ex2(z[k].y));
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            l2[k & 3] = add2(l2[k & 3], z[k]);
            pk[k] = Half<T>::pack(z[k].x, z[k].y);
          }
          tmem_st_32x32b_x16(tp + c / 2, pk);
        }
        s_ready = j + kStep < hi && mbar_test(&s_full[w], (nb + 1) & 1);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[w]);
        l2[0] = add2(add2(l2[0], l2[1]), add2(l2[2], l2[3]));
        l += l2[0].x + l2[0].y;
      }
      if (!ok) break;
      const int item = idx;
      idx = sched_next(sched, n, a.status);            // its tile is looked up while the last products run
      if (idx >= 0) now = Mine(a, FwdItem(a, idx), w);
      const bool covered = row < a.T && st <= row;
      float lse2 = -INFINITY;
      bool bad = false;
      constexpr int kCols = SPLIT ? D / 2 : D;         // columns of O that this group stores, from c0
      const int c0 = SPLIT ? w * kCols : 0;
      T* orow = static_cast<T*>(a.o) + row * a.o_ld + static_cast<long>(h) * D;
      const bool mine = hi > lo, theirs = SPLIT && hi > lo + (w ? -1 : 1);         // who has blocks
      if (mine || theirs) {
        float f = 1.f, g = 0.f, top = m;               // factors of this group's O and of the other's
        if (SPLIT) {
          s_ml[(live & 1) * 256 + w * 128 + threadIdx.x % 128] = make_float2(m, l);
          __syncwarp();
          if (lane == 0) mbar_arrive(&ml_full[w]);
          // what the other group waited for before it came here tells which phase its O's barrier is in
          if (!warp_wait(&ml_full[w ^ 1], live & 1, a.status)) {
            ok = false;
            break;
          }
          const float2 other = s_ml[(live & 1) * 256 + (w ^ 1) * 128 + threadIdx.x % 128];
          ++live;
          top = fmaxf(m, other.x);
          f = m == -INFINITY ? 0.f : ex2(m - top);
          g = other.x == -INFINITY ? 0.f : ex2(other.x - top);
          l = l * f + other.y * g;
          if (theirs) {
            other_nb += (hi - (w ? lo - 1 : lo + 1) + 1) / 2;
            if (!warp_wait(&o_full[w ^ 1], (F::kOver ? other_items : other_nb - 1) & 1, a.status)) {
              ok = false;
              break;
            }
            ++other_items;
          }
        }
        if (mine) {
          if (!warp_wait(&o_full[w], (F::kOver ? items : nb - 1) & 1, a.status)) {
            ok = false;
            break;
          }
          ++items;
        }
        tc_fence_after();
        const float inv = 1.f / l;
        float chk = 0.f;
        lse2 = top + log2f(l);
        const uint32_t from = tbase + F::kO + lane_off + c0;
#pragma unroll
        for (int c = 0; c < kCols; c += 32) {
          uint32_t o[32];
          if (SPLIT) {
            uint32_t p[32];
            if (mine) tmem_ld_32x32b_x32(from + w * D + c, o);
            if (theirs) tmem_ld_32x32b_x32(from + (w ^ 1) * D + c, p);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k)               // O without a block is not there, not even as zeros
              o[k] = __float_as_uint((mine ? __uint_as_float(o[k]) * f : 0.f) + (theirs ? __uint_as_float(p[k]) * g : 0.f));
          } else {
            tmem_ld_32x32b_x32(from + w * D + c, o);
            tmem_wait_ld();
          }
          if (c + 32 == kCols) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0 && mine) mbar_arrive(&o_free[w]);
            if (lane == 0 && theirs) mbar_arrive(&o_free[w ^ 1]);
          }
#pragma unroll
          for (int k = 0; k < 32; k += 8) {
            uint32_t y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float y0 = __uint_as_float(o[k + 2 * e]) * inv, y1 = __uint_as_float(o[k + 2 * e + 1]) * inv;
              chk = fmaf(y0, 0.f, fmaf(y1, 0.f, chk));
              y[e] = Half<T>::pack(y0, y1);
            }
            if (covered) *reinterpret_cast<uint4*>(orow + c0 + c + k) = make_uint4(y[0], y[1], y[2], y[3]);
          }
        }
        bad = covered && chk != 0.f && fabsf(lse2) < INFINITY;
      }
      if (row < a.T) {
        if (!SPLIT || w == 0) a.lse[static_cast<long>(h) * a.T + row] = covered ? lse2 * kLn2 : -INFINITY;
        if (!covered && a.fill)
#pragma unroll
          for (int c = 0; c < kCols; c += 8) *reinterpret_cast<uint4*>(orow + c0 + c) = make_uint4(0, 0, 0, 0);
      }
      later.add(__ballot_sync(0xffffffffu, bad), item);
    }
    later.run(lists, [&](int item, int finder, int who) {
      const Mine m(a, FwdItem(a, item), finder / 4);
      constexpr int kCols = SPLIT ? D / 2 : D;
      const int c0 = SPLIT ? finder / 4 * kCols : 0;
      slow_o<D, T>(a, m.q0 + finder % 4 * 32 + who, m.h, c0, c0 + kCols);
    });
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kIssuer) tmem_dealloc(tbase, 512);
}

template <int D, typename T, bool SPLIT>
static void launch(const CUtensorMap& tm, const Args& a, unsigned items, cudaStream_t stream) {
  using F = Fwd<D, SPLIT>;
  cudaFuncSetAttribute(fwd_kernel<D, T, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::kSmem);
  fwd_kernel<D, T, SPLIT><<<items, kThreads, F::kSmem, stream>>>(tm, a);
}

template <typename T>
static void launch_typed(int D, const CUtensorMap& tm, const Args& a, unsigned items, cudaStream_t stream) {
  if (D == 64) a.split_keys ? launch<64, T, true>(tm, a, items, stream) : launch<64, T, false>(tm, a, items, stream);
  else launch<128, T, false>(tm, a, items, stream);
}

void launch_fwd(int D, bool half, const CUtensorMap& tm, const Args& a, unsigned items, cudaStream_t stream) {
  half ? launch_typed<__half>(D, tm, a, items, stream) : launch_typed<__nv_bfloat16>(D, tm, a, items, stream);
}

}  // namespace pa
}  // namespace sb

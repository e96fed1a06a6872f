// Causal attention over packed sequences on the 5th-generation tensor cores (sm_100a).
//
//   s = scale q k^T for the keys start(q) <= k <= q,  p = exp(s - lse),  o = p v,  lse = log sum exp s
//   dp = do v^T,  delta = do . o,  ds = p (dp - delta),  dq = scale ds k,  dk = scale ds^T q,  dv = p^T do
//
// Rows are tiled by 128 without regard to where sequences begin: what a query sees is the interval [start(q), q], and
// what sees a key is [key, stop(key)), so a tile that holds several sequences masks by two numbers a row, the number of
// tiles is known to the host, and short sequences share tiles (tiles of one sequence each would take 128 rows for every
// sequence of one token).  Only blocks at an interval's border pay for the mask.
//
// All kernels run persistently: a CTA takes its next tile from the hardware's list of CTAs that have not started
// (cluster launch control), the costliest tiles first.  Twelve warps: two groups of four softmax warps (a thread has one
// row of 128), one warp that loads tiles by TMA, one that issues tcgen05.mma.  Scores live in tensor memory; the
// probabilities go back there as 16-bit operands of the second product and never to shared memory.
//
// What is rounded to 16 bits: P and dS, since the tensor cores take them so (two operands for each, the value and what its
// rounding left, would double the products that bound these kernels), o, from which delta is taken, and the results.  Scores,
// statistics and sums are fp32; the sum behind lse takes P unrounded.  Outputs are 1.1 to 1.5 times as far from 64 bits as fp32
// arithmetic that rounds its results alone.
//
// What others hold.  Products run over whole blocks, so a masked value is a product with zero, which is zero unless the
// other factor is infinite or NaN.  Rows that no sequence covers are cleared in shared memory after they were loaded.  Rows
// of other sequences (or later ones of the same) that are not finite would leave NaN in a result: results that are not finite
// are recognised when they are stored and, where such a row met them, computed again row by row from what they see.  That may
// take long, so it comes after a CTA's last item, when no wait of its pipeline hangs on it.
//
// Every wait is bounded; on expiry the kernel records a status code and winds down.
#pragma once
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "attention_packed.h"
#include "common.cuh"
#include "lowp.cuh"

namespace sb {
namespace pa {

constexpr int kThreads = 384;      // 8 softmax warps, loader, MMA issuer, two idle (a whole group of four for setmaxnreg)
constexpr int kLoader = 8, kIssuer = 9;
constexpr int kReaders = 10;       // warps that read a scheduling slot
constexpr int kChunk = 128 * 128;  // bytes of 128 rows of 64 16-bit columns
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// O is rescaled only when a row's maximum rises by more than 2^8 over the one in use: the probabilities then stay below
// 2^8 (fp16 holds them), and after a row's first blocks it hardly ever happens.
constexpr float kRescale = 8.f;

SB_DEVICE float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// True in one lane of a converged warp.  What issues to the tensor cores runs under it as a whole: the compiler then keeps
// descriptors and barriers in uniform registers, where those instructions take them from (under `lane == 0` the sixteen
// products of a 128 x 128 block of heads of 128 took 2900 clocks to issue; they run in 1024).
SB_DEVICE bool elect_one() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}

// two fp32 operations in one instruction
SB_DEVICE float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
  return d;
}
SB_DEVICE float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}
SB_DEVICE float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}

SB_DEVICE float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 2^x of two values on the FMA and integer pipes, for x <= 127: x = j + r with j the nearest whole number (left in the low
// bits of x + 1.5 * 2^23) and r in [-1/2, 1/2]; 2^r by a polynomial of degree 4 that is 1 at 0, fitted to the relative error
// over that interval (least squares, reweighted; at most 2.9e-6), times 2^j.  At -127 and below, masked -inf among
// it, 2^j is exactly 0: a masked probability must not carry another row's value, however large that is.  NaN stays NaN.
__device__ constexpr float kEx2[5] = {1.f, 0.693124175f, 0.240240991f, 0.0559064262f, 0.00958285294f};
SB_DEVICE float max_nan(float a, float b) {            // NaN where one of them is
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
SB_DEVICE float2 ex2_fma(float2 x) {
  x.x = max_nan(x.x, -127.f);
  x.y = max_nan(x.y, -127.f);
  const float2 t = add2(x, make_float2(12582912.f, 12582912.f));
  const float2 j = add2(t, make_float2(-12582912.f, -12582912.f));
  const float2 r = fma2(j, make_float2(-1.f, -1.f), x);
  float2 p = fma2(make_float2(kEx2[4], kEx2[4]), r, make_float2(kEx2[3], kEx2[3]));
  p = fma2(p, r, make_float2(kEx2[2], kEx2[2]));
  p = fma2(p, r, make_float2(kEx2[1], kEx2[1]));
  p = fma2(p, r, make_float2(kEx2[0], kEx2[0]));
  return mul2(p, make_float2(__uint_as_float((__float_as_uint(t.x) << 23) + 0x3f800000u),
                             __uint_as_float((__float_as_uint(t.y) << 23) + 0x3f800000u)));
}

// Whether a barrier's phase is over; asked early, since the answer takes a hundred clocks.
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
// The wait of a whole warp; `ready`: the answer to an earlier question.
SB_DEVICE bool warp_wait(uint64_t* bar, uint32_t phase, int* status, bool ready = false) {
  if (__all_sync(0xffffffffu, ready)) return true;
  return __all_sync(0xffffffffu, mbar_wait(bar, phase, status));
}

// Before a CTA ends: the last `n` copies to these barriers' stages have landed in its memory.  They have, unless a wait ran out,
// and then they take no longer than this.
SB_DEVICE void landed(uint64_t* full, int stages, int n) {
  for (int i = max(0, n - stages); i < n; ++i) mbar_wait(&full[i % stages], (i / stages) & 1, nullptr, 10000000ull);
}

// Bits [from, to] of a word, clipped to it: which of 32 columns are seen.
SB_DEVICE uint32_t seen(int from, int to) {
  const uint32_t low = to >= 31 ? 0xffffffffu : to < 0 ? 0u : (2u << to) - 1u;
  return from <= 0 ? low : from > 31 ? 0u : low & (0xffffffffu << from);
}

template <typename T>
struct Half;
template <>
struct Half<__nv_bfloat16> {
  static constexpr uint32_t kFormat = 1;
  static SB_DEVICE uint32_t pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
};
template <>
struct Half<__half> {
  static constexpr uint32_t kFormat = 0;
  static SB_DEVICE uint32_t pack(float lo, float hi) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
};

// instruction descriptor: fp32 accumulator, operands of type T, B along N where b_mn
template <typename T>
constexpr uint32_t idesc(int M, int N, int b_mn) {
  return (1u << 4) | (Half<T>::kFormat << 7) | (Half<T>::kFormat << 10) | (static_cast<uint32_t>(b_mn) << 16) |
         (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}
SB_DEVICE uint64_t kdesc(uint32_t addr) { return make_sw128_desc(addr, 16, 1024); }
// B along N: the second 64 columns lie `next` bytes behind the first
SB_DEVICE uint64_t mndesc(uint32_t addr, uint32_t next) { return make_sw128_desc(addr, next, 1024); }

SB_DEVICE void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

template <int N>
SB_DEVICE void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
SB_DEVICE void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
// 384 threads are launched with 168 registers each: 256 x 216 + 128 x 72 = 384 x 168
constexpr int kLaunchRegs = 168, kSoftRegs = 216, kOtherRegs = 72;
static_assert(256 * kSoftRegs + 128 * kOtherRegs == kThreads * kLaunchRegs, "register shares");

// ---------------------------------------------------------------------------
// Scheduling: request n (made while item n is worked on) has the answer's slot n & 1.
// ---------------------------------------------------------------------------
struct Sched {
  uint4* answer;              // [2]
  uint64_t* full;             // [2]
  uint64_t* empty;            // [2], kReaders arrivals
};
SB_DEVICE bool sched_request(const Sched& s, int n, int* status) {
  const int b = n & 1;
  if (!mbar_wait(&s.empty[b], ((n >> 1) & 1) ^ 1, status)) return false;
  mbar_arrive_expect_tx(&s.full[b], 16);
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                   smem_u32(&s.answer[b])),
               "r"(smem_u32(&s.full[b]))
               : "memory");
  return true;
}
// The next item, or -1 (none left, or a wait ran out).  By a whole warp, or (WARP false) by the one lane that runs.
template <bool WARP = true>
SB_DEVICE int sched_next(const Sched& s, int n, int* status) {
  const int b = n & 1;
  bool there = mbar_wait(&s.full[b], (n >> 1) & 1, status);
  if (WARP) there = __all_sync(0xffffffffu, there);
  if (!there) return -1;
  uint32_t ok, x = 0;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b128 r;\n\t"
      "ld.shared.b128 r, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n\t}"
      : "=r"(ok), "+r"(x)
      : "r"(smem_u32(&s.answer[b]))
      : "memory");
  fence_proxy_async_smem();
  if (WARP) __syncwarp();
  if (!WARP || threadIdx.x % 32 == 0) mbar_arrive(&s.empty[b]);
  return ok != 0 ? static_cast<int>(x) : -1;
}

// Rows [row0, row0 + n) of a loaded tile (64-column chunks `next` bytes apart) that no sequence covers become zeros.
SB_DEVICE void clear_rows(uint8_t* tile, int n, int chunks, int next, int row0, int first, int last) {
  const int lane = threadIdx.x % 32;
  for (int r = lane / 8; r < n; r += 4)
    if (row0 + r < first || row0 + r >= last)
      for (int c = 0; c < chunks; ++c)
        *reinterpret_cast<uint4*>(tile + c * next + r * 128 + (lane % 8) * 16) = make_uint4(0, 0, 0, 0);
}

// ---------------------------------------------------------------------------
// Results that are computed again.  A warp keeps those that it found in a list through global memory, a slot for each of its
// items; when the CTA has no item left its eight softmax warps share all of them, row by row.
// ---------------------------------------------------------------------------
struct Later {
  int2* slots;                // [items][8]: a bit for each row (lane), the slot before or -1
  int last;
  SB_DEVICE void add(unsigned bits, int item) {        // by a whole warp
    if (bits == 0) return;
    const int slot = item * 8 + static_cast<int>(threadIdx.x) / 32;
    if (threadIdx.x % 32 == 0) slots[slot] = make_int2(static_cast<int>(bits), last);
    last = slot;
  }
  // `again(item, warp that found it, row's lane)`; `heads`: shared memory of 8 ints
  template <typename F>
  SB_DEVICE void run(int* heads, const F& again) const {
    const int warp = threadIdx.x / 32;
    if (threadIdx.x % 32 == 0) heads[warp] = last;
    __syncwarp();
    asm volatile("bar.sync 1, 256;" ::: "memory");     // the softmax warps alone
    int n = 0;
    for (int w = 0; w < 8; ++w)
      for (int slot = heads[w]; slot >= 0;) {
        const int2 s = slots[slot];
        for (unsigned bits = static_cast<unsigned>(s.x); bits != 0; bits &= bits - 1)
          if (n++ % 8 == warp) again(slot / 8, w, __ffs(bits) - 1);
        slot = s.y;
      }
  }
};

// A warp has four rows of an operand at a time, eight lanes a row: this lane's D / 8 columns, from `first_column`.
template <int D>
SB_DEVICE int first_column() { return static_cast<int>(threadIdx.x) % 8 * (D / 8); }
SB_DEVICE int quarter() { return static_cast<int>(threadIdx.x) % 32 / 8; }
template <int D, typename T>
SB_DEVICE void load_part(const T* p, float* f) {
  const uint4* v = reinterpret_cast<const uint4*>(p + first_column<D>());
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    const uint4 u = v[i];
    const T* x = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int k = 0; k < 8; ++k) f[i * 8 + k] = to_float(x[k]);
  }
}
template <int N>
SB_DEVICE float dot(const float* a, const float* b) {   // over a row's eight lanes
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) s += a[i] * b[i];
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}
// the four quarters' sums joined, to columns [c0, c1) of 16-bit rows
template <int D, typename T>
SB_DEVICE void store_part(T* out, float* acc, float scale, int c0, int c1) {
#pragma unroll
  for (int i = 0; i < D / 8; ++i) {
    acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], 8);
    acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], 16);
    acc[i] *= scale;
  }
  const int c = first_column<D>();
  if (quarter() != 0 || out == nullptr) return;
#pragma unroll
  for (int i = 0; i < D / 8; i += 8)
    if (c + i >= c0 && c + i < c1)
      *reinterpret_cast<uint4*>(out + c + i) =
          make_uint4(Half<T>::pack(acc[i], acc[i + 1]), Half<T>::pack(acc[i + 2], acc[i + 3]),
                     Half<T>::pack(acc[i + 4], acc[i + 5]), Half<T>::pack(acc[i + 6], acc[i + 7]));
}

// Whether rows [lo, st) and [end, hi) of an operand, which a result's masked zeros met, have something there that zero times
// it is NaN, in a column that is not NaN by the result's own rows (`own`: a bit for each of this lane's columns).  Where they
// have not, what is not finite in the result is its own, and a step that has gone wrong as a whole takes no longer for it.
template <int D, typename T>
SB_DEVICE bool touched(const T* p, long ld, int lo, int st, int end, int hi, uint32_t own) {
  constexpr int N = D / 8;
  constexpr int kMost = 1024;                          // rows: with more of them it is the result that is computed
  const bool open = (~own & ((1u << N) - 1)) != 0;
  if (!__any_sync(0xffffffffu, open)) return false;
  const int before = max(st - lo, 0), n = before + max(hi - end, 0);
  if (n > kMost) return true;
  uint32_t bad = 0;
#pragma unroll 4
  for (int i = quarter(); i < n; i += 4) {
    float f[N];
    load_part<D>(p + static_cast<long>(i < before ? lo + i : end + i - before) * ld, f);
#pragma unroll
    for (int k = 0; k < N; ++k) bad |= fabsf(f[k]) < INFINITY ? 0u : 1u << k;
  }
  return __any_sync(0xffffffffu, (bad & ~own) != 0);
}
template <int N>
SB_DEVICE uint32_t nan_columns(const float* f) {
  uint32_t bits = 0;
#pragma unroll
  for (int k = 0; k < N; ++k) bits |= f[k] != f[k] ? 1u << k : 0u;
  return bits;
}

// Columns [c0, c1) of one row of O by a whole warp, from what the row sees alone, if others have got into it.
template <int D, typename T>
__device__ __noinline__ void slow_o(const Args& a, int row, int h, int c0, int c1) {
  constexpr int N = D / 8;
  const T* x = static_cast<const T*>(a.qkv);
  const long kc = static_cast<long>(a.Hq + h / a.group) * D, vc = kc + static_cast<long>(a.Hkv) * D;
  float q[N], k[N], v[N], acc[N] = {};
  load_part<D>(x + row * a.ld + vc, v);
  const int q0 = row / 128 * 128, st = a.start[row];
  if (!touched<D>(x + vc, a.ld, a.start[q0] / 128 * 128, st, row + 1, min(q0 + 128, a.T), nan_columns<N>(v))) return;
  const float lse2 = a.lse[static_cast<long>(h) * a.T + row] * kLog2e;
  load_part<D>(x + row * a.ld + static_cast<long>(h) * D, q);
#pragma unroll 2
  for (int j0 = st; j0 <= row; j0 += 4) {              // the same number of times in every lane
    const int j = min(j0 + quarter(), row);
    load_part<D>(x + j * a.ld + kc, k);
    load_part<D>(x + j * a.ld + vc, v);
    const float p = ex2(dot<N>(q, k) * a.scale_log2 - lse2);
    if (j0 + quarter() <= row)
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] += p * v[i];
  }
  store_part<D>(static_cast<T*>(a.o) + row * a.o_ld + static_cast<long>(h) * D, acc, 1.f, c0, c1);
}

// P of the backward pass is normalised, so over 16384 keys a usual one is where fp16's numbers lose bits and below 3e-8 it would
// be 0.  It is at most 1 and fp16 goes to 2^16: the row values that it is computed from hold 15 more, and dV is scaled back.
template <typename T>
__device__ constexpr int kUpP = Half<T>::kFormat == 0 ? 15 : 0;

SB_DEVICE const float* row_block(const Args& a, int h, int q) {      // kUpP - lse, -delta of query q (64 apart)
  return a.rows + (static_cast<long>(h) * (a.tiles * 2) + q / 64) * 128 + q % 64;
}

// What dS is multiplied by before it is rounded to T, as a power of two's exponent: fp16 would lose the small gradients of a
// long row (do of 1e-4 over 1000 keys: dS near 1e-6, where its steps are 6e-8) and overflow with large ones.  The largest |do|
// times it lies in [1, 2): of the query's own row and head for dQ, and for dK and dV of the rows that see the key, from it to
// its sequence's end, in the heads of its group.  So what scales a row's sums hangs on what is in them and on nothing else.
// Nothing for bf16, which has fp32's range.
SB_DEVICE int shift_for(float top) {
  const int e = __float_as_int(top) >> 23;             // 0: no gradient, 255: an infinite one
  return e == 0 || e == 255 ? 0 : max(-100, min(100, 127 - e));
}
template <typename T>
SB_DEVICE int query_shift(const Args& a, int h, int row) {
  if constexpr (Half<T>::kFormat == 0) return shift_for(a.tops[static_cast<long>(h) * (a.tiles * 128) + row]);
  return 0;
}
template <typename T>
SB_DEVICE int key_shift(const Args& a, int kvh, int row) {
  if constexpr (Half<T>::kFormat == 0) return a.shifts[static_cast<long>(kvh) * (a.tiles * 128) + row];
  return 0;
}

// Columns [c0, c1) of one row of dQ.
template <int D, typename T>
__device__ __noinline__ void slow_dq(const Args& a, int row, int h, int c0, int c1) {
  constexpr int N = D / 8;
  const T* x = static_cast<const T*>(a.qkv);
  const long kc = static_cast<long>(a.Hq + h / a.group) * D, vc = kc + static_cast<long>(a.Hkv) * D;
  float q[N], g[N], k[N], v[N], acc[N] = {};
  const float* rb = row_block(a, h, row);
  const float nl = rb[0] - kUpP<T>, nd = rb[64];
  const int q0 = row / 128 * 128, st = a.start[row];
  const uint32_t own = nl != nl || nd != nd ? ~0u : 0u;
  if (!touched<D>(x + kc, a.ld, a.start[q0] / 128 * 128, st, row + 1, min(q0 + 128, a.T), own)) return;
  load_part<D>(x + row * a.ld + static_cast<long>(h) * D, q);
  load_part<D>(static_cast<const T*>(a.dout) + row * a.do_ld + static_cast<long>(h) * D, g);
#pragma unroll 2
  for (int j0 = st; j0 <= row; j0 += 4) {
    const int j = min(j0 + quarter(), row);
    load_part<D>(x + j * a.ld + kc, k);
    load_part<D>(x + j * a.ld + vc, v);
    const float p = ex2(dot<N>(q, k) * a.scale_log2 + nl), ds = p * (dot<N>(g, v) + nd);
    if (j0 + quarter() <= row)
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] += ds * k[i];
  }
  store_part<D>(static_cast<T*>(a.dqkv) + row * a.dqkv_ld + static_cast<long>(h) * D, acc, a.scale, c0, c1);
}

// One row of dK (want_k) or dV of key head kvh, over query heads [h0, h1), to 16 bits or, where a split's sum follows, fp32.
template <int D, typename T>
__device__ __noinline__ void slow_dkv(const Args& a, int row, int kvh, int h0, int h1, bool want_k, float* partial) {
  constexpr int N = D / 8;
  const T* x = static_cast<const T*>(a.qkv);
  const T* dout = static_cast<const T*>(a.dout);
  const long kc = static_cast<long>(a.Hq + kvh) * D, vc = kc + static_cast<long>(a.Hkv) * D;
  float q[N], g[N], k[N], v[N], acc[N] = {};
  const int k0 = row / 128 * 128, hi = min(k0 + (a.stop[min(k0 + 127, a.T - 1)] - k0 + 127) / 128 * 128, a.T);
  const int end = a.stop[row];
  uint32_t own = 0;
  for (int h = h0; h < h1; ++h) {
    const float* rb = row_block(a, h, row);
    load_part<D>(dout + row * a.do_ld + static_cast<long>(h) * D, g);
    own |= rb[0] != rb[0] || (want_k && rb[64] != rb[64]) ? ~0u : want_k ? 0u : nan_columns<N>(g);
  }
  bool others = false;
  for (int h = h0; h < h1 && !others; ++h)
    others = touched<D>((want_k ? x : dout) + static_cast<long>(h) * D, want_k ? a.ld : a.do_ld, k0, row, end, hi, own);
  if (!others) return;
  load_part<D>(x + row * a.ld + kc, k);
  load_part<D>(x + row * a.ld + vc, v);
  for (int h = h0; h < h1; ++h)
#pragma unroll 2
    for (int j0 = row; j0 < end; j0 += 4) {
      const int j = min(j0 + quarter(), end - 1);
      load_part<D>(x + j * a.ld + static_cast<long>(h) * D, q);
      load_part<D>(dout + j * a.do_ld + static_cast<long>(h) * D, g);
      const float* rb = row_block(a, h, j);
      const float p = ex2(dot<N>(q, k) * a.scale_log2 + (rb[0] - kUpP<T>));
      const float ds = p * (dot<N>(g, v) + rb[64]);
      if (j0 + quarter() < end)
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] += want_k ? ds * q[i] : p * g[i];
    }
  T* out = static_cast<T*>(a.dqkv) + row * a.dqkv_ld + (want_k ? kc : vc);
  store_part<D>(partial != nullptr ? static_cast<T*>(nullptr) : out, acc, want_k ? a.scale : 1.f, 0, D);
  if (partial != nullptr && quarter() == 0)
#pragma unroll
    for (int i = 0; i < N; i += 4)
      *reinterpret_cast<float4*>(partial + first_column<D>() + i) = make_float4(acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
}

}  // namespace pa
}  // namespace sb

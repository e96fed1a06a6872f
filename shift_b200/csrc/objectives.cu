// Losses of label log-probabilities, straight from the logits: the log-probability of every row's label with its gradient,
// the clipped policy loss with a KL term, the preference loss of pairs of sequences.
//
//   lse = log sum_v exp z_v,   logp = z_label - lse,   dL/dz_v = d ([v = label] - exp(z_v - lse)),   d = dL/dlogp
//
// All of them move logits: a row has V values of 2 or 4 bytes and a few of its own.  Rows are cut over a cluster of 1, 2,
// 4 or 8 CTAs (joined over distributed shared memory in rank order) where a slice would not stay in shared memory, or
// where there are too few rows for the SMs.  Maxima are fp32, one running pair of maximum and sum a thread; the sums are
// joined in 64 bits, and so is computed what follows from a row's sum (its logarithm, ratios, the clip's comparison), because
// a ratio next to the clip's border decides a whole row's gradient and a pair of sequences adds up hundreds of rows.  A row's
// log-probability is off by 1e-8 (rms, 32768 logits of a model's spread; on average by less than 1e-9).
#include <cooperative_groups.h>

#include "common.cuh"
#include "lowp.cuh"
#include "objectives.h"

namespace cg = cooperative_groups;

namespace sb {
namespace obj {

constexpr float kLog2e = 1.4426950408889634f;

SB_DEVICE float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// exp(z - m); m is finite.  The difference is rounded before it is scaled, so the error goes with |z - m|, not with |z|.  For
// sums log2(e) has 48 bits: with 24 a value far below the maximum is too large, by 8e-8 at -6 and 1.9e-7 at -14.
constexpr float kLog2eLow = 1.9259630e-8f;
SB_DEVICE float exp_diff(float z, float m) { return ex2(__fmaf_rn(z - m, kLog2e, (z - m) * kLog2eLow)); }

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
SB_DEVICE float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
  return d;
}
// the same of two values, two operations an instruction; `minus`: -m twice
SB_DEVICE float2 exp_sum2(float2 z, float2 minus) {
  z = add2(z, minus);
  z = fma2(z, make_float2(kLog2e, kLog2e), mul2(z, make_float2(kLog2eLow, kLog2eLow)));
  return make_float2(ex2(z.x), ex2(z.y));
}
// for a gradient's value, which is rounded by itself
SB_DEVICE float2 exp_diff2(float2 z, float2 minus) {
  z = mul2(add2(z, minus), make_float2(kLog2e, kLog2e));
  return make_float2(ex2(z.x), ex2(z.y));
}

// A 16-byte vector as pairs of fp32 values, back, and its largest value (NaN apart; 16-bit values two at a time).
template <typename T>
struct Elem;
template <>
struct Elem<__nv_bfloat16> {
  static SB_DEVICE void unpack(const uint4& u, float2* f) {
    f[0] = unpack_bf16x2(u.x);
    f[1] = unpack_bf16x2(u.y);
    f[2] = unpack_bf16x2(u.z);
    f[3] = unpack_bf16x2(u.w);
  }
  static SB_DEVICE uint4 pack(const float2* f) {
    return make_uint4(pack_bf16x2(f[0].x, f[0].y), pack_bf16x2(f[1].x, f[1].y), pack_bf16x2(f[2].x, f[2].y),
                      pack_bf16x2(f[3].x, f[3].y));
  }
  static SB_DEVICE float top(const uint4& u, const float2*) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
    const float2 m = __bfloat1622float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    return fmaxf(m.x, m.y);
  }
};
template <>
struct Elem<__half> {
  static SB_DEVICE void unpack(const uint4& u, float2* f) {
    const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __half22float2(h[i]);
  }
  static SB_DEVICE uint4 pack(const float2* f) {
    uint4 u;
    __half2* h = reinterpret_cast<__half2*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(f[i].x, f[i].y);
    return u;
  }
  static SB_DEVICE float top(const uint4& u, const float2*) {
    const __half2* h = reinterpret_cast<const __half2*>(&u);
    const float2 m = __half22float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    return fmaxf(m.x, m.y);
  }
};
template <>
struct Elem<float> {
  static SB_DEVICE void unpack(const uint4& u, float2* f) {
    f[0] = make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
    f[1] = make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
  }
  static SB_DEVICE uint4 pack(const float2* f) {
    return make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y), __float_as_uint(f[1].x), __float_as_uint(f[1].y));
  }
  static SB_DEVICE float top(const uint4&, const float2* f) { return fmaxf(fmaxf(f[0].x, f[0].y), fmaxf(f[1].x, f[1].y)); }
};

// The part of a row that one CTA of a cluster has: whole 16-byte vectors [v0, v1) of the row's aligned middle; rank 0 also
// the single values before and behind it (a row may start on any value's alignment).
template <typename T>
struct Slice {
  static constexpr int E = 16 / sizeof(T);
  T* row;
  int head, tail, V, v0, v1;
  bool edges;
  SB_DEVICE Slice(T* r, int V_, int rank, int ranks) : row(r), V(V_) {
    head = min(V, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(r) & 15)) & 15) / static_cast<int>(sizeof(T)));
    const int nv = (V - head) / E;
    tail = V - head - nv * E;
    v0 = static_cast<int>(static_cast<long>(nv) * rank / ranks);
    v1 = static_cast<int>(static_cast<long>(nv) * (rank + 1) / ranks);
    edges = rank == 0;
  }
  SB_DEVICE uint4* vec(int v) const { return reinterpret_cast<uint4*>(row + head) + v; }
  // the edge value of this thread, or -1 (there are at most 2 E - 2 of them)
  SB_DEVICE int edge() const {
    const int t = threadIdx.x;
    return !edges || t >= head + tail ? -1 : t < head ? t : V - tail + (t - head);
  }
};

// The hardware's exponential is too small on average: by 2.2e-8 over arguments in [-ln 2, 0] and 5.05e-8 below (of 4 million
// each), 3.6e-8 where arguments are spread evenly and count by their values; at 0 it is exact.  All sums of a row would share
// that, and a pair of sequences adds up hundreds of rows, so sums put it back.
constexpr float kTooSmall = 3.6e-8f;
SB_DEVICE float too_small(float x) { return x > -0.6931472f ? 2.2e-8f : 5.05e-8f; }

// Running (maximum, sum of exp(z - maximum)); an empty one, or one of -inf alone, has maximum -inf and sum 0.  The sum is
// s + low: beside the term of a likely label, which is 1, the roundings of a thread's additions would be as large as the rest
// (rows whose label has 20 more than the others: off by 1.2e-7 rms instead of 4.2e-8, where the kernel saves 2 %).
struct Run {
  float m = -INFINITY, s = 0.f, low = 0.f;
  SB_DEVICE void rise(float b) {
    if (b > m) {
      const float f = m == -INFINITY ? 0.f : exp_diff(m, b);
      s = __fmaf_rn(s, f, __fmaf_rn(s, f * too_small(m - b), low * f));            // rounded once, after it was put back
      low = 0.f;
      m = b;
    }
  }
  SB_DEVICE void plus(float x) {                   // exactly: what t does not hold goes to `low`
    const float t = s + x, y = t - s;
    low += (s - (t - y)) + (x - y);
    s = t;
  }
  // One vector of values that are at most m, or one value.  NaN has no place in a maximum, so a row of NaN and -inf alone gets
  // here with m = -inf; among infinite values the sum counts those, so that its logarithm adds nothing.
  template <int N>
  SB_DEVICE void add(const float2* z) {
    if (m == INFINITY) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        s += (z[i].x == INFINITY ? 1.f : exp_diff(z[i].x, m)) + (z[i].y == INFINITY ? 1.f : exp_diff(z[i].y, m));
      return;
    }
    const float at = m == -INFINITY ? 0.f : -m;
    float2 part = exp_sum2(z[0], make_float2(at, at));
#pragma unroll
    for (int i = 1; i < N; ++i) part = add2(part, exp_sum2(z[i], make_float2(at, at)));
    plus(part.x + part.y);
  }
  SB_DEVICE void add(float z) {
    rise(z);
    plus(z == INFINITY ? 1.f : exp_diff(z, m == -INFINITY ? 0.f : m));
  }
  // in 64 bits; the largest term was exact
  SB_DEVICE double sum() const {
    const double t = static_cast<double>(s) + static_cast<double>(low);
    return s > 1.f && m < INFINITY ? t + static_cast<double>(kTooSmall) * (t - 1.0) : t;
  }
};

// The same of a whole row, or of a part of it, in 64 bits.
struct RowRun {
  float m = -INFINITY;
  double s = 0.0;
  // the sum over another maximum, at least this one
  SB_DEVICE double over(float top) const {
    if (m == top) return s;
    if (m == -INFINITY) return s == s ? 0.0 : s;
    return s * (static_cast<double>(exp_diff(m, top)) * (1.0 + too_small(m - top)));
  }
};

// All threads' runs joined over the CTA and the cluster, in an order that does not change; every thread gets the result.
// The maximum first, so that every sum is scaled once.
SB_DEVICE RowRun join_all(Run r, int ranks) {
  __shared__ float tops[kThreads / 32], mine_m;
  __shared__ double sums[kThreads / 32], mine_s;
  const int warp = threadIdx.x / 32;
  RowRun all;
  all.m = warp_max(r.m);
  if (threadIdx.x % 32 == 0) tops[warp] = all.m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) all.m = fmaxf(all.m, tops[w]);
  RowRun own;
  own.m = r.m;
  own.s = r.sum();
  double s = own.over(all.m);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (threadIdx.x % 32 == 0) sums[warp] = s;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) all.s += sums[w];
  if (ranks == 1) return all;
  if (threadIdx.x == 0) {
    mine_m = all.m;
    mine_s = all.s;
  }
  cg::cluster_group cl = cg::this_cluster();
  cl.sync();
  RowRun row;
  for (int k = 0; k < ranks; ++k) row.m = fmaxf(row.m, *cl.map_shared_rank(&mine_m, k));
  for (int k = 0; k < ranks; ++k) {
    RowRun one;
    one.m = *cl.map_shared_rank(&mine_m, k);
    one.s = *cl.map_shared_rank(&mine_s, k);
    row.s += one.over(row.m);
  }
  cl.sync();                                       // nobody leaves while it is read
  return row;
}

// d (onehot - softmax) of one vector; `p` of two values is their softmax
template <typename T, typename P>
SB_DEVICE uint4 grad_of(const uint4& u, int v, int owner, int at, float d, const P& p) {
  constexpr int N = Slice<T>::E / 2;
  float2 z[N];
  Elem<T>::unpack(u, z);
#pragma unroll
  for (int i = 0; i < N; ++i) z[i] = mul2(p(z[i]), make_float2(-d, -d));
  if (v == owner) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (2 * i == at) z[i].x += d;
      if (2 * i + 1 == at) z[i].y += d;
    }
  }
  return Elem<T>::pack(z);
}
// the slice's vector that holds the label, or -1
template <typename T>
SB_DEVICE int label_vec(const Slice<T>& s, int label) {
  return label >= s.head && label < s.V - s.tail ? (label - s.head) / Slice<T>::E : -1;
}
template <typename T, typename P>
SB_DEVICE void write_edge(const Slice<T>& s, int label, float d, const P& p) {
  const int e = s.edge();
  if (e >= 0) s.row[e] = from_float<T>((e == label ? d : 0.f) - d * p(make_float2(to_float(s.row[e]), 0.f)).x);
}
// rows without a label, or clipped: no value of theirs is looked at
template <typename T>
SB_DEVICE void write_zeros(const Slice<T>& s) {
  for (int v = s.v0 + threadIdx.x; v < s.v1; v += kThreads) *s.vec(v) = make_uint4(0, 0, 0, 0);
  const int e = s.edge();
  if (e >= 0) s.row[e] = from_float<T>(0.f);
}
template <typename T, typename P>
SB_DEVICE void write_grad(const Slice<T>& s, int label, float d, const P& p) {
  const int owner = label_vec(s, label), at = owner < 0 ? 0 : (label - s.head) % Slice<T>::E;
  constexpr int U = 4;                             // vectors in flight
  for (int v = s.v0 + threadIdx.x; v < s.v1; v += U * kThreads) {
    uint4 u[U];
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (v + k * kThreads < s.v1) u[k] = *s.vec(v + k * kThreads);
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (v + k * kThreads < s.v1) *s.vec(v + k * kThreads) = grad_of<T>(u[k], v + k * kThreads, owner, at, d, p);
  }
  write_edge(s, label, d, p);
}

template <typename T>
SB_DEVICE void add_edge(Run& r, const Slice<T>& s) {
  const int e = s.edge();
  if (e >= 0) r.add(to_float(s.row[e]));
}
// This thread's vectors of [v0, v1), four at a time, whose maximum is taken first: it then rises a few times a row.
template <typename T, typename L>
SB_DEVICE void add_vectors(Run& r, int v0, int v1, const L& load) {
  constexpr int U = 4, N = Slice<T>::E / 2;
  for (int v = v0 + static_cast<int>(threadIdx.x); v < v1; v += U * kThreads) {
    uint4 u[U];
    float2 z[N];
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (v + k * kThreads < v1) u[k] = load(v + k * kThreads);
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (v + k * kThreads < v1) {
        Elem<T>::unpack(u[k], z);
        top = fmaxf(top, Elem<T>::top(u[k], z));
      }
    r.rise(top);
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (v + k * kThreads < v1) {
        Elem<T>::unpack(u[k], z);
        r.add<N>(z);
      }
  }
}
template <typename T>
SB_DEVICE Run read_row(const Slice<T>& s) {
  Run r;
  add_vectors<T>(r, s.v0, s.v1, [&](int v) { return *s.vec(v); });
  add_edge(r, s);
  return r;
}

// logp and lse of every row: one pass over the logits.
template <typename T>
__global__ void __launch_bounds__(kThreads) logp_kernel(const Args a) {
  const long r = blockIdx.x / a.ranks;
  const Slice<T> s(static_cast<T*>(a.logits) + r * a.stride, a.V, blockIdx.x % a.ranks, a.ranks);
  const RowRun run = join_all(read_row(s), a.ranks);
  if (threadIdx.x == 0 && s.edges) {
    const int label = a.labels[r];
    const bool live = label >= 0 && label < a.V;
    const double l = log(run.s);
    const double logp = live ? static_cast<double>(to_float(s.row[label])) - static_cast<double>(run.m) - l : 0.0;
    const double lse = static_cast<double>(run.m) + l, left = lse - static_cast<double>(static_cast<float>(lse));
    a.lse[r] = static_cast<float>(lse);
    if (a.lse_low != nullptr) a.lse_low[r] = left == left ? static_cast<float>(left) : 0.f;     // infinities have none
    if (a.logp64 != nullptr) a.logp64[r] = logp;
    else a.logp[r] = static_cast<float>(logp);
  }
}

// The gradient at the logits, over them, from lse and dL/dlogp: read and write once.
template <typename T>
__global__ void __launch_bounds__(kThreads) grad_kernel(const Args a) {
  const long r = blockIdx.x / a.ranks;
  const Slice<T> s(static_cast<T*>(a.logits) + r * a.stride, a.V, blockIdx.x % a.ranks, a.ranks);
  const int label = a.labels[r];
  const float d = label >= 0 && label < a.V ? a.dlogp[r] : 0.f;
  const float lse = a.lse[r];
  // lse near 1000 has steps of 6e-5, which every softmax value would carry; what it left comes in with the scaling
  const float low = a.lse_low != nullptr ? a.lse_low[r] * -kLog2e : 0.f;
  if (d == 0.f) write_zeros(s);
  else
    write_grad(s, label, d, [&](float2 z) {
      z = fma2(add2(z, make_float2(-lse, -lse)), make_float2(kLog2e, kLog2e), make_float2(low, low));
      return make_float2(ex2(z.x), ex2(z.y));
    });
}

SB_DEVICE void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
SB_DEVICE void bulk_store(void* dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(smem_u32(src)), "r"(bytes)
               : "memory");
}

// Loss, log-probability and gradient of every row in one pass: the row's slice waits in shared memory (KEEP) for its sum.
// It comes and goes by bulk copies in kParts parts, so that all of it is in flight at once and three CTAs an SM keep the
// memory busy while one of them computes.  16384 x 32768 bf16: with loads and stores of the threads 494 us (16 KB in flight
// a CTA), in 8 / 4 / 2 / 1 parts 452 / 412 / 392 / 401 us; CTAs that go on to their next rows 468 us.
constexpr int kParts = 2;

template <typename T, bool KEEP>
__global__ void __launch_bounds__(kThreads) policy_kernel(const Args a) {
  extern __shared__ uint4 held[];
  __shared__ uint64_t bar[kParts];
  __shared__ float s_d;
  const long r = blockIdx.x / a.ranks;
  const Slice<T> s(static_cast<T*>(a.logits) + r * a.stride, a.V, blockIdx.x % a.ranks, a.ranks);
  const int n = s.v1 - s.v0;
  auto part = [&](int c) { return s.v0 + static_cast<int>(static_cast<long>(n) * c / kParts); };
  if (KEEP && threadIdx.x == 0) {
    for (int c = 0; c < kParts; ++c) mbar_init(&bar[c], 1);
    fence_barrier_init();
    for (int c = 0; c < kParts; ++c) {
      const uint32_t bytes = static_cast<uint32_t>(part(c + 1) - part(c)) * 16;
      mbar_arrive_expect_tx(&bar[c], bytes);
      if (bytes > 0) bulk_load(held + (part(c) - s.v0), s.vec(part(c)), bytes, &bar[c]);
    }
  }
  const int label = a.labels[r];
  const bool live = label >= 0 && label < a.V;
  double zl = 0, old = 0, adv = 0, ref = 0, weight = 1;
  const bool kl = a.t.ref != nullptr && a.t.kl != 0.0;
  if (threadIdx.x == 0 && live) {                  // early; the label's logit before any CTA of the row writes over it
    zl = to_float(s.row[label]);
    old = a.t.old[r];
    adv = a.t.adv[r];
    if (kl) ref = a.t.ref[r];
    if (a.t.weight != nullptr) weight = a.t.weight[r];
  }
  Run mine;
  bool late = false;
  if (KEEP) {
    __syncthreads();                               // the barriers are there
    for (int c = 0; c < kParts; ++c) {
      late |= !mbar_wait(&bar[c], 0, a.status);
      add_vectors<T>(mine, part(c), part(c + 1), [&](int v) { return held[v - s.v0]; });
    }
    add_edge(mine, s);
    if (late)                                      // the status says so; what was on its way here lands before anything else
      for (int c = 0; c < kParts; ++c) mbar_wait(&bar[c], 0, nullptr, 10000000ull);
  } else {
    mine = read_row(s);
  }
  const RowRun run = join_all(mine, a.ranks);
  if (threadIdx.x == 0) {
    double loss = 0, logp = 0, d = 0;
    if (live) {
      logp = zl - static_cast<double>(run.m) - log(run.s);
      const double ratio = exp(logp - old), clipped = fmin(fmax(ratio, 1.0 - a.t.low), 1.0 + a.t.high);
      const double gain = adv == 0.0 && ratio == ratio ? 0.0 : ratio * adv, cut = clipped * adv;
      const bool open = gain <= cut;
      loss = -(open ? gain : cut);
      d = open ? -gain : 0.0;
      if (gain != gain) loss = d = gain;
      if (kl) {
        const double gap = ref - logp, e = expm1(gap);
        loss += a.t.kl * (e - gap);
        d -= a.t.kl * e;
      }
      d *= a.t.scale * weight;
    }
    s_d = static_cast<float>(d);
    if (s.edges) {
      a.t.loss[r] = static_cast<float>(loss);
      a.logp[r] = static_cast<float>(logp);
    }
  }
  __syncthreads();
  const float d = s_d, inv = static_cast<float>(1.0 / run.s), m = run.m;
  if (d == 0.f) {
    write_zeros(s);
    return;
  }
  auto p = [&](float2 z) { return mul2(exp_diff2(z, make_float2(-m, -m)), make_float2(inv, inv)); };
  if (!KEEP) {
    write_grad(s, label, d, p);
    return;
  }
  const int owner = label_vec(s, label), at = owner < 0 ? 0 : (label - s.head) % Slice<T>::E;
  for (int c = 0; c < kParts; ++c) {
    const int end = part(c + 1);
    for (int v = part(c) + threadIdx.x; v < end; v += kThreads)
      held[v - s.v0] = grad_of<T>(held[v - s.v0], v, owner, at, d, p);
    fence_proxy_async_smem();
    __syncthreads();
    if (threadIdx.x == 0 && part(c + 1) > part(c))
      bulk_store(s.vec(part(c)), held + (part(c) - s.v0), static_cast<uint32_t>(part(c + 1) - part(c)) * 16);
  }
  write_edge(s, label, d, p);
  if (threadIdx.x == 0) {                          // shared memory stays until it was read
    bulk_commit_group();
    bulk_wait_group_read<0>();
  }
}

// Pairs of sequences (2 p chosen, 2 p + 1 rejected): one CTA a pair sums logp - ref over each sequence's labelled rows,
// and writes the loss, the margin and every row's dL/dlogp.  Rows of no pair get 0.
__global__ void __launch_bounds__(kThreads)
pair_kernel(const double* __restrict__ logp, const float* __restrict__ ref, const int* __restrict__ labels, int V,
            const int* __restrict__ offs, int T, float beta, float scale, float* __restrict__ loss,
            float* __restrict__ margin, float* __restrict__ dlogp) {
  __shared__ int bound[3];
  __shared__ double part[kThreads / 32];
  const int p = blockIdx.x, warp = threadIdx.x / 32;
  if (threadIdx.x < 3) bound[threadIdx.x] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i <= 2 * p + 2; i += kThreads) {       // an offset below one before counts as that one
    const int b = min(offs[i], T);
    for (int k = max(0, i - 2 * p); k < 3; ++k) atomicMax(&bound[k], b);
  }
  __syncthreads();
  double sums[2];
  for (int k = 0; k < 2; ++k) {
    double sum = 0;
    for (int r = bound[k] + threadIdx.x; r < bound[k + 1]; r += kThreads)
      if (labels[r] >= 0 && labels[r] < V) sum += logp[r] - static_cast<double>(ref[r]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (threadIdx.x % 32 == 0) part[warp] = sum;
    __syncthreads();
    sums[k] = part[0];
    for (int w = 1; w < kThreads / 32; ++w) sums[k] += part[w];
    __syncthreads();
  }
  const double h = static_cast<double>(beta) * (sums[0] - sums[1]);
  if (threadIdx.x == 0) {
    margin[p] = static_cast<float>(h);
    loss[p] = static_cast<float>(fmax(-h, 0.0) + log1p(exp(-fabs(h))));
    if (h != h) loss[p] = static_cast<float>(h);
  }
  const float d = static_cast<float>(static_cast<double>(beta) * scale / (1.0 + exp(h)));
  for (int r = bound[0] + threadIdx.x; r < bound[2]; r += kThreads) dlogp[r] = r < bound[1] ? -d : d;
  if (p == 0)
    for (int r = threadIdx.x; r < bound[0]; r += kThreads) dlogp[r] = 0.f;
  if (p == static_cast<int>(gridDim.x) - 1)
    for (int r = bound[2] + threadIdx.x; r < T; r += kThreads) dlogp[r] = 0.f;
}

template <typename F>
static cudaError_t launch(F* kernel, const Args& a, size_t smem, cudaStream_t stream) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(a.rows * a.ranks));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(a.ranks);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // Without opting in a kernel has 48 KB, its static shared memory (some 100 bytes: barriers, sums) among it.
  if (smem > 40 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kHeldMost);
    if (e != cudaSuccess) return e;
  }
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <typename T>
static cudaError_t run_typed(Kernel k, const Args& a, cudaStream_t stream) {
  switch (k) {
    case kLogp: return launch(logp_kernel<T>, a, 0, stream);
    case kGrad: return launch(grad_kernel<T>, a, 0, stream);
    default: break;
  }
  const size_t held = (static_cast<size_t>(a.V) * sizeof(T) / 16 / a.ranks + 1) * 16;
  return held <= kHeldMost ? launch(policy_kernel<T, true>, a, held, stream) : launch(policy_kernel<T, false>, a, 0, stream);
}

cudaError_t run(Kernel k, Type type, const Args& a, cudaStream_t stream) {
  return type == kBf16 ? run_typed<__nv_bfloat16>(k, a, stream)
         : type == kF16 ? run_typed<__half>(k, a, stream) : run_typed<float>(k, a, stream);
}

cudaError_t run_pairs(int pairs, const double* logp, const float* ref, const int* labels, int V, const int* offs, int T,
                      float beta, float scale, float* loss, float* margin, float* dlogp, cudaStream_t stream) {
  pair_kernel<<<pairs, kThreads, 0, stream>>>(logp, ref, labels, V, offs, T, beta, scale, loss, margin, dlogp);
  return cudaGetLastError();
}

}  // namespace obj
}  // namespace sb

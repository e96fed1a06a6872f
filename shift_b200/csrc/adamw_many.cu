// One AdamW update of many tensors, moments in fp32 or in 8 bits.
//
// With bias corrections c1 = 1 - beta1^t and c2 = sqrt(1 - beta2^t):
//   g  = grad * grad_scale
//   w  = w (1 - lr wd)
//   m += (g - m) (1 - beta1)          v = beta2 v + (1 - beta2) g^2
//   w -= lr / c1 * m / (sqrt(v) / c2 + eps)
// in fp32, the order of the single-buffer step in xent_adam.cu.  The 8-bit
// form keeps m and r = sqrt(v) as e4m3 codes with a power-of-two scale per 128
// elements (fp8.cuh).  r instead of v halves the exponent range that the codes
// have to cover.  Magnitudes are rounded up with the probability of their
// distance from the code below: v moves by a thousandth per step against a
// half step of 6 %, so rounding to nearest would freeze it.  A root above zero
// never goes to code 0, though: m of the same element may keep a code, and an
// update divided by nothing is hundreds of learning rates (an element 1e-6 of
// its block's largest).  At code 1 its update is too small instead.  The random
// bits are a counter hash of (seed, tensor number, element), hence the same for
// any launch shape; elements 2^32 apart share them.  Codes and scales are those
// of the CPU's statement, bit for bit but for the sign of a zero.
//
// Bound: DRAM with 32-bit moments (0.494 B elements: 2.07 ms, 6.7 TB/s);
// instructions with 8-bit ones (2.03 ms, 3.9 TB/s, 105 instructions an element).
// The tensors' pointers travel as kernel parameters, so a step is one launch
// per 320 tensors, needs no device table and can be captured.  One pass of 8
// elements a thread: four passes of a CTA, for one search of its tensor, were
// slower (134 M elements: 516 us against 481).
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <memory>
#include <utility>

#include "fp8.cuh"

namespace sb {
namespace adam {

constexpr int kThreads = 256;
constexpr int kVec = 8;                        // elements per thread and pass
constexpr int kChunk = kThreads * kVec;        // elements per CTA: 16 blocks of 128
constexpr int kMaxTensors = 320;

struct Entry {
  void* p;             // parameter
  float* w;            // fp32 master copy, or null: the parameter itself is updated
  const void* g;
  void *m, *v;         // fp32, or codes
  uint8_t *ms, *vs;    // scales of the codes
  long n;
};

struct Table {
  Entry e[kMaxTensors];
  uint32_t end[kMaxTensors];   // chunks of tensors 0..t, cumulated
  uint16_t number[kMaxTensors];   // the tensor's number in the caller's list | 0x8000: vectors are aligned
  int count;
};

struct StepArgs {
  // 1 - beta is taken in double on the host: in fp32 it would lose the digits that beta has in common with 1
  float lr, beta2, one_minus_beta1, one_minus_beta2, eps, wd, c1, c2, grad_scale;
  uint32_t seed;
  const int* sdev;       // optional: seed, lr, c1, c2 from device memory
  const int* skip;       // optional: a non-zero word leaves everything as it is
  int* nonfinite;        // optional: set where a scaled gradient is not finite
};

// Integer mix of two multiplications, constants and shifts as Chris Wellons published them ("Prospecting for hash
// functions", 2018); stated again in ops/reference.py.
SB_DEVICE uint32_t mix32(uint32_t h) {
  h = (h ^ (h >> 16)) * 0x7FEB352Du;
  h = (h ^ (h >> 15)) * 0x846CA68Bu;
  return h ^ (h >> 16);
}

// y in [-448, 448] to the e4m3 value next to it towards zero or away from it:
// random bits (16, in place) are added below the three kept fraction bits, then
// cut off; in sign and magnitude that needs no care for the sign.  Below the
// smallest normal value 2^-6 the grid is uniform, as it is in [2^-6, 2^-5), so
// y is moved there and back.
SB_DEVICE float round_up_sometimes(float y, uint32_t bits) {
  const float shift = fabsf(y) < 0.015625f ? __uint_as_float(0x3C800000u | (__float_as_uint(y) & 0x80000000u)) : 0.f;
  return __uint_as_float((__float_as_uint(y + shift) + bits) & ~0xFFFFFu) - shift;
}

// One-instruction root (off by at most 2^-22 relative, zero and infinity exact).
SB_DEVICE float root(float x) {
  float r;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

template <typename T>
SB_DEVICE float as_float(T x);
template <>
SB_DEVICE float as_float<float>(float x) { return x; }
template <>
SB_DEVICE float as_float<__half>(__half x) { return __half2float(x); }
template <>
SB_DEVICE float as_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
SB_DEVICE T from_float(float x);
template <>
SB_DEVICE float from_float<float>(float x) { return x; }
template <>
SB_DEVICE __half from_float<__half>(float x) { return __float2half(x); }
template <>
SB_DEVICE __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16(x); }

template <typename T>
SB_DEVICE void load8(const T* p, int valid, bool vec, float* f) {
  if (vec && valid == kVec) {
    constexpr int W = sizeof(T) * kVec / 4;
    uint32_t raw[W];
    if constexpr (W >= 4) {
#pragma unroll
      for (int i = 0; i < W / 4; ++i) reinterpret_cast<uint4*>(raw)[i] = reinterpret_cast<const uint4*>(p)[i];
    } else {
      *reinterpret_cast<uint2*>(raw) = *reinterpret_cast<const uint2*>(p);
    }
#pragma unroll
    for (int i = 0; i < kVec; ++i) f[i] = as_float<T>(reinterpret_cast<const T*>(raw)[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i) f[i] = i < valid ? as_float<T>(p[i]) : 0.f;
  }
}

template <typename T>
SB_DEVICE void store8(T* p, int valid, bool vec, const float* f) {
  if (vec && valid == kVec) {
    T t[kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i) t[i] = from_float<T>(f[i]);
    const uint4* raw = reinterpret_cast<const uint4*>(t);
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = raw[i];
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      if (i < valid) p[i] = from_float<T>(f[i]);
  }
}

// Eight codes of a block times its scale.
SB_DEVICE void load_codes(const uint8_t* p, float scale, int valid, bool vec, float* f) {
  uint32_t raw[2] = {0, 0};
  if (vec && valid == kVec) {
    *reinterpret_cast<uint2*>(raw) = *reinterpret_cast<const uint2*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      if (i < valid) raw[i / 4] |= static_cast<uint32_t>(p[i]) << (8 * (i % 4));
  }
#pragma unroll
  for (int i = 0; i < kVec / 2; ++i) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(
        static_cast<__nv_fp8x2_storage_t>(raw[i / 2] >> (16 * (i % 2))), __NV_E4M3);
    const float2 v = __half22float2(__half2(h));
    f[2 * i] = v.x * scale;
    f[2 * i + 1] = v.y * scale;
  }
}

// Eight values of a block of 128 (16 lanes) to codes; returns the scale byte.
// ROOT: values of zero or more, of which those above zero get code 1 at least.
template <bool ROOT>
SB_DEVICE int store_codes(uint8_t* p, float* f, const uint32_t* bits, int valid, bool vec) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < kVec; ++i) top = fmaxf(top, fabsf(f[i]));
  if (top == INFINITY) {                         // infinities do not count (fmaxf passes over NaN)
    top = 0.f;
#pragma unroll
    for (int i = 0; i < kVec; ++i) top = fmaxf(top, fabsf(f[i]) < INFINITY ? fabsf(f[i]) : 0.f);
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const int byte = fp8::scale_byte(top, fp8::kE4M3);
  const float inv = fp8::inv_scale(byte);
  if constexpr (ROOT) {
    const float one = fp8::scale_of(byte) * 0.001953125f;      // what code 1 stands for, exactly
    float low = f[0];
#pragma unroll
    for (int i = 1; i < kVec; ++i) low = fminf(low, f[i]);
    if (low < one) {                             // rare: a look at each of the eight only then
#pragma unroll
      for (int i = 0; i < kVec; ++i) f[i] = f[i] > 0.f ? fmaxf(f[i], one) : f[i];
    }
  }
  uint32_t raw[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < kVec; i += 2) {
    float y[2];
#pragma unroll
    for (int j = 0; j < 2; ++j)                  // 0 x adds nothing to a finite value and makes NaN of any other
      y[j] = __fmaf_rn(f[i + j], 0.f, round_up_sometimes(f[i + j] * inv, bits[i + j]));
    raw[i / 4] |= fp8::pack2(y[0], y[1], fp8::kE4M3) << (16 * ((i / 2) % 2));
  }
  if (vec && valid == kVec) {
    *reinterpret_cast<uint2*>(p) = make_uint2(raw[0], raw[1]);
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      if (i < valid) p[i] = static_cast<uint8_t>(raw[i / 4] >> (8 * (i % 4)));
  }
  return byte;
}

template <typename P, typename Gr, bool EIGHT>
__global__ void __launch_bounds__(kThreads)
adamw_many_kernel(const __grid_constant__ Table tab, StepArgs a) {
  if (a.skip != nullptr && *a.skip != 0) return;
  if (a.sdev != nullptr) {
    a.seed = static_cast<uint32_t>(a.sdev[0]);
    a.lr = __int_as_float(a.sdev[1]);
    a.c1 = __int_as_float(a.sdev[2]);
    a.c2 = __int_as_float(a.sdev[3]);
  }
  // the tensor whose chunks cover this CTA
  int lo = 0, hi = tab.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (tab.end[mid] > blockIdx.x) hi = mid;
    else lo = mid + 1;
  }
  const Entry& e = tab.e[lo];
  const uint32_t first = lo == 0 ? 0 : tab.end[lo - 1];
  const bool vec = (tab.number[lo] & 0x8000u) != 0;
  const uint32_t key = mix32(mix32(a.seed) ^ ((tab.number[lo] & 0x7FFFu) * 0x9E3779B1u));
  const long i0 = static_cast<long>(blockIdx.x - first) * kChunk + threadIdx.x * kVec;
  const int valid = static_cast<int>(max(0l, min(static_cast<long>(kVec), e.n - i0)));

  float g[kVec], w[kVec], m[kVec], v[kVec];
  load8<Gr>(static_cast<const Gr*>(e.g) + i0, valid, vec, g);
  if (e.w != nullptr) load8<float>(e.w + i0, valid, vec, w);
  else load8<P>(static_cast<const P*>(e.p) + i0, valid, vec, w);
  const long block = i0 / 128;
  if constexpr (EIGHT) {
    const float sm = valid > 0 ? fp8::scale_of(e.ms[block]) : 0.f, sv = valid > 0 ? fp8::scale_of(e.vs[block]) : 0.f;
    load_codes(static_cast<const uint8_t*>(e.m) + i0, sm, valid, vec, m);
    load_codes(static_cast<const uint8_t*>(e.v) + i0, sv, valid, vec, v);
#pragma unroll
    for (int i = 0; i < kVec; ++i) v[i] *= v[i];
  } else {
    load8<float>(static_cast<const float*>(e.m) + i0, valid, vec, m);
    load8<float>(static_cast<const float*>(e.v) + i0, valid, vec, v);
  }
  float bad = 0.f, r[kVec];                      // 0 g adds nothing unless g is not finite
  const float keep = 1.f - a.lr * a.wd, rate = a.lr / a.c1, inv_c2 = 1.f / a.c2;
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const float gi = __fmul_rn(g[i], a.grad_scale);
    bad = __fmaf_rn(gi, 0.f, bad);
    if constexpr (EIGHT) {
      // Each operation rounded by itself, as on the CPU: a last bit decides between two codes, 2^-3 apart, so only the
      // same last bits make the same codes (0.494 B elements: 2.03 ms; 1.90 with fused additions and the short root).
      m[i] = __fadd_rn(m[i], __fmul_rn(__fsub_rn(gi, m[i]), a.one_minus_beta1));
      v[i] = __fadd_rn(__fmul_rn(v[i], a.beta2), __fmul_rn(__fmul_rn(a.one_minus_beta2, gi), gi));
      r[i] = __fsqrt_rn(v[i]);
    } else {
      // The root only divides the update, whose error of 2^-21 is below the weight's last bit (2.07 ms; 2.11 with the
      // exact root and separate additions, 2.16 with an exact division too).
      m[i] += (gi - m[i]) * a.one_minus_beta1;
      v[i] = v[i] * a.beta2 + a.one_minus_beta2 * gi * gi;
      r[i] = root(v[i]);
    }
    w[i] = w[i] * keep - rate * __fdividef(m[i], r[i] * inv_c2 + a.eps);
  }
  if constexpr (EIGHT) {
    uint32_t um[kVec], uv[kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const uint32_t u = mix32(static_cast<uint32_t>(i0 + i) * 0x9E3779B1u + key);
      um[i] = (u << 4) & 0xFFFF0u;               // in place below the kept fraction bits
      uv[i] = (u >> 12) & 0xFFFF0u;
    }
    const int bm = store_codes<false>(static_cast<uint8_t*>(e.m) + i0, m, um, valid, vec);
    const int bv = store_codes<true>(static_cast<uint8_t*>(e.v) + i0, r, uv, valid, vec);
    if (threadIdx.x % 16 == 0 && valid > 0) {
      e.ms[block] = static_cast<uint8_t>(bm);
      e.vs[block] = static_cast<uint8_t>(bv);
    }
  } else {
    store8<float>(static_cast<float*>(e.m) + i0, valid, vec, m);
    store8<float>(static_cast<float*>(e.v) + i0, valid, vec, v);
  }
  if (e.w != nullptr) store8<float>(e.w + i0, valid, vec, w);
  store8<P>(static_cast<P*>(e.p) + i0, valid, vec, w);
  if (bad != 0.f && a.nonfinite != nullptr) atomicOr(a.nonfinite, 1);
}

template <typename P, typename Gr>
static void launch_many(const Table& t, const StepArgs& a, bool eight, cudaStream_t st) {
  const unsigned blocks = t.end[t.count - 1];
  if (eight) adamw_many_kernel<P, Gr, true><<<blocks, kThreads, 0, st>>>(t, a);
  else adamw_many_kernel<P, Gr, false><<<blocks, kThreads, 0, st>>>(t, a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

template <typename P>
static void launch_types(at::ScalarType g, const Table& t, const StepArgs& a, bool eight, cudaStream_t st) {
  if (g == at::kFloat) launch_many<P, float>(t, a, eight, st);
  else if (g == at::kBFloat16) launch_many<P, __nv_bfloat16>(t, a, eight, st);
  else launch_many<P, __half>(t, a, eight, st);
}

// The tensors of an optimizer, checked once; kept by its Python object.  w, ms
// and vs may be empty.  Addresses are read from the tensors at every step.
struct Many {
  std::vector<at::Tensor> p, w, m, ms, v, vs;
  c10::Device dev;
};

std::shared_ptr<Many> adamw_many_plan(std::vector<at::Tensor> p, std::vector<at::Tensor> w, std::vector<at::Tensor> m,
                                      std::vector<at::Tensor> ms, std::vector<at::Tensor> v,
                                      std::vector<at::Tensor> vs) {
  const c10::Device dev = p.at(0).device();
  return std::make_shared<Many>(
      Many{std::move(p), std::move(w), std::move(m), std::move(ms), std::move(v), std::move(vs), dev});
}

static bool is_float(at::ScalarType x) { return x == at::kFloat || x == at::kBFloat16 || x == at::kHalf; }

// What a step refuses of its gradients, and of the tensors as they are by now.
void adamw_many_check(const Many& t, const std::vector<at::Tensor>& g) {
  TORCH_CHECK_VALUE(g.size() == t.p.size(), "AdamWMany: ", g.size(), " gradients for ", t.p.size(), " parameters");
  const auto dev = t.dev;
  const bool eight = !t.ms.empty();
  for (size_t i = 0; i < g.size(); ++i) {
    const long n = t.p[i].numel();
    TORCH_CHECK_VALUE(is_float(g[i].scalar_type()) && g[i].numel() == n && g[i].is_contiguous() && g[i].device() == dev,
                      "AdamWMany: gradient ", i, ": contiguous, ", n, " elements, fp32 / bf16 / fp16, on ", dev);
    // a tensor can be given other memory (.data, resize_) of any type after the check at construction
    auto still = [&](const at::Tensor& x, at::ScalarType type, long size) {
      return x.scalar_type() == type && x.numel() == size && x.is_contiguous() && x.device() == dev;
    };
    const auto moment = eight ? at::kFloat8_e4m3fn : at::kFloat;
    TORCH_CHECK_VALUE(is_float(t.p[i].scalar_type()) && still(t.p[i], t.p[i].scalar_type(), n) && still(t.m[i], moment, n) &&
                          still(t.v[i], moment, n) && (t.w.empty() || still(t.w[i], at::kFloat, n)) &&
                          (!eight || (still(t.ms[i], at::kFloat8_e8m0fnu, (n + 127) / 128) &&
                                      still(t.vs[i], at::kFloat8_e8m0fnu, (n + 127) / 128))),
                      "AdamWMany: tensor ", i, " has changed its type, size or place");
  }
}

void adamw_many(const Many& t, const std::vector<at::Tensor>& g, double lr, double beta1, double beta2, double eps,
                double wd, int64_t step, double grad_scale, int64_t seed, const c10::optional<at::Tensor>& step_dev,
                const c10::optional<at::Tensor>& skip, const c10::optional<at::Tensor>& nonfinite) {
  adamw_many_check(t, g);
  if (g.empty()) return;
  const auto dev = t.dev;
  const bool eight = !t.ms.empty();
  const std::pair<const char*, const c10::optional<at::Tensor>*> words[] = {
      {"step_dev", &step_dev}, {"skip", &skip}, {"nonfinite", &nonfinite}};
  for (const auto& [name, x] : words)
    TORCH_CHECK_VALUE(!x->has_value() || ((*x)->scalar_type() == at::kInt && (*x)->is_contiguous() && (*x)->device() == dev &&
                                          (*x)->numel() >= (x == &step_dev ? 4 : 1)),
                      "AdamWMany: ", name, ": int32 on ", dev);
  // one CTA writes the flag while others have yet to read these words
  if (nonfinite.has_value())
    for (const auto* x : {&skip, &step_dev})
      TORCH_CHECK_VALUE(!x->has_value() || nonfinite->data_ptr<int>() < (*x)->data_ptr<int>() ||
                            nonfinite->data_ptr<int>() >= (*x)->data_ptr<int>() + (x == &step_dev ? 4 : 1),
                        "AdamWMany: nonfinite is a word that the step reads");
  // As any write in place: autograd notices.  Before the first launch: a tensor made in inference mode refuses it.
  for (const auto& x : t.p) x.unsafeGetTensorImpl()->bump_version();
  const at::cuda::CUDAGuard guard(dev);
  StepArgs a;
  a.lr = static_cast<float>(lr);
  a.beta2 = static_cast<float>(beta2);
  a.one_minus_beta1 = static_cast<float>(1.0 - beta1);
  a.one_minus_beta2 = static_cast<float>(1.0 - beta2);
  a.eps = static_cast<float>(eps);
  a.wd = static_cast<float>(wd);
  a.c1 = static_cast<float>(1.0 - std::pow(beta1, static_cast<double>(step)));
  a.c2 = static_cast<float>(std::sqrt(1.0 - std::pow(beta2, static_cast<double>(step))));
  a.grad_scale = static_cast<float>(grad_scale);
  a.seed = static_cast<uint32_t>(seed);
  a.sdev = step_dev.has_value() ? step_dev->data_ptr<int>() : nullptr;
  a.skip = skip.has_value() ? skip->data_ptr<int>() : nullptr;
  a.nonfinite = nonfinite.has_value() ? nonfinite->data_ptr<int>() : nullptr;
  auto st = at::cuda::getCurrentCUDAStream();
  // one table after another for each pair of parameter and gradient types that occurs
  std::vector<std::pair<at::ScalarType, at::ScalarType>> kinds;
  for (size_t i = 0; i < g.size(); ++i) {
    const auto k = std::make_pair(t.p[i].scalar_type(), g[i].scalar_type());
    if (std::find(kinds.begin(), kinds.end(), k) == kinds.end()) kinds.push_back(k);
  }
  Table tab;
  for (const auto& [pt, gt] : kinds) {
    tab.count = 0;
    uint64_t chunks = 0;
    auto flush = [&] {
      if (tab.count == 0) return;
      if (pt == at::kFloat) launch_types<float>(gt, tab, a, eight, st);
      else if (pt == at::kBFloat16) launch_types<__nv_bfloat16>(gt, tab, a, eight, st);
      else launch_types<__half>(gt, tab, a, eight, st);
      tab.count = 0;
      chunks = 0;
    };
    for (size_t i = 0; i < g.size(); ++i) {
      const long n = t.p[i].numel();
      if (n == 0 || t.p[i].scalar_type() != pt || g[i].scalar_type() != gt) continue;
      const uint64_t add = (static_cast<uint64_t>(n) + kChunk - 1) / kChunk;
      TORCH_CHECK(add < (1ull << 31), "AdamWMany: a tensor is too long");
      if (tab.count == kMaxTensors || chunks + add >= (1ull << 31)) flush();
      Entry& e = tab.e[tab.count];
      e.p = t.p[i].data_ptr();
      e.w = t.w.empty() ? nullptr : t.w[i].data_ptr<float>();
      e.g = g[i].data_ptr();
      e.m = t.m[i].data_ptr();
      e.v = t.v[i].data_ptr();
      e.ms = eight ? static_cast<uint8_t*>(t.ms[i].data_ptr()) : nullptr;
      e.vs = eight ? static_cast<uint8_t*>(t.vs[i].data_ptr()) : nullptr;
      e.n = n;
      const uintptr_t all = reinterpret_cast<uintptr_t>(e.p) | reinterpret_cast<uintptr_t>(e.w) |
                            reinterpret_cast<uintptr_t>(e.g) | reinterpret_cast<uintptr_t>(e.m) |
                            reinterpret_cast<uintptr_t>(e.v);
      chunks += add;
      tab.end[tab.count] = static_cast<uint32_t>(chunks);
      tab.number[tab.count] = static_cast<uint16_t>((i & 0x7FFF) | ((all & 15) == 0 ? 0x8000 : 0));
      ++tab.count;
    }
    flush();
  }
}

}  // namespace adam
}  // namespace sb

// called by bindings.cpp, which has no other reason to know the plan's type
void bind_adamw_many(pybind11::module& m) {
  namespace py = pybind11;
  py::class_<sb::adam::Many, std::shared_ptr<sb::adam::Many>>(m, "AdamWManyPlan");
  m.def("adamw_many_plan", &sb::adam::adamw_many_plan);
  m.def("adamw_many_check", &sb::adam::adamw_many_check);
  m.def("adamw_many", &sb::adam::adamw_many, "AdamW over many tensors, moments in fp32 or 8 bits");
}

// Block quantiser: bf16 / fp16 / fp32 matrices to 8-bit floating point with a
// power-of-two scale per 128 columns of a row, optionally together with the
// transposed copy (scales per 128 rows of a column), or with one scale per
// 128 x 128 tile shared by both orientations (weights).
//
// Bound: DRAM.  It reads each value once and writes one byte per orientation;
// a CTA owns one 128 x 128 tile, holds it in registers, and finds the row and
// column maxima there, so the second orientation costs no second read.
// 16384 x 1024 bf16: 14 us for one orientation (3.5 TB/s), 18.4 us for both
// (3.7 TB/s); what is left is waiting, 24 warps fit an SM.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp16.h>

#include "fp8.cuh"

namespace sb {
namespace fp8 {

constexpr int kQThreads = 256;

// Sixteen consecutive values of a row in 32-bit words as loaded: pairs of
// 2-byte values, or single fp32 values.
template <typename T>
struct alignas(16) Row16 {
  static constexpr int kWords = 4 * sizeof(T);
  uint32_t w[kWords];
};

SB_DEVICE float value(const Row16<float>& r, int j) { return __uint_as_float(r.w[j]); }
SB_DEVICE float value(const Row16<__nv_bfloat16>& r, int j) {
  return __uint_as_float(j % 2 ? r.w[j / 2] & 0xFFFF0000u : r.w[j / 2] << 16);
}
SB_DEVICE float value(const Row16<__half>& r, int j) {
  const __half2 h = *reinterpret_cast<const __half2*>(&r.w[j / 2]);
  return j % 2 ? __high2float(h) : __low2float(h);
}
// Magnitudes of a word's values, and the larger ones of two words: both values
// of a pair at once.  NaN loses against a number.
template <typename T>
SB_DEVICE uint32_t magnitude(uint32_t w) { return w & (sizeof(T) == 4 ? 0x7FFFFFFFu : 0x7FFF7FFFu); }
template <typename T>
SB_DEVICE uint32_t larger(uint32_t a, uint32_t b);
template <>
SB_DEVICE uint32_t larger<float>(uint32_t a, uint32_t b) {
  return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
}
template <>
SB_DEVICE uint32_t larger<__nv_bfloat16>(uint32_t a, uint32_t b) {
  const __nv_bfloat162 m = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}
template <>
SB_DEVICE uint32_t larger<__half>(uint32_t a, uint32_t b) {
  const __half2 m = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}
// Value `hi` of a word of magnitudes.
template <typename T>
SB_DEVICE float part(uint32_t w, int hi) {
  Row16<T> r;
  r.w[0] = w;
  return value(r, sizeof(T) == 4 ? 0 : hi);
}

SB_DEVICE float as_float(float x) { return x; }
SB_DEVICE float as_float(__half x) { return __half2float(x); }
SB_DEVICE float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }

struct QuantArgs {
  const void* x;
  uint8_t *q, *s, *qt, *st;
  long ld, gstride;        // input strides, elements
  int rows, cols;          // of one group
  int groups;
  int rb, cb;              // tiles per group
  long ldq, ldqt;          // output row strides
  long all_rows, all_cols; // groups * rows, groups * cols: rows of the scale planes
  bool vec;                // 16-byte loads are aligned
};

// Thread (rg, cg): rows 4 rg .. +4, columns 16 cg .. +16 of the tile, so 8 lanes
// hold a row, a thread stores 16 codes of a row at once, and four rows of a
// column are one word of the transposed tile.  Maxima are taken on pairs as
// they were loaded.  (8 columns by 8 rows a thread, in fp32, issued 17 and 24
// instructions a value for one and two orientations: 22.5 and 27.6 us for
// 16384 x 1024.)
template <typename T, int FMT, bool TILES, bool BOTH>
__global__ void __launch_bounds__(kQThreads, BOTH && sizeof(T) == 2 ? 3 : 1)
quantize_kernel(const QuantArgs a) {
  using R = Row16<T>;
  constexpr int kWords = R::kWords, kPer = 16 / kWords;   // values of a word
  constexpr bool kCols = BOTH && !TILES;
  __shared__ uint32_t s_max[8][8 * kWords];               // [warp][column group, word]: largest of a warp's 16 rows
  __shared__ float s_inv[128];
  __shared__ alignas(16) uint32_t s_t[BOTH ? 128 * 32 : 4];
  const int cg = threadIdx.x % 8, rg = threadIdx.x / 8;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const unsigned per = static_cast<unsigned>(a.rb) * a.cb;
  const int g = a.groups == 1 ? 0 : static_cast<int>(blockIdx.x / per);
  const unsigned tile = blockIdx.x - g * per;
  const int tr = tile / static_cast<unsigned>(a.cb), tc = tile - tr * a.cb;
  const int r0 = tr * 128 + rg * 4, c0 = tc * 128 + cg * 16;
  const T* x = reinterpret_cast<const T*>(a.x) + g * a.gstride + static_cast<long>(r0) * a.ld + c0;

  R v[4];
  if (a.vec && c0 + 16 <= a.cols && r0 + 4 <= a.rows) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int q = 0; q < kWords / 4; ++q)
        reinterpret_cast<uint4*>(v[i].w)[q] = __ldg(reinterpret_cast<const uint4*>(x + i * a.ld) + q);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int q = 0; q < kWords; ++q) v[i].w[q] = 0u;
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (r0 + i < a.rows && c0 + j < a.cols) reinterpret_cast<T*>(v[i].w)[j] = x[i * a.ld + j];
    }
  }

  // The largest magnitudes, of the rows and (pairwise) of the columns.  Infinities do not count: a thread that meets
  // one puts zeros in their place and looks again; their codes are set apart, from the input, at the end.
  float rmax[4];
  uint32_t cmax[kWords];
  bool infinite = false;
#pragma unroll 1
  while (true) {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t m = 0u;
#pragma unroll
      for (int q = 0; q < kWords; ++q) {
        const uint32_t w = magnitude<T>(v[i].w[q]);
        m = larger<T>(m, w);
        if (kCols) cmax[q] = i == 0 ? larger<T>(0u, w) : larger<T>(cmax[q], w);
      }
      rmax[i] = fmaxf(part<T>(m, 0), part<T>(m, 1));
      top = fmaxf(top, rmax[i]);
    }
    if (top != INFINITY) break;
    infinite = true;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int q = 0; q < kWords; ++q)
#pragma unroll
        for (int h = 0; h < kPer; ++h)
          if (fabsf(part<T>(v[i].w[q], h)) == INFINITY) v[i].w[q] &= kPer == 1 ? 0u : (h ? 0x0000FFFFu : 0xFFFF0000u);
  }
  // code of an infinity: NaN in e4m3, which has none
  auto infinity_code = [](float f) -> uint8_t { return FMT == kE4M3 ? 0x7F : (f > 0.f ? 0x7C : 0xFC); };

  int rbyte[4];
  float rinv[4];
  if constexpr (TILES) {
    float m = warp_max(fmaxf(fmaxf(rmax[0], rmax[1]), fmaxf(rmax[2], rmax[3])));
    float* s = reinterpret_cast<float*>(&s_max[0][0]);
    if (lane == 0) s[warp] = m;
    __syncthreads();
    m = s[0];
#pragma unroll
    for (int w = 1; w < 8; ++w) m = fmaxf(m, s[w]);
    rbyte[0] = scale_byte(m, FMT);
    rinv[0] = inv_scale(rbyte[0]);
#pragma unroll
    for (int i = 1; i < 4; ++i) rbyte[i] = rbyte[0], rinv[i] = rinv[0];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) rmax[i] = fmaxf(rmax[i], __shfl_xor_sync(0xffffffffu, rmax[i], o));
      rbyte[i] = scale_byte(rmax[i], FMT);
      rinv[i] = inv_scale(rbyte[i]);
    }
  }

  // codes along the rows
  uint8_t* q = a.q + (static_cast<long>(g) * a.rows + r0) * a.ldq + c0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t w[4];
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      float y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = value(v[i], 4 * h + j) * rinv[i];
      w[h] = pack2(y[0], y[1], FMT) | (pack2(y[2], y[3], FMT) << 16);
    }
    if (r0 + i < a.rows && c0 < a.cols) *reinterpret_cast<uint4*>(q + i * a.ldq) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  if (infinite) {
#pragma unroll 1
    for (int e = 0; e < 64; ++e) {
      const int i = e / 16, j = e % 16;
      if (r0 + i >= a.rows || c0 + j >= a.cols) continue;
      const float f = as_float(x[i * a.ld + j]);
      if (fabsf(f) == INFINITY) q[i * a.ldq + j] = infinity_code(f);
    }
  }
  // scale bytes of this tile, and zeros for the columns that the last word lacks: four lanes of a row group, a row each
  if (cg < 4 && r0 + cg < a.rows) {
    const int byte = cg == 0 ? rbyte[0] : cg == 1 ? rbyte[1] : cg == 2 ? rbyte[2] : rbyte[3];
    uint8_t* s = a.s + ((tc / 4) * a.all_rows + static_cast<long>(g) * a.rows + r0 + cg) * 4;
    s[tc % 4] = static_cast<uint8_t>(byte);
    if (tc == a.cb - 1)
      for (int j = tc % 4 + 1; j < 4; ++j) s[j] = 0;
  }

  if constexpr (BOTH) {
    // The values are unpacked anew: kept from above they would fill 64 registers and halve the CTAs of an SM.
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int w = 0; w < kWords; ++w) asm volatile("" : "+r"(v[i].w[w]));
    if constexpr (kCols) {
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        cmax[w] = larger<T>(cmax[w], __shfl_xor_sync(0xffffffffu, cmax[w], 8));
        cmax[w] = larger<T>(cmax[w], __shfl_xor_sync(0xffffffffu, cmax[w], 16));
        if (lane < 8) s_max[warp][cg * kWords + w] = cmax[w];
      }
      __syncthreads();
    }
    if (threadIdx.x < 128) {
      const int c = tc * 128 + threadIdx.x;
      int byte = rbyte[0];
      if constexpr (kCols) {
        uint32_t m = s_max[0][threadIdx.x / kPer];
#pragma unroll
        for (int w = 1; w < 8; ++w) m = larger<T>(m, s_max[w][threadIdx.x / kPer]);
        byte = scale_byte(part<T>(m, threadIdx.x % kPer), FMT);
        s_inv[threadIdx.x] = inv_scale(byte);
      }
      if (c < a.cols) {
        uint8_t* s = a.st + ((tr / 4) * a.all_cols + static_cast<long>(g) * a.cols + c) * 4;
        s[tr % 4] = static_cast<uint8_t>(byte);
        if (tr == a.rb - 1)
          for (int j = tr % 4 + 1; j < 4; ++j) s[j] = 0;
      }
    }
    if constexpr (kCols) __syncthreads();
    // Word rg of column c lies at rg ^ 4 (c / 16): the eight column groups and four row groups of a warp store to 32
    // different banks, and four words that make 16 bytes of a column stay together.
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float inv = kCols ? s_inv[cg * 16 + j] : rinv[0];
      float y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = value(v[i], j) * inv;
      uint32_t w = pack2(y[0], y[1], FMT) | (pack2(y[2], y[3], FMT) << 16);
      s_t[(cg * 16 + j) * 32 + (rg ^ (4 * cg))] = w;
    }
    if (infinite) {
#pragma unroll 1
      for (int e = 0; e < 64; ++e) {
        const int i = e / 16, j = e % 16;
        if (r0 + i >= a.rows || c0 + j >= a.cols) continue;
        const float f = as_float(x[i * a.ld + j]);
        if (fabsf(f) == INFINITY)
          reinterpret_cast<uint8_t*>(&s_t[(cg * 16 + j) * 32 + (rg ^ (4 * cg))])[i] = infinity_code(f);
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int idx = k * kQThreads + threadIdx.x;
      const int c = idx / 8, ch = idx % 8;        // column of the tile, 16-row chunk
      const int col = tc * 128 + c, row = tr * 128 + ch * 16;
      if (col < a.cols && row < a.rows)
        *reinterpret_cast<uint4*>(a.qt + (static_cast<long>(g) * a.cols + col) * a.ldqt + row) =
            *reinterpret_cast<const uint4*>(&s_t[c * 32 + ((4 * ch) ^ (4 * (c / 16)))]);
    }
  }
}

template <typename T, int FMT>
static void launch_quant(const QuantArgs& a, bool tiles, bool both, long blocks, cudaStream_t st) {
  const unsigned n = static_cast<unsigned>(blocks);
  if (tiles && both) quantize_kernel<T, FMT, true, true><<<n, kQThreads, 0, st>>>(a);
  else if (tiles) quantize_kernel<T, FMT, true, false><<<n, kQThreads, 0, st>>>(a);
  else if (both) quantize_kernel<T, FMT, false, true><<<n, kQThreads, 0, st>>>(a);
  else quantize_kernel<T, FMT, false, false><<<n, kQThreads, 0, st>>>(a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// x [rows, cols] or [groups, rows, cols], inner stride 1.  Returns
// (codes, scales) or (codes, scales, codes of the transpose, its scales);
// codes [groups * rows, round_up(cols, 16)], scales [words, rows, 4].
std::vector<at::Tensor> quantize(const at::Tensor& x, int64_t fmt, bool tiles, bool both) {
  TORCH_CHECK(x.is_cuda(), "quantize: CUDA tensor required");
  const at::cuda::CUDAGuard guard(x.device());
  const long groups = x.dim() == 3 ? x.size(0) : 1;
  const long rows = x.size(-2), cols = x.size(-1);
  TORCH_CHECK(rows < (1l << 31) - 128 && cols < (1l << 31) - 512, "quantize: a side is too long");
  TORCH_CHECK(x.stride(-1) == 1 || cols <= 1, "quantize: the inner dimension must be contiguous");
  const auto codes = x.options().dtype(fmt == kE4M3 ? at::kFloat8_e4m3fn : at::kFloat8_e5m2);
  const auto scales = x.options().dtype(at::kFloat8_e8m0fnu);
  const long ldq = (cols + 15) / 16 * 16, ldqt = (rows + 15) / 16 * 16;
  std::vector<at::Tensor> out = {at::empty({groups * rows, ldq}, codes), at::empty({(cols + 511) / 512, groups * rows, 4}, scales)};
  if (both) {
    out.push_back(at::empty({groups * cols, ldqt}, codes));
    out.push_back(at::empty({(rows + 511) / 512, groups * cols, 4}, scales));
  }
  if (x.numel() == 0) return out;
  QuantArgs a;
  a.x = x.data_ptr();
  a.q = static_cast<uint8_t*>(out[0].data_ptr());
  a.s = static_cast<uint8_t*>(out[1].data_ptr());
  a.qt = both ? static_cast<uint8_t*>(out[2].data_ptr()) : nullptr;
  a.st = both ? static_cast<uint8_t*>(out[3].data_ptr()) : nullptr;
  a.ld = x.stride(-2);
  a.gstride = x.dim() == 3 ? x.stride(0) : 0;
  a.groups = static_cast<int>(groups);
  a.rows = static_cast<int>(rows);
  a.cols = static_cast<int>(cols);
  a.rb = static_cast<int>((rows + 127) / 128);
  a.cb = static_cast<int>((cols + 127) / 128);
  a.ldq = ldq;
  a.ldqt = ldqt;
  a.all_rows = groups * rows;
  a.all_cols = groups * cols;
  const long es = x.element_size();
  a.vec = aligned16(a.x) && (a.ld * es) % 16 == 0 && (a.gstride * es) % 16 == 0;
  const long blocks = groups * static_cast<long>(a.rb) * a.cb;
  TORCH_CHECK(blocks < (1l << 31), "quantize: too many blocks");
  auto st = at::cuda::getCurrentCUDAStream();
#define SB_QUANT(T)                                                        \
  do {                                                                     \
    if (fmt == kE4M3) launch_quant<T, kE4M3>(a, tiles, both, blocks, st);  \
    else launch_quant<T, kE5M2>(a, tiles, both, blocks, st);               \
  } while (0)
  if (x.scalar_type() == at::kBFloat16) SB_QUANT(__nv_bfloat16);
  else if (x.scalar_type() == at::kHalf) SB_QUANT(__half);
  else if (x.scalar_type() == at::kFloat) SB_QUANT(float);
  else TORCH_CHECK(false, "quantize: bf16, fp16 or fp32 input required");
#undef SB_QUANT
  return out;
}

}  // namespace fp8
}  // namespace sb

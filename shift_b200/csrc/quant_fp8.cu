// Block quantiser: bf16 / fp16 / fp32 matrices to 8-bit floating point with a
// power-of-two scale per 128 columns of a row, optionally together with the
// transposed copy (scales per 128 rows of a column), or with one scale per
// 128 x 128 tile shared by both orientations (weights).
//
// Bound: DRAM.  It reads each value once and writes one byte per orientation;
// a CTA owns one 128 x 128 tile, holds it in registers, and finds the row and
// column maxima there, so the second orientation costs no second read.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp16.h>

#include "fp8.cuh"

namespace sb {
namespace fp8 {

constexpr int kQThreads = 256;

// Eight consecutive values of a row as loaded (16 bytes, or 32 for fp32).
template <typename T>
struct alignas(16) Vec8 {
  T v[8];
};

template <typename T>
SB_DEVICE float to_f(T x);
template <>
SB_DEVICE float to_f<float>(float x) { return x; }
template <>
SB_DEVICE float to_f<__half>(__half x) { return __half2float(x); }
template <>
SB_DEVICE float to_f<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

SB_DEVICE float finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;      // false for NaN too
}

// The conversion saturates: an infinity becomes NaN in e4m3, which has none, and stays one in e5m2.
template <int FMT>
SB_DEVICE uint32_t patch_infinities(uint32_t w, const float* y) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (isinf(y[j])) w = (w & ~(0xFFu << (8 * j))) | ((FMT == kE4M3 ? 0x7Fu : (y[j] > 0 ? 0x7Cu : 0xFCu)) << (8 * j));
  return w;
}

struct QuantArgs {
  const void* x;
  uint8_t *q, *s, *qt, *st;
  long ld, gstride;        // input strides, elements
  int rows, cols;          // of one group
  int rb, cb;              // tiles per group
  long ldq, ldqt;          // output row strides
  long all_rows, all_cols; // groups * rows, groups * cols: rows of the scale planes
  bool vec;                // 16-byte loads are aligned
};

// thread (rg, cg): rows rg * 8 .. +8, columns cg * 8 .. +8 of the tile, so 16
// lanes read 256 contiguous bytes of a row (2-byte types) and a column's codes
// of 8 rows are one 8-byte word of the transposed tile.
template <typename T, int FMT, bool TILES, bool BOTH>
__global__ void __launch_bounds__(kQThreads)
quantize_kernel(const QuantArgs a) {
  __shared__ float s_max[8][128];
  __shared__ float s_inv[128];
  __shared__ uint64_t s_t[BOTH ? 128 * 16 : 1];
  const int cg = threadIdx.x % 16, rg = threadIdx.x / 16;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const long per = static_cast<long>(a.rb) * a.cb;
  const long g = blockIdx.x / per;
  const int tile = static_cast<int>(blockIdx.x - g * per);
  const int tr = tile / a.cb, tc = tile % a.cb;
  const int r0 = tr * 128 + rg * 8, c0 = tc * 128 + cg * 8;
  const T* x = reinterpret_cast<const T*>(a.x) + g * a.gstride;

  Vec8<T> v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = r0 + i;
    const T* p = x + static_cast<long>(r) * a.ld + c0;
    uint4* dst = reinterpret_cast<uint4*>(&v[i]);
    if (r < a.rows && a.vec && c0 + 8 <= a.cols) {
      const uint4* src = reinterpret_cast<const uint4*>(p);
#pragma unroll
      for (int w = 0; w < static_cast<int>(sizeof(T)) / 2; ++w) dst[w] = __ldg(src + w);
    } else {
#pragma unroll
      for (int w = 0; w < static_cast<int>(sizeof(T)) / 2; ++w) dst[w] = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (r < a.rows && c0 + j < a.cols) v[i].v[j] = p[j];
    }
  }

  // fmaxf passes over NaN; a maximum of infinity sends the thread through its values once more without them
  float rmax[8], cmax[8], top = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) cmax[j] = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    rmax[i] = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float f = fabsf(to_f<T>(v[i].v[j]));
      rmax[i] = fmaxf(rmax[i], f);
      if (BOTH && !TILES) cmax[j] = fmaxf(cmax[j], f);
    }
    top = fmaxf(top, rmax[i]);
  }
  const bool infinite = top == INFINITY;
  if (infinite) {
#pragma unroll
    for (int j = 0; j < 8; ++j) cmax[j] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      rmax[i] = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float f = finite_abs(to_f<T>(v[i].v[j]));
        rmax[i] = fmaxf(rmax[i], f);
        if (BOTH && !TILES) cmax[j] = fmaxf(cmax[j], f);
      }
    }
  }
  float rinv[8];
  int rbyte[8];
  if constexpr (TILES) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, rmax[i]);
    m = warp_max(m);
    if (lane == 0) s_max[0][warp] = m;
    __syncthreads();
    m = s_max[0][0];
#pragma unroll
    for (int w = 1; w < 8; ++w) m = fmaxf(m, s_max[0][w]);
    const int byte = scale_byte(m, FMT);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      rbyte[i] = byte;
      rinv[i] = inv_scale(byte);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) rmax[i] = fmaxf(rmax[i], __shfl_xor_sync(0xffffffffu, rmax[i], o));
      rbyte[i] = scale_byte(rmax[i], FMT);
      rinv[i] = inv_scale(rbyte[i]);
    }
  }

  // codes along the rows
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = r0 + i;
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = to_f<T>(v[i].v[4 * h + j]) * rinv[i];
      w[h] = pack2(y[0], y[1], FMT) | (pack2(y[2], y[3], FMT) << 16);
      if (infinite) w[h] = patch_infinities<FMT>(w[h], y);
    }
    if (r < a.rows && c0 < a.cols)
      *reinterpret_cast<uint2*>(a.q + (g * a.rows + r) * a.ldq + c0) = make_uint2(w[0], w[1]);
    // scale bytes of this tile, and zeros for the columns that the last word lacks
    if (cg == 0 && r < a.rows) {
      uint8_t* s = a.s + ((tc / 4) * a.all_rows + g * a.rows + r) * 4;
      s[tc % 4] = static_cast<uint8_t>(rbyte[i]);
      if (tc == a.cb - 1)
        for (int j = tc % 4 + 1; j < 4; ++j) s[j] = 0;
    }
  }
  if constexpr (BOTH) {
    float cinv[8];
    if constexpr (TILES) {
#pragma unroll
      for (int j = 0; j < 8; ++j) cinv[j] = rinv[0];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        cmax[j] = fmaxf(cmax[j], __shfl_xor_sync(0xffffffffu, cmax[j], 16));
        if (lane < 16) s_max[warp][cg * 8 + j] = cmax[j];
      }
      __syncthreads();
    }
    if (threadIdx.x < 128) {
      const int c = tc * 128 + threadIdx.x;
      int byte = rbyte[0];
      if constexpr (!TILES) {
        float m = s_max[0][threadIdx.x];
#pragma unroll
        for (int w = 1; w < 8; ++w) m = fmaxf(m, s_max[w][threadIdx.x]);
        byte = scale_byte(m, FMT);
        s_inv[threadIdx.x] = inv_scale(byte);
      }
      if (c < a.cols) {
        uint8_t* s = a.st + ((tr / 4) * a.all_cols + g * a.cols + c) * 4;
        s[tr % 4] = static_cast<uint8_t>(byte);
        if (tr == a.rb - 1)
          for (int j = tr % 4 + 1; j < 4; ++j) s[j] = 0;
      }
    }
    if constexpr (!TILES) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; ++j) cinv[j] = s_inv[cg * 8 + j];
    }
    // 8 rows of a column are one 8-byte word; words are swizzled by the column
    // group so that the 16 lanes of a row group write 16 different banks pairs
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      uint32_t w[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = to_f<T>(v[4 * h + i].v[j]) * cinv[j];
        w[h] = pack2(y[0], y[1], FMT) | (pack2(y[2], y[3], FMT) << 16);
        if (infinite) w[h] = patch_infinities<FMT>(w[h], y);
      }
      s_t[(cg * 8 + j) * 16 + (rg ^ cg)] = static_cast<uint64_t>(w[1]) << 32 | w[0];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int idx = k * kQThreads + threadIdx.x;
      const int c = idx / 8, ch = idx % 8;        // column of the tile, 16-row chunk
      const int col = tc * 128 + c, row = tr * 128 + ch * 16;
      if (col < a.cols && row < a.rows) {
        const uint64_t lo = s_t[c * 16 + ((2 * ch) ^ (c / 8))], hi = s_t[c * 16 + ((2 * ch + 1) ^ (c / 8))];
        *reinterpret_cast<ulonglong2*>(a.qt + (g * a.cols + col) * a.ldqt + row) = make_ulonglong2(lo, hi);
      }
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

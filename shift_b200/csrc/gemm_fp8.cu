// Products of 8-bit matrices with a power-of-two scale per block of 128.
//
//   D[m, n] (+)= sum_b 2^(ea[m, b] + eb[n, b]) sum_{k in block b} A[m, k] B[n, k]
//
// Both operands have the contraction inside (K-major), see fp8.cuh for their
// layout.  Row groups: A and D rows are cut into segments by offs[0..G], group
// g multiplies with B rows [g N, (g + 1) N).  K groups: the contraction is cut
// into segments that start on a block, group g writes D rows [g M, (g + 1) M).
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "fp8.cuh"

namespace sb {
namespace fp8 {

enum Mode : int { kRowGroups = 0, kKGroups = 1 };

struct Args {
  const uint8_t *a, *b;
  const uint8_t *sa, *sb;
  long lda, ldb;
  long rows_a, rows_b;     // rows of the scale planes
  int M, N, K, G, mode;
  const int* offs;
  void* D;
  long ldd;
  bool f32, acc, a_e5m2, b_e5m2;
  int* status;
};

SB_DEVICE float decode8(uint8_t c, bool e5m2) {
  const __half_raw h = __nv_cvt_fp8_to_halfraw(c, e5m2 ? __NV_E5M2 : __NV_E4M3);
  return __half2float(__half(h));
}

// One CTA per 64 x 64 tile of one group, blocks of 32 along K in fp32.
__global__ void __launch_bounds__(256) matmul_kernel(const Args p) {
  __shared__ float sA[32][65], sB[32][65];
  const int tiles_n = (p.N + 63) / 64;
  int g = blockIdx.y;
  int lo = 0, hi = p.mode == kRowGroups ? p.M : p.K;
  if (p.offs != nullptr) {
    const int lim = hi;
    lo = min(max(p.offs[g], 0), lim);
    hi = min(max(p.offs[g + 1], lo), lim);
    if (p.mode == kKGroups && lo % 128 != 0 && hi > lo) {
      if (threadIdx.x == 0) record_status(p.status, kBadShape);
      return;
    }
  }
  const int tm = blockIdx.x / tiles_n, tn = blockIdx.x % tiles_n;
  const int m_end = p.mode == kRowGroups ? hi : p.M;
  const int m0 = (p.mode == kRowGroups ? lo : 0) + tm * 64, n0 = tn * 64;
  if (m0 >= m_end) return;
  const int k_lo = p.mode == kRowGroups ? 0 : lo, k_hi = p.mode == kRowGroups ? p.K : hi;
  const long b_row0 = p.mode == kRowGroups ? static_cast<long>(g) * p.N : 0;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  float acc[4][4] = {};
  for (int k0 = k_lo; k0 < k_hi; k0 += 32) {
    for (int i = threadIdx.x; i < 64 * 32; i += 256) {
      const int r = i / 32, k = k0 + i % 32;
      float fa = 0.f, fb = 0.f;
      if (m0 + r < m_end && k < k_hi)
        fa = decode8(p.a[static_cast<long>(m0 + r) * p.lda + k], p.a_e5m2) *
             scale_of(p.sa[((k / 512) * p.rows_a + m0 + r) * 4 + k / 128 % 4]);
      if (n0 + r < p.N && k < k_hi)
        fb = decode8(p.b[(b_row0 + n0 + r) * p.ldb + k], p.b_e5m2) *
             scale_of(p.sb[((k / 512) * p.rows_b + b_row0 + n0 + r) * 4 + k / 128 % 4]);
      sA[i % 32][r] = fa;
      sB[i % 32][r] = fb;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 32; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += sA[k][ty + 16 * i] * sB[k][tx + 16 * j];
    __syncthreads();
  }
  const long d_row0 = p.mode == kRowGroups ? 0 : static_cast<long>(g) * p.M;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = m0 + ty + 16 * i;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + tx + 16 * j;
      if (m >= m_end || n >= p.N) continue;
      const long at = (d_row0 + m) * p.ldd + n;
      if (p.f32) {
        float* d = static_cast<float*>(p.D) + at;
        *d = p.acc ? *d + acc[i][j] : acc[i][j];
      } else {
        __nv_bfloat16* d = static_cast<__nv_bfloat16*>(p.D) + at;
        *d = __float2bfloat16(p.acc ? __bfloat162float(*d) + acc[i][j] : acc[i][j]);
      }
    }
  }
}

// a, b: codes [rows, ld] with scales [words, rows, 4]; D [rows, N] (row mode)
// or [G * M, N] (K mode), bf16 or fp32, inner stride 1.
void matmul(const at::Tensor& a, const at::Tensor& sa, const at::Tensor& b, const at::Tensor& sb, at::Tensor& D,
            const c10::optional<at::Tensor>& offs, int64_t M, int64_t N, int64_t K, int64_t G, int64_t mode,
            bool accumulate, const at::Tensor& status) {
  const at::cuda::CUDAGuard guard(a.device());
  if (M == 0 || N == 0 || G == 0) return;
  Args p;
  p.a = static_cast<const uint8_t*>(a.data_ptr());
  p.b = static_cast<const uint8_t*>(b.data_ptr());
  p.sa = static_cast<const uint8_t*>(sa.data_ptr());
  p.sb = static_cast<const uint8_t*>(sb.data_ptr());
  p.lda = a.stride(0);
  p.ldb = b.stride(0);
  p.rows_a = a.size(0);
  p.rows_b = b.size(0);
  p.M = static_cast<int>(M);
  p.N = static_cast<int>(N);
  p.K = static_cast<int>(K);
  p.G = static_cast<int>(G);
  p.mode = static_cast<int>(mode);
  p.offs = offs.has_value() ? offs->data_ptr<int>() : nullptr;
  p.D = D.data_ptr();
  p.ldd = D.stride(0);
  p.f32 = D.scalar_type() == at::kFloat;
  p.acc = accumulate;
  p.a_e5m2 = a.scalar_type() == at::kFloat8_e5m2;
  p.b_e5m2 = b.scalar_type() == at::kFloat8_e5m2;
  p.status = status.data_ptr<int>();
  const dim3 grid(static_cast<unsigned>(((M + 63) / 64) * ((N + 63) / 64)), static_cast<unsigned>(G));
  matmul_kernel<<<grid, 256, 0, at::cuda::getCurrentCUDAStream()>>>(p);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace fp8
}  // namespace sb

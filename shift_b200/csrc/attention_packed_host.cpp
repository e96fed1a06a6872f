// Causal attention over packed sequences: arguments, workspaces and launches.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>

#include <cmath>
#include <mutex>

#include "apart.h"
#include "attention_packed.h"

namespace sb {
namespace pa {

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
    TORCH_CHECK(e == cudaSuccess && q == cudaDriverEntryPointSuccess && ptr, "cannot resolve cuTensorMapEncodeTiled");
    fn = reinterpret_cast<EncodeFn>(ptr);
  });
  return fn;
}

static int64_t row_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

// boxes of `rows` rows of 64 columns, 128-byte swizzle; rows behind the last one read as zeros
static CUtensorMap tile_map(const at::Tensor& t, int rows) {
  CUtensorMap m;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(t.size(1)), static_cast<cuuint64_t>(t.size(0))};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(row_stride(t) * 2)};
  cuuint32_t box[2] = {64, static_cast<cuuint32_t>(rows)};
  cuuint32_t es[2] = {1, 1};
  const CUresult r = encode_fn()(
      &m, t.scalar_type() == at::kHalf ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
      t.data_ptr(), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "packed attention: cuTensorMapEncodeTiled failed with code ", static_cast<int>(r));
  return m;
}

static void check_rows(const at::Tensor& t, const at::Tensor& qkv, int64_t rows, int64_t cols, const char* who,
                       const char* what) {
  TORCH_CHECK(t.is_cuda() && t.device() == qkv.device() && t.scalar_type() == qkv.scalar_type(), who, ": ", what,
              " is ", t.scalar_type(), " on ", t.device(), ", qkv ", qkv.scalar_type(), " on ", qkv.device());
  TORCH_CHECK(t.dim() == 2 && t.size(0) == rows && t.size(1) == cols, who, ": ", what, " [", rows, ", ", cols,
              "] is expected");
  TORCH_CHECK(t.stride(1) == 1 && (rows <= 1 || (t.stride(0) >= cols && t.stride(0) % 8 == 0)) &&
                  reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0,
              who, ": ", what, " of inner stride 1 in rows that do not overlap, start on 16 bytes and lie a multiple of 16 "
              "bytes apart");
}

struct Plan {                        // of packed.cu's sequences()
  const int *start, *stop, *ends, *q_order, *q2_order, *k_order;
};

static Args base_args(const at::Tensor& qkv, const at::Tensor& plan, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                      double scale, const at::Tensor& status, const char* who, Plan& pl) {
  TORCH_CHECK(qkv.scalar_type() == at::kBFloat16 || qkv.scalar_type() == at::kHalf, who, ": bf16 or fp16, got ",
              qkv.scalar_type());
  TORCH_CHECK(D == 64 || D == 128, who, ": heads of 64 or 128 columns, got ", D);
  TORCH_CHECK(Hq >= 1 && Hkv >= 1 && Hq % Hkv == 0 && Hq <= (1 << 20), who, ": ", Hq, " query heads for ", Hkv,
              " key heads");
  TORCH_CHECK(std::isfinite(scale) && scale > 0, who, ": scale ", scale, ", a number above 0 is expected");
  const int64_t nt = (T + 127) / 128, nt2 = (T + 255) / 256;
  check_rows(qkv, qkv, T, (Hq + 2 * Hkv) * D, who, "qkv");
  TORCH_CHECK(plan.scalar_type() == at::kInt && plan.is_contiguous() && plan.numel() == 3 * T + 2 + 2 * nt + nt2 &&
                  plan.device() == qkv.device(),
              who, ": the plan of another buffer, or on another device (ops.packed.sequences of ", T, " rows beside qkv)");
  const int* p = plan.data_ptr<int>();
  const int* o = p + 3 * T + 2;
  pl = Plan{p, p + 2 * T, p + 3 * T, o, o + nt, o + nt + nt2};
  TORCH_CHECK(nt * Hq <= (1L << 28), who, ": too many rows and heads");
  Args a{};
  a.T = static_cast<int>(T);
  a.Hq = static_cast<int>(Hq);
  a.Hkv = static_cast<int>(Hkv);
  a.group = static_cast<int>(Hq / Hkv);
  a.split = 1;
  a.tiles = static_cast<int>(nt);
  a.start = pl.start;
  a.stop = pl.stop;
  a.ends = pl.ends;
  a.scale = static_cast<float>(scale);
  a.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  a.qkv = qkv.data_ptr();
  a.ld = row_stride(qkv);
  a.status = status.data_ptr<int>();
  return a;
}

std::vector<at::Tensor> fwd(const at::Tensor& qkv, const at::Tensor& plan, int64_t rows, int64_t Hq, int64_t Hkv,
                            int64_t D, double scale, const c10::optional<at::Tensor>& out, const at::Tensor& status) {
  const char* who = "attention_fwd";
  Plan pl;
  Args a = base_args(qkv, plan, rows, Hq, Hkv, D, scale, status, who, pl);
  const at::cuda::CUDAGuard guard(qkv.device());
  auto o = out.has_value() ? *out : at::empty({a.T, Hq * D}, qkv.options());
  if (out.has_value()) {
    check_rows(o, qkv, a.T, Hq * D, who, "out");
    TORCH_CHECK(!share_memory(o, qkv), who, ": out overlaps qkv");
  }
  auto lse = at::empty({Hq, a.T}, qkv.options().dtype(at::kFloat));
  if (a.T == 0) return {o, lse};
  a.fill = out.has_value() ? 0 : 1;
  a.o = o.data_ptr();
  a.o_ld = row_stride(o);
  a.lse = lse.data_ptr<float>();
  // Two heads of one key head share every key block and have the same causal cost; without such pairs two consecutive
  // tiles of a head do.
  a.pair_heads = a.group % 2 == 0;
  // With at most two tiles an SM an item is one tile, whose key blocks the two groups share (one sequence, 16 / 4 heads of
  // 64: 512 rows 16.4 -> 14.3 us, 1024 22.5 -> 18.4, 2048 36.9 -> 34.8).  Not for heads of 128, where a block is then loaded
  // for one tile in as long as it takes for two, and shared memory has no stages left to hide it (2048 rows 41 -> 57 us).
  a.split_keys = D == 64 && a.tiles * Hq <= 2 * at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  a.order = a.split_keys || a.pair_heads ? pl.q_order : pl.q2_order;
  const unsigned items = static_cast<unsigned>(a.split_keys     ? a.tiles * Hq
                                               : a.pair_heads ? a.tiles * (Hq / 2)
                                                              : (a.T + 255) / 256 * Hq);
  const auto later = c10::cuda::CUDACachingAllocator::get()->allocate(items * 8 * sizeof(int2));
  a.later = static_cast<int2*>(later.get());
  const CUtensorMap tm = tile_map(qkv, 128);
  const bool half = qkv.scalar_type() == at::kHalf;
  launch_fwd(static_cast<int>(D), half, tm, a, items, at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {o, lse};
}

at::Tensor bwd(const at::Tensor& qkv, const at::Tensor& o, const at::Tensor& lse, const at::Tensor& dout,
               const at::Tensor& plan, int64_t rows, int64_t Hq, int64_t Hkv, int64_t D, double scale,
               const c10::optional<at::Tensor>& out, const at::Tensor& status) {
  const char* who = "attention_bwd";
  Plan pl;
  Args a = base_args(qkv, plan, rows, Hq, Hkv, D, scale, status, who, pl);
  check_rows(o, qkv, a.T, Hq * D, who, "o");
  check_rows(dout, qkv, a.T, Hq * D, who, "do");
  TORCH_CHECK(lse.scalar_type() == at::kFloat && lse.is_contiguous() && lse.device() == qkv.device() && lse.dim() == 2 &&
                  lse.size(0) == Hq && lse.size(1) == a.T,
              who, ": lse [", Hq, ", ", a.T, "] fp32, contiguous, beside qkv");
  const at::cuda::CUDAGuard guard(qkv.device());
  auto dqkv = out.has_value() ? *out : at::empty({a.T, (Hq + 2 * Hkv) * D}, qkv.options());
  if (out.has_value()) {
    check_rows(dqkv, qkv, a.T, (Hq + 2 * Hkv) * D, who, "out");
    TORCH_CHECK(!share_memory(dqkv, qkv) && !share_memory(dqkv, o) && !share_memory(dqkv, dout), who,
                ": out overlaps qkv, o or do");
  }
  if (a.T == 0) return dqkv;
  a.fill = out.has_value() ? 0 : 1;
  a.o = o.data_ptr();
  a.o_ld = row_stride(o);
  a.lse = lse.data_ptr<float>();
  a.dout = dout.data_ptr();
  a.do_ld = row_stride(dout);
  a.dqkv = dqkv.data_ptr();
  a.dqkv_ld = row_stride(dqkv);
  auto row_values = at::empty({Hq * a.tiles * (256 + 16)}, lse.options());     // behind them [tiles * Hq][8] pairs of ints
  a.later = reinterpret_cast<int2*>(row_values.data_ptr<float>() + Hq * a.tiles * 256);
  at::Tensor scales;
  if (qkv.scalar_type() == at::kHalf) {              // fp16 holds dS over some 2^30: rows and keys scale it by powers of two
    TORCH_CHECK(Hkv <= 65535, who, ": at most 65535 key heads in fp16, got ", Hkv);
    scales = at::empty({(Hq + Hkv) * a.tiles * 128}, lse.options());
    a.tops = scales.data_ptr<float>();
    a.shifts = reinterpret_cast<int*>(a.tops + Hq * a.tiles * 128);
  }
  // A key tile meets every later query of its sequence in every head of its group: with few tiles the group's heads are
  // dealt out over several CTAs, whose fp32 sums are added up in order afterwards.
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  at::Tensor partial;
  while (a.group % (a.split * 2) == 0 && static_cast<int64_t>(a.tiles) * Hkv * a.split * 2 <= 2 * sms) a.split *= 2;
  if (a.split > 1) {
    partial = at::empty({a.split * Hkv * a.T * 2 * D}, lse.options());
    a.partial = partial.data_ptr<float>();
  }
  launch_bwd(static_cast<int>(D), qkv.scalar_type() == at::kHalf, tile_map(qkv, 128), tile_map(qkv, 64), tile_map(dout, 128),
             tile_map(dout, 64), a, pl.q_order, pl.k_order, row_values.data_ptr<float>(),
             at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return dqkv;
}

}  // namespace pa
}  // namespace sb

void bind_packed_attention(pybind11::module& m) {
  m.def("packed_attn_fwd", &sb::pa::fwd, "causal attention over packed sequences");
  m.def("packed_attn_bwd", &sb::pa::bwd, "its backward pass");
}

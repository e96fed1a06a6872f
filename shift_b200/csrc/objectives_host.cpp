// Losses of label log-probabilities: arguments, workspaces and launches.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "objectives.h"

namespace sb {
namespace obj {

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
static int64_t size_of(const at::Tensor& t) { return t.element_size(); }

static void go(Kernel k, const Args& a, const at::Tensor& logits) {
  TORCH_CHECK(a.rows * a.ranks < (1L << 31), "objectives: too many rows for one launch");
  const auto t = logits.scalar_type();
  C10_CUDA_CHECK(run(k, t == at::kBFloat16 ? kBf16 : t == at::kHalf ? kF16 : kF32, a, at::cuda::getCurrentCUDAStream()));
}

static Args base_args(const at::Tensor& logits, const at::Tensor& labels, const char* who) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && logits.size(1) >= 1, who, ": logits [rows, vocabulary] on the device");
  TORCH_CHECK(logits.scalar_type() == at::kBFloat16 || logits.scalar_type() == at::kHalf ||
                  logits.scalar_type() == at::kFloat, who, ": logits in bf16, fp16 or fp32, got ", logits.scalar_type());
  TORCH_CHECK((logits.size(1) <= 1 || logits.stride(1) == 1) && (logits.size(0) <= 1 || logits.stride(0) >= logits.size(1)),
              who, ": logits of inner stride 1 whose rows do not overlap");
  TORCH_CHECK(logits.size(1) <= (1 << 30), who, ": at most 2^30 logits a row");
  TORCH_CHECK(labels.scalar_type() == at::kInt && labels.dim() == 1 && labels.numel() == logits.size(0) &&
                  labels.is_contiguous() && labels.device() == logits.device(),
              who, ": labels are int32, one for each of the ", logits.size(0), " rows, contiguous, beside the logits");
  Args a{};
  a.logits = logits.data_ptr();
  a.labels = labels.data_ptr<int>();
  a.rows = logits.size(0);
  a.stride = a.rows > 1 ? logits.stride(0) : 0;
  a.V = static_cast<int>(logits.size(1));
  a.ranks = 1;
  return a;
}

static float* row_floats(const at::Tensor& t, const at::Tensor& logits, const char* who, const char* what) {
  TORCH_CHECK(t.scalar_type() == at::kFloat && t.dim() == 1 && t.numel() == logits.size(0) && t.is_contiguous() &&
                  t.device() == logits.device(),
              who, ": ", what, " is fp32, one for each of the ", logits.size(0), " rows, contiguous, beside the logits");
  return t.data_ptr<float>();
}

// CTAs a row: enough that a slice can be held (where `hold`), and more while the grid would leave SMs idle and a slice
// keeps at least 8 KB.  (token_logp_fwd, one row: 100003 of bf16 20.5 us by one CTA, 10.4 by eight; 8192 of fp32 8.2 us by one,
// two or four CTAs, 9.3 by eight, of slices of 4 KB.)
static int pick_ranks(const Args& a, int64_t bytes, bool hold) {
  const int64_t sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount, row = bytes * a.V;
  int c = 1;
  while (c < 8 && ((hold && row / c > kHeld) || (a.rows * c < sms && row / (2 * c) >= 8192))) c *= 2;
  return c;
}

std::vector<at::Tensor> logp_fwd(const at::Tensor& logits, const at::Tensor& labels) {
  Args a = base_args(logits, labels, "token_logp_fwd");
  const at::cuda::CUDAGuard guard(logits.device());
  auto logp = at::empty({a.rows}, logits.options().dtype(at::kFloat)), lse = at::empty_like(logp);
  if (a.rows == 0) return {logp, lse};
  a.logp = logp.data_ptr<float>();
  a.lse = lse.data_ptr<float>();
  a.ranks = pick_ranks(a, size_of(logits), false);
  go(kLogp, a, logits);
  return {logp, lse};
}

void logp_bwd(at::Tensor& logits, const at::Tensor& labels, const at::Tensor& lse, const at::Tensor& dlogp) {
  Args a = base_args(logits, labels, "token_logp_bwd");
  a.lse = row_floats(lse, logits, "token_logp_bwd", "lse");
  a.dlogp = row_floats(dlogp, logits, "token_logp_bwd", "dlogp");
  if (a.rows == 0) return;
  const at::cuda::CUDAGuard guard(logits.device());
  a.ranks = pick_ranks(a, size_of(logits), false);
  go(kGrad, a, logits);
}

std::vector<at::Tensor> policy(at::Tensor& logits, const at::Tensor& labels, const at::Tensor& old, const at::Tensor& adv,
                               const c10::optional<at::Tensor>& ref, const c10::optional<at::Tensor>& weight, double low,
                               double high, double kl, double scale, const at::Tensor& status) {
  const char* who = "policy_loss_fwd_bwd";
  TORCH_CHECK(low >= 0 && high >= 0, who, ": clipped to 1 - ", low, ", 1 + ", high);
  TORCH_CHECK(kl == 0 || ref.has_value(), who, ": a KL term needs ref_logp");
  Args a = base_args(logits, labels, who);
  a.t.old = row_floats(old, logits, who, "old_logp");
  a.t.adv = row_floats(adv, logits, who, "adv");
  a.t.ref = ref.has_value() ? row_floats(*ref, logits, who, "ref_logp") : nullptr;
  a.t.weight = weight.has_value() ? row_floats(*weight, logits, who, "weight") : nullptr;
  a.t.low = low;
  a.t.high = high;
  a.t.kl = kl;
  a.t.scale = scale;
  a.status = status.data_ptr<int>();
  const at::cuda::CUDAGuard guard(logits.device());
  auto loss = at::empty({a.rows}, logits.options().dtype(at::kFloat)), logp = at::empty_like(loss);
  if (a.rows == 0) return {loss, logp};
  a.t.loss = loss.data_ptr<float>();
  a.logp = logp.data_ptr<float>();
  a.ranks = pick_ranks(a, size_of(logits), true);
  go(kPolicy, a, logits);
  return {loss, logp};
}

std::vector<at::Tensor> preference(at::Tensor& logits, const at::Tensor& labels, const at::Tensor& ref,
                                   const at::Tensor& offs, double beta, double scale) {
  const char* who = "preference_loss_fwd_bwd";
  Args a = base_args(logits, labels, who);
  const float* rp = row_floats(ref, logits, who, "ref_logp");
  TORCH_CHECK(offs.scalar_type() == at::kInt && offs.dim() == 1 && offs.numel() >= 3 && offs.numel() % 2 == 1 &&
                  offs.is_contiguous() && offs.device() == logits.device(),
              who, ": offs are int32 [2 pairs + 1], contiguous, beside the logits");
  TORCH_CHECK(a.rows < (1L << 31), who, ": too many rows");
  const at::cuda::CUDAGuard guard(logits.device());
  const int64_t pairs = offs.numel() / 2;
  auto rows = at::empty({3, a.rows}, logits.options().dtype(at::kFloat));
  auto logp = at::empty({a.rows}, logits.options().dtype(at::kDouble));
  auto loss = at::empty({pairs}, rows.options()), margin = at::empty_like(loss);
  a.logp64 = logp.data_ptr<double>();
  a.lse = rows.data_ptr<float>();
  a.lse_low = a.lse + a.rows;
  float* dlogp = a.lse_low + a.rows;
  a.dlogp = dlogp;
  a.ranks = pick_ranks(a, size_of(logits), false);
  if (a.rows > 0) go(kLogp, a, logits);
  C10_CUDA_CHECK(run_pairs(static_cast<int>(pairs), a.logp64, rp, a.labels, a.V, offs.data_ptr<int>(), static_cast<int>(a.rows),
                           static_cast<float>(beta), static_cast<float>(scale), loss.data_ptr<float>(),
                           margin.data_ptr<float>(), dlogp, at::cuda::getCurrentCUDAStream()));
  if (a.rows > 0) go(kGrad, a, logits);
  return {loss, margin};
}

}  // namespace obj
}  // namespace sb

void bind_objectives(pybind11::module& m) {
  m.def("token_logp_fwd", &sb::obj::logp_fwd, "log-probability of every row's label, and the row's log-sum-exp");
  m.def("token_logp_bwd", &sb::obj::logp_bwd, "its gradient at the logits, over them");
  m.def("policy_loss", &sb::obj::policy, "clipped policy loss with a KL term; logits become its gradient");
  m.def("preference_loss", &sb::obj::preference, "loss of pairs of sequences; logits become its gradient");
}

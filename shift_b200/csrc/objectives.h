// Losses of label log-probabilities: what their host side (objectives_host.cpp) and their kernels (objectives.cu) share.
#pragma once
#include <cuda_runtime.h>

namespace sb {
namespace obj {

constexpr int kThreads = 256;
constexpr int kHeld = 72 * 1024;        // shared memory of a slice: three CTAs an SM
constexpr int kHeldMost = 216 * 1024;

// What a row's loss hangs on, per kernel
struct Terms {
  const float* old;
  const float* adv;
  const float* ref;       // may be null
  const float* weight;    // may be null
  float* loss;
  double low, high, kl, scale;
};

struct Args {
  void* logits;
  const int* labels;
  long stride;
  long rows;
  int V, ranks;
  float* logp;
  double* logp64;         // instead of logp, unrounded, for sums of many
  float* lse;             // written by the forward pass, read by the backward pass
  float* lse_low;         // and what its rounding left, where both belong to one call; may be null
  const float* dlogp;
  Terms t;
  int* status;
};

enum Kernel { kLogp, kGrad, kPolicy };
enum Type { kBf16, kF16, kF32 };
cudaError_t run(Kernel k, Type type, const Args& a, cudaStream_t stream);
cudaError_t run_pairs(int pairs, const double* logp, const float* ref, const int* labels, int V, const int* offs, int T,
                      float beta, float scale, float* loss, float* margin, float* dlogp, cudaStream_t stream);

}  // namespace obj
}  // namespace sb

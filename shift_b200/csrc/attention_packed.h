// Causal attention over packed sequences: what its host side (attention_packed_host.cpp) and its kernels
// (attention_packed_fwd.cu, attention_packed_bwd.cu) share.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

namespace sb {
namespace pa {

struct Args {
  int T, Hq, Hkv, group;
  int pair_heads;             // forward: an item is two heads over 128 queries (they share keys); else 256 queries of a head
  int split_keys;             // forward: an item is one tile of a head, its key blocks dealt out to the two groups
  int split;                  // dK / dV: CTAs that share a key tile's query heads
  int tiles;
  const int* start;
  const int* stop;
  const int* ends;
  const int* order;
  float scale, scale_log2;
  const void* qkv;
  long ld;                    // elements
  void* o;
  long o_ld;
  float* lse;
  const void* dout;
  long do_ld;
  const float* rows;          // backward: [Hq][tiles * 2][2][64]: -lse log2(e) and -delta of 64 queries
  void* dqkv;
  long dqkv_ld;
  float* partial;             // split > 1: fp32 [split][Hkv][T][2 D]
  float* tops;                // backward, fp16: [Hq][tiles * 128] the largest |do| of a row of a head, else null
  int* shifts;                // and [Hkv][tiles * 128] what dS of a key is scaled by
  int2* later;                // [items][8 warps]: results to be computed again
  int fill;                   // rows that no sequence covers get zeros
  int* status;
};

// D is 64 or 128.  The maps have boxes of 64 columns and as many rows as they say.
void launch_fwd(int D, bool half, const CUtensorMap& qkv, const Args& a, unsigned items, cudaStream_t stream);
void launch_bwd(int D, bool half, const CUtensorMap& qkv128, const CUtensorMap& qkv64, const CUtensorMap& do128,
                const CUtensorMap& do64, const Args& a, const int* q_order, const int* k_order, float* rows,
                cudaStream_t stream);

}  // namespace pa
}  // namespace sb

// Packed sequences: what a buffer's offsets say of every row, and rotary positions.
//
// A packed buffer holds sequences of different lengths one after the other:
// sequence g is rows [offs[g], offs[g + 1]).  Offsets rise; they are cut to the
// buffer, and one below the one before counts as that one.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <limits>

#include "apart.h"
#include "common.cuh"
#include "lowp.cuh"

namespace sb {
namespace packed {

constexpr int kRows = 256;     // rows (and threads) of a CTA of the plan's first kernel
constexpr int kBins = 4096;    // costs of the tile orders; larger ones share the last bin

// start, pos, stop of every row.  A row's sequence begins at the last offset at or before it and ends at the first one
// behind it, so the offsets that fall into a CTA's 256 rows are marked in a bit set and the nearest ones outside are kept
// beside it: no search per row.  Every CTA walks all offsets (a prefix maximum, 256 at a time).
template <int ROWS>
SB_DEVICE void find_rows(const int* __restrict__ offs, int n, int T, int* start, int* pos, int* stop, int* ends) {
  __shared__ unsigned mark[ROWS / 32];
  __shared__ int part[ROWS / 32], s_before, s_after;
  const int r0 = blockIdx.x * ROWS, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x < ROWS / 32) mark[threadIdx.x] = 0;
  if (threadIdx.x == 0) {
    s_before = -1;
    s_after = INT_MAX;
  }
  int carry = 0;                 // the largest offset so far, at least 0
  __syncthreads();
  for (int base = 0; base < n; base += ROWS) {
    const int i = base + threadIdx.x;
    int b = i < n ? min(offs[i], T) : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, b, o);
      if (lane >= o) b = max(b, up);
    }
    if (lane == 31) part[warp] = b;
    __syncthreads();
    int top = carry;
    for (int w = 0; w < ROWS / 32; ++w) {
      if (w < warp) b = max(b, part[w]);
      top = max(top, part[w]);
    }
    b = max(b, carry);
    carry = top;
    if (i < n) {
      if (b < r0) atomicMax(&s_before, b);
      else if (b < r0 + ROWS) atomicOr(&mark[(b - r0) / 32], 1u << ((b - r0) % 32));
      else atomicMin(&s_after, b);
      if (blockIdx.x == 0 && i == 0) ends[0] = b;
    }
    __syncthreads();             // part is written again
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) ends[1] = carry;
  const int r = r0 + threadIdx.x;
  if (r >= T) return;
  int first = s_before, behind = s_after;
  unsigned m = mark[warp] & (0xffffffffu >> (31 - lane));            // offsets at rows up to this one
  int w = warp;
  while (m == 0 && w > 0) m = mark[--w];
  if (m != 0) first = r0 + w * 32 + 31 - __clz(m);
  m = lane == 31 ? 0 : mark[warp] & (0xffffffffu << (lane + 1));
  w = warp;
  while (m == 0 && w < ROWS / 32 - 1) m = mark[++w];
  if (m != 0) behind = r0 + w * 32 + __ffs(m) - 1;
  const bool covered = first >= 0 && behind != INT_MAX;
  start[r] = covered ? first : r + 1;
  pos[r] = covered ? r - first : -1;
  stop[r] = covered ? behind : r;
}

// How many blocks of 128 rows a tile meets.  which: 0 tiles of 128 queries, 1 of 256 queries, 2 of 128 keys.
SB_DEVICE int tile_cost(int which, const int* start, const int* stop, int T, int t) {
  const int rows = which == 1 ? 256 : 128, lo = t * rows, hi = min(lo + rows, T);
  return which == 2 ? (stop[hi - 1] - lo + 127) / 128 : (hi + 127) / 128 - start[lo] / 128;
}

// Orders of the attention kernels' tiles, the costliest first: a counting sort by the number of 128-row blocks that a
// tile meets.  The order decides when a tile runs, nothing else.  By 1024 threads.
SB_DEVICE void find_order(int which, const int* start, const int* stop, int T, int* out) {
  __shared__ __align__(16) int bins[kBins];
  const int rows = which == 1 ? 256 : 128;
  const int nt = (T + rows - 1) / rows;
  auto cost = [&](int t) { return kBins - 1 - max(0, min(tile_cost(which, start, stop, T, t), kBins - 1)); };
  for (int i = threadIdx.x; i < kBins; i += 1024) bins[i] = 0;
  __syncthreads();
  for (int t = threadIdx.x; t < nt; t += 1024) atomicAdd(&bins[cost(t)], 1);
  __syncthreads();
  // exclusive sum over the bins, four to a thread
  __shared__ int warps[32];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  int4 b = reinterpret_cast<int4*>(bins)[threadIdx.x];
  const int mine = b.x + b.y + b.z + b.w;
  int run = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += up;
  }
  if (lane == 31) warps[warp] = run;
  __syncthreads();
  run -= mine;
  for (int w = 0; w < warp; ++w) run += warps[w];
  reinterpret_cast<int4*>(bins)[threadIdx.x] = make_int4(run, run + b.x, run + b.x + b.y, run + b.x + b.y + b.z);
  __syncthreads();
  for (int t = threadIdx.x; t < nt; t += 1024) out[atomicAdd(&bins[cost(t)], 1)] = t;
}

__global__ void __launch_bounds__(kRows)
rows_kernel(const int* __restrict__ offs, int n, int T, int* start, int* pos, int* stop, int* ends) {
  find_rows<kRows>(offs, n, T, start, pos, stop, ends);
}
__global__ void __launch_bounds__(1024)
order_kernel(const int* start, const int* stop, int T, int* fwd, int* fwd2, int* bwd) {
  find_order(blockIdx.x, start, stop, T, blockIdx.x == 0 ? fwd : blockIdx.x == 1 ? fwd2 : bwd);
}
// both for a buffer of at most 1024 rows: one launch of 4.0 us instead of two of 5.1 together (200 rows), and 3 us less of host
__global__ void __launch_bounds__(1024)
small_kernel(const int* __restrict__ offs, int n, int T, int* start, int* pos, int* stop, int* ends, int* fwd, int* fwd2,
             int* bwd) {
  find_rows<1024>(offs, n, T, start, pos, stop, ends);
  __syncthreads();
  // at most eight tiles: one warp an order, a lane a tile, whose place is the number of costlier ones (or alike and before)
  const int which = threadIdx.x / 32, t = threadIdx.x % 32;
  if (which >= 3) return;
  const int rows = which == 1 ? 256 : 128, nt = (T + rows - 1) / rows;
  const int mine = t < nt ? tile_cost(which, start, stop, T, t) : -1;
  int place = 0;
  for (int k = 0; k < nt; ++k) {
    const int other = __shfl_sync(0xffffffffu, mine, k);
    place += other > mine || (other == mine && k < t);
  }
  if (t < nt) (which == 0 ? fwd : which == 1 ? fwd2 : bwd)[place] = t;
}

// The plan: start, pos, stop of every row | first covered row, row behind the last one | tile orders (of 128 queries, 256
// queries, 128 keys).
at::Tensor sequences(const at::Tensor& offs, int64_t rows) {
  TORCH_CHECK(offs.is_cuda() && offs.scalar_type() == at::kInt && offs.dim() == 1 && offs.numel() >= 2 &&
                  offs.is_contiguous(),
              "sequences: offs are int32 [sequences + 1], contiguous, on the device");
  TORCH_CHECK(rows >= 0 && rows <= (1 << 29), "sequences: 0 to 2^29 rows, got ", rows);
  const at::cuda::CUDAGuard guard(offs.device());
  const int64_t nt = (rows + 127) / 128, nt2 = (rows + 255) / 256;
  auto plan = at::empty({3 * rows + 2 + 2 * nt + nt2}, offs.options());
  auto stream = at::cuda::getCurrentCUDAStream();
  const int T = static_cast<int>(rows);
  int* p = plan.data_ptr<int>();
  const int n = static_cast<int>(offs.numel());
  int* o = p + 3L * T + 2;
  if (T <= 1024) {
    small_kernel<<<1, 1024, 0, stream>>>(offs.data_ptr<int>(), n, T, p, p + T, p + 2L * T, p + 3L * T, o, o + nt,
                                         o + nt + nt2);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    return plan;
  }
  rows_kernel<<<(T + kRows - 1) / kRows, kRows, 0, stream>>>(offs.data_ptr<int>(), n, T, p, p + T, p + 2L * T, p + 3L * T);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  order_kernel<<<3, 1024, 0, stream>>>(p, p + 2L * T, T, o, o + nt, o + nt + nt2);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return plan;
}

// ---------------------------------------------------------------------------
// Rotary positions:  y1 = m (x1 cos a - x2 sin a),  y2 = m (x2 cos a + x1 sin a),  a = pos * f
//
// The frequency of a pair is given as a 64-bit fraction of a turn, F = f / (2 pi) * 2^64.  pos * F modulo 2^64 is then
// the angle's fraction of a turn, exact for every position (in fp32, pos * f is off by 0.06 rad at a million), and no
// table of cosines is read.  A thread has `V` elements of one row's pairs (16 bytes where alignment allows), computes
// their sines once and rotates them in up to kHeads heads.  Bound by memory: each rotated value read and written once.  20
// heads of 128 in 16384 rows, bf16: 33 us in place, 39 us into another buffer (84 MB each way; a copy of them takes 33 us);
// one thread for all 20 heads 59 us.
// ---------------------------------------------------------------------------
constexpr int kHeads = 4;

struct RotaryArgs {
  const void* x;
  void* out;
  const int* pos;
  const long long* turns;     // [rot / 2]
  long xs, os;                // row strides, elements
  int T, heads, dim, rot, chunks, live;   // chunks of a head a thread each; the first `live` rotate, the others copy
  float size;
  int inverse;
};

template <typename T, int V, int ALIGN>
struct alignas(ALIGN) Vec {
  T e[V];
};

// ALIGN: alignment of a chunk in bytes; below sizeof(T) * V its elements are read one by one
template <typename T, int V, bool INTER, int ALIGN>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryArgs a) {
  using VT = Vec<T, V, ALIGN>;
  const int c = blockIdx.z * blockDim.x + threadIdx.x;
  const long row = static_cast<long>(blockIdx.x) * blockDim.y + threadIdx.y;
  if (row >= a.T || c >= a.chunks) return;
  const int h0 = blockIdx.y * kHeads, nh = min(kHeads, a.heads - h0);
  const T* xr = static_cast<const T*>(a.x) + row * a.xs + static_cast<long>(h0) * a.dim;
  T* yr = static_cast<T*>(a.out) + row * a.os + static_cast<long>(h0) * a.dim;
  if (c >= a.live) {                                       // columns behind the rotated ones
    const int at = a.rot + (c - a.live) * V;
    if (at + V > a.dim) {                                  // the last column of an odd head, whose pairs still go by two
      for (int h = 0; h < nh; ++h)
        for (int k = at; k < a.dim; ++k) yr[h * a.dim + k] = xr[h * a.dim + k];
      return;
    }
#pragma unroll
    for (int h = 0; h < kHeads; ++h)
      if (h < nh) *reinterpret_cast<VT*>(yr + h * a.dim + at) = *reinterpret_cast<const VT*>(xr + h * a.dim + at);
    return;
  }
  constexpr int P = INTER ? V / 2 : V;                     // pairs
  const int p0 = c * P, at = c * V, half = a.rot / 2;
  VT u[kHeads], v[kHeads];                                 // on their way while the angles are computed
#pragma unroll
  for (int h = 0; h < kHeads; ++h)
    if (h < nh) {
      u[h] = *reinterpret_cast<const VT*>(xr + h * a.dim + at);
      if (!INTER) v[h] = *reinterpret_cast<const VT*>(xr + h * a.dim + half + at);
    }
  float cs[P], sn[P];
  const long long pos = a.pos[row];
#pragma unroll
  for (int j = 0; j < P; ++j) {
    const long long frac = static_cast<long long>(static_cast<unsigned long long>(pos) *
                                                  static_cast<unsigned long long>(a.turns[p0 + j]));
    // half turns in [-1, 1): the 64-bit fraction keeps its leading bits however small the angle is
    const float turn = __ll2float_rn(frac) * 1.0842021724855044e-19f /* 2^-63 */;
    // Within half a turn the hardware's sines are off by 2^-21, so a rotated value by 2^-20 of its pair's size: far below a
    // 16-bit rounding of values of that size, more than that of the few that come out near 0.
    if constexpr (sizeof(T) == 2) {
      sn[j] = __sinf(turn * 3.14159265f);
      cs[j] = __cosf(turn * 3.14159265f);
    } else {
      sincospif(turn, &sn[j], &cs[j]);
    }
    cs[j] *= a.size;
    sn[j] *= a.inverse ? -a.size : a.size;
  }
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    if (h >= nh) break;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      T& e1 = INTER ? u[h].e[2 * j] : u[h].e[j];
      T& e2 = INTER ? u[h].e[2 * j + 1] : v[h].e[j];
      const float x1 = to_float(e1), x2 = to_float(e2);
      // spelled out, so that every width of access rounds alike
      e1 = from_float<T>(__fmaf_rn(x1, cs[j], -__fmul_rn(x2, sn[j])));
      e2 = from_float<T>(__fmaf_rn(x2, cs[j], __fmul_rn(x1, sn[j])));
    }
    *reinterpret_cast<VT*>(yr + h * a.dim + at) = u[h];
    if (!INTER) *reinterpret_cast<VT*>(yr + h * a.dim + half + at) = v[h];
  }
}

template <typename T, int V, int ALIGN = V * static_cast<int>(sizeof(T))>
static void rotary_launch(RotaryArgs a, bool inter, bool copy, cudaStream_t stream) {
  a.live = (inter ? a.rot : a.rot / 2) / V;
  a.chunks = a.live + (copy ? (a.dim - a.rot + V - 1) / V : 0);
  // a row of threads has a row's chunks, so that no index is divided
  const int bx = std::min(a.chunks, 256), by = 256 / bx;
  const dim3 block(bx, by), grid((a.T + by - 1) / by, (a.heads + kHeads - 1) / kHeads, (a.chunks + bx - 1) / bx);
  TORCH_CHECK(grid.y <= 65535 && grid.z <= 65535, "rotary: too many heads, or columns of one, for one launch");
  if (inter) {
    if constexpr (V >= 2) rotary_kernel<T, V, true, ALIGN><<<grid, block, 0, stream>>>(a);
  } else {
    rotary_kernel<T, V, false, ALIGN><<<grid, block, 0, stream>>>(a);
  }
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// Elements per access: the most, up to 16 bytes, that divide every column that a chunk begins at, the row strides and the
// bases.  (16384 rows of 24 heads of 64, bf16: 16-byte accesses 25 us, 2-byte ones 33 us.)
template <typename T>
static void rotary_typed(const RotaryArgs& a, bool inter, bool copy, cudaStream_t stream) {
  const uint64_t all = static_cast<uint64_t>(a.dim) | static_cast<uint64_t>(inter ? a.rot : a.rot / 2) |
                       static_cast<uint64_t>(a.rot) | static_cast<uint64_t>(a.xs) | static_cast<uint64_t>(a.os) |
                       reinterpret_cast<uint64_t>(a.x) / sizeof(T) | reinterpret_cast<uint64_t>(a.out) / sizeof(T);
  if constexpr (sizeof(T) == 2) {
    if (all % 8 == 0) return rotary_launch<T, 8>(a, inter, copy, stream);
  }
  if (all % 4 == 0) return rotary_launch<T, 4>(a, inter, copy, stream);
  if (all % 2 == 0) return rotary_launch<T, 2>(a, inter, copy, stream);
  if (inter) return rotary_launch<T, 2, sizeof(T)>(a, inter, copy, stream);
  rotary_launch<T, 1>(a, inter, copy, stream);
}

void rotary(const at::Tensor& x, at::Tensor& out, const at::Tensor& pos, const at::Tensor& turns, int64_t heads,
            int64_t dim, int64_t rot, bool inter, double size, bool inverse) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && out.dim() == 2, "rotary: matrices [rows, columns] on the device");
  TORCH_CHECK(x.device() == out.device() && x.device() == pos.device() && x.device() == turns.device(),
              "rotary: x, out, positions and the plan on one device");
  TORCH_CHECK(x.size(0) <= (1 << 29), "rotary: at most 2^29 rows, got ", x.size(0));
  TORCH_CHECK(x.scalar_type() == out.scalar_type(), "rotary: out is ", out.scalar_type(), ", x ", x.scalar_type());
  TORCH_CHECK(pos.scalar_type() == at::kInt && pos.dim() == 1 && pos.numel() == x.size(0) && pos.is_contiguous(),
              "rotary: positions are int32, one for each of the ", x.size(0), " rows, contiguous");
  TORCH_CHECK(heads >= 0 && x.size(1) >= heads * dim && out.size(1) >= heads * dim && out.size(0) == x.size(0),
              "rotary: ", heads, " heads of ", dim, " columns do not fit x [", x.size(0), ", ", x.size(1), "] or out [",
              out.size(0), ", ", out.size(1), "]");
  TORCH_CHECK(turns.scalar_type() == at::kLong && turns.is_contiguous() && turns.numel() == rot / 2 && rot >= 2 &&
                  rot % 2 == 0 && rot <= dim, "rotary: a plan of another size");
  for (const at::Tensor& t : {x, out})
    TORCH_CHECK((t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1)),
                "rotary: rows of stride 1 inside that do not overlap");
  const bool same = x.data_ptr() == out.data_ptr() && (x.size(0) <= 1 || x.stride(0) == out.stride(0));
  TORCH_CHECK(same || !share_memory(x, out), "rotary: out overlaps x and is not x itself");
  if (x.size(0) == 0 || heads == 0) return;
  const at::cuda::CUDAGuard guard(x.device());
  RotaryArgs a{x.data_ptr(), out.data_ptr(), pos.data_ptr<int>(),
               reinterpret_cast<const long long*>(turns.data_ptr<int64_t>()),
               x.size(0) > 1 ? x.stride(0) : 0, x.size(0) > 1 ? out.stride(0) : 0, static_cast<int>(x.size(0)),
               static_cast<int>(heads), static_cast<int>(dim), static_cast<int>(rot), 0, 0, static_cast<float>(size),
               inverse ? 1 : 0};
  auto stream = at::cuda::getCurrentCUDAStream();
  const bool copy = !same && dim > rot;
  switch (x.scalar_type()) {
    case at::kBFloat16: rotary_typed<__nv_bfloat16>(a, inter, copy, stream); break;
    case at::kHalf: rotary_typed<__half>(a, inter, copy, stream); break;
    case at::kFloat: rotary_typed<float>(a, inter, copy, stream); break;
    default: TORCH_CHECK(false, "rotary: bf16, fp16 or fp32, got ", x.scalar_type());
  }
}

}  // namespace packed
}  // namespace sb

void bind_packed(pybind11::module& m) {
  m.def("packed_sequences", &sb::packed::sequences, "start, position and end of every row of a packed buffer, tile orders");
  m.def("rotary", &sb::packed::rotary, "rotary positions of the first heads of every row");
}

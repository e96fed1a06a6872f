// 8-bit floating point with one power-of-two scale per block of 128 values:
// what the quantiser, the products and the optimizer share.
//
// A value is code * 2^e.  e is the smallest integer that brings the block's
// largest finite magnitude within the type's largest value 1.75 * 2^top
// (top = 8 for e4m3, 15 for e5m2), kept as a byte e + 127.  Because the scale
// is a power of two, multiplying by it or its reciprocal is exact: the only
// rounding is the conversion to 8 bits.
//
// A matrix [rows, cols] is stored as codes [rows, ld], ld = cols rounded up to
// 16, and scale bytes [ceil(cols / 512)][rows][4]: byte j of word (w, r) is the
// scale of columns [512 w + 128 j, +128) of row r, 0 where there is no such
// column.
#pragma once
#include <cuda_fp8.h>

#include "common.cuh"

namespace sb {
namespace fp8 {

enum Format : int { kE4M3 = 0, kE5M2 = 1 };

// Scale byte of a block whose largest finite magnitude is `amax`: the exponent
// of amax is read from its bits, one more where its fraction is above 1.75.
// Zero (and anything below the smallest scale) gives byte 0, 2^-127.
SB_DEVICE int scale_byte(float amax, int fmt) {
  const int ex = static_cast<int>((__float_as_uint(amax) + 0x1FFFFFu) >> 23);   // biased exponent, carried
  return max(0, min(254, ex - (fmt == kE4M3 ? 8 : 15)));
}
// 2^(127 - byte), the factor that takes values to codes (byte <= 254).
SB_DEVICE float inv_scale(int byte) {
  const int e = 254 - byte;
  return __uint_as_float(e > 0 ? static_cast<uint32_t>(e) << 23 : 0x400000u);
}
// 2^(byte - 127)
SB_DEVICE float scale_of(int byte) {
  return __uint_as_float(byte > 0 ? static_cast<uint32_t>(byte) << 23 : 0x400000u);
}

// Two values to two codes, nearest-even; magnitudes are within range by the
// choice of the scale, so saturation only ever meets infinities (patched by
// the caller).
SB_DEVICE uint32_t pack2(float a, float b, int fmt) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, fmt == kE4M3 ? __NV_E4M3 : __NV_E5M2);
}

}  // namespace fp8
}  // namespace sb

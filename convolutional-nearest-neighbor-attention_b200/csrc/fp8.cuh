// 8-bit values (e4m3) with one float32 scale per block of 128 channels, as the norm, the quantisers and the product's
// epilogue write them.
//   scale = max(amax|block| / 448, 2^-126),  q = e4m3(v * (1 / scale)),  the value that is meant is q * scale
// 448 is the type's largest value.  The bound below keeps 1 / scale finite and a block of zeros at zero.  e4m3 keeps four
// significant bits, so a value is off by at most 2^-4 of itself (or 2^-10 of the scale, where that is more); scales are not
// rounded to powers of two, since nothing downstream asks for it.  A block that holds a NaN or an infinity means NaN
// throughout: its scale is NaN, or infinite over zeros and NaN.
#pragma once
#include <stdint.h>

namespace convnn {
constexpr int kFp8Block = 128;
constexpr float kFp8Least = 1.17549435e-38f;               // 2^-126

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// The largest magnitude of a block as bits (so that NaN, above infinity, is kept) -> its scale.
__device__ __forceinline__ float fp8_scale(uint32_t amax) {
    const float s = __uint_as_float(amax) * (1.0f / 448.0f);
    return s < kFp8Least ? kFp8Least : s;                   // (a comparison with NaN keeps NaN)
}
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) { return e4m3x2(a, b) | (e4m3x2(c, d) << 16); }
}  // namespace convnn

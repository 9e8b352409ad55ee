// rows8.cuh -- rows kept in 8 bits: groups of 32 neighbouring values share a
// scale 2^(byte - 127), the least power of two with |x| <= 127 of them; a value's
// code is x / scale rounded to the nearest integer (ties to even).
//
// A scale that is a power of two makes x / scale and code * scale exact, so codes
// depend on the values alone and not on how a device divides.  Against a scale of
// max|x| / 127 it gives up one bit at most; groups of 32 with one byte each take the
// same room as groups of 128 with an f32 scale, and their maxima lie lower.
// The rounding is at most half a scale, max|x| / 127 (of the group).  Scales below
// 2^-127 do not exist: there the rounding is 2^-128.  A group that holds an infinity
// or a NaN has the byte 255 and reads as NaN.
#pragma once

#include "sequence_common.cuh"

namespace to_b200 {
namespace seq {

constexpr int kGroup8 = 32;

struct Packed {
  int8_t* codes;    // [tokens][width]
  uint8_t* scales;  // [tokens][(width + 31) / 32]
  long long code_stride, scale_stride;
};

inline Packed packed_of(const to_rows8& r) {
  return {static_cast<int8_t*>(r.codes), static_cast<uint8_t*>(r.scales), r.code_stride, r.scale_stride};
}

// The byte of a group whose largest |x| has these bits.
__device__ __forceinline__ int scale_byte(uint32_t most) {
  if (most >= 0x7f800000u) return 255;
  const int b = static_cast<int>(most >> 23) - 6 + ((most & 0x7fffffu) > 0x7e0000u);  // 127 = 1.984375 * 2^6
  return b < 0 ? 0 : b;
}

__device__ __forceinline__ float scale_of(int byte) {
  return __uint_as_float(byte == 255 ? 0x7fc00000u : byte ? static_cast<uint32_t>(byte) << 23 : 0x00400000u);
}

// 1 / scale; 0 for a group that is not finite (whose codes are 0).
__device__ __forceinline__ float inverse_scale(int byte) {
  return byte == 255 ? 0.f : __uint_as_float(static_cast<uint32_t>(254 - byte) << 23);
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// x / scale to the nearest integer, in the low byte (adding 1.5 * 2^23 leaves the
// integer in the sum's last bits; |x / scale| <= 127).
__device__ __forceinline__ uint32_t code_bits(float x, float inverse) {
  return __float_as_uint(fmaf(x, inverse, 12582912.f));
}
__device__ __forceinline__ uint32_t code_of(float x, float inverse, bool finite) {
  return finite ? code_bits(x, inverse) & 0xffu : 0u;
}
// Four of them as a word.
__device__ __forceinline__ uint32_t codes_of(const float* x, float inverse, bool finite) {
  const uint32_t low = __byte_perm(code_bits(x[0], inverse), code_bits(x[1], inverse), 0x0040);
  const uint32_t high = __byte_perm(code_bits(x[2], inverse), code_bits(x[3], inverse), 0x0040);
  return finite ? __byte_perm(low, high, 0x5410) : 0u;
}

// Four codes of a word.
__device__ __forceinline__ void codes_to_f32(uint32_t word, float scale, float (&x)[4]) {
  const uint32_t biased = word ^ 0x80808080u;  // code + 128, put behind the bits of 2^23
#pragma unroll
  for (int i = 0; i < 4; ++i)
    x[i] = (__uint_as_float(__byte_perm(biased, 0x4b000000u, 0x7440 + i)) - 8388736.f) * scale;
}

__device__ __forceinline__ float code_to_f32(int8_t code, float scale) {
  return (__uint_as_float(0x4b000000u | (static_cast<uint32_t>(static_cast<uint8_t>(code)) ^ 0x80u)) - 8388736.f) * scale;
}

// Checks of rows in 8 bits; `tokens` == 0 needs no data.
inline int check_rows8(const char* who, const char* name, const to_rows8& r, int64_t tokens, int32_t width) {
  if (tokens == 0) return ok();
  if (!r.codes || !r.scales) return set_error(TO_ERR_INVALID_ARGUMENT, "%s: %s has no codes or no scales", who, name);
  const int groups = (width + kGroup8 - 1) / kGroup8;
  if (tokens > 1 && (r.code_stride < width || r.scale_stride < groups || r.code_stride > (1ll << 40) ||
                     r.scale_stride > (1ll << 40)))
    return set_error(TO_ERR_INVALID_ARGUMENT, "%s: %s strides (%lld, %lld) for %d values in %d groups", who, name,
                     (long long)r.code_stride, (long long)r.scale_stride, int(width), groups);
  return ok();
}

inline Span codes_span(const char* name, const to_rows8& r, int64_t tokens, int32_t width) {
  return {name, static_cast<const char*>(r.codes), tokens > 1 ? r.code_stride : 0, 0, width, tokens, r.codes ? 1 : 0};
}

inline Span scales_span(const char* name, const to_rows8& r, int64_t tokens, int32_t width) {
  return {name, static_cast<const char*>(r.scales), tokens > 1 ? r.scale_stride : 0, 0,
          (width + kGroup8 - 1) / kGroup8, tokens, r.scales ? 1 : 0};
}

}  // namespace seq
}  // namespace to_b200

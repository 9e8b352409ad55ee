// sequence_common.cuh -- what the sequence operators share: rows of
// [tokens][heads][width] values in bf16 or f32, their vector loads and stores
// (f32 in registers), and the checks of their C-ABI arguments.
#pragma once

#include <cuda_bf16.h>

#include <atomic>
#include <cstdint>

#include "common.hpp"

namespace to_b200 {
namespace seq {

struct Rows {
  char* p;
  long long ts, hs;  // strides in elements
};

inline Rows rows_of(const to_rows& r) {
  return {static_cast<char*>(r.data), r.token_stride, r.head_stride};
}

template <typename T>
__device__ __forceinline__ T* row_ptr(const Rows& r, long long token, int head) {
  return reinterpret_cast<T*>(r.p) + token * r.ts + head * r.hs;
}

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}

// 2^x and 1 / x to about an ulp; results below 2^-126 are zero.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float reciprocal(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int BYTES>
struct Raw;
template <>
struct Raw<2> { using type = uint16_t; };
template <>
struct Raw<4> { using type = uint32_t; };
template <>
struct Raw<8> { using type = uint2; };
template <>
struct Raw<16> { using type = uint4; };

// N consecutive values as f32; the address is aligned to min(16, N * sizeof(T)) bytes.
template <typename T, int N>
__device__ __forceinline__ void load_vec(const T* p, float (&x)[N]) {
  constexpr int kBytes = N * int(sizeof(T));
  constexpr int kStep = kBytes > 16 ? 16 : kBytes;
  constexpr int kPer = kStep / int(sizeof(T));
  using R = typename Raw<kStep>::type;
#pragma unroll
  for (int i = 0; i < kBytes / kStep; ++i) {
    union { R r; T t[kPer]; } u;
    u.r = *(reinterpret_cast<const R*>(p) + i);
#pragma unroll
    for (int j = 0; j < kPer; ++j) x[i * kPer + j] = to_f32(u.t[j]);
  }
}

template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[N]) {
  constexpr int kBytes = N * int(sizeof(T));
  constexpr int kStep = kBytes > 16 ? 16 : kBytes;
  constexpr int kPer = kStep / int(sizeof(T));
  using R = typename Raw<kStep>::type;
#pragma unroll
  for (int i = 0; i < kBytes / kStep; ++i) {
    union { R r; T t[kPer]; } u;
#pragma unroll
    for (int j = 0; j < kPer; ++j) u.t[j] = from_f32<T>(x[i * kPer + j]);
    *(reinterpret_cast<R*>(p) + i) = u.r;
  }
}

// Allow `kernel` its dynamic shared memory on the current device, once a device
// (`done`: a bit for each of the first 64; others are set every time).
template <typename K>
int allow_shared(K* kernel, size_t bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  const int sms = device_sm_count(&dev);
  if (sms <= 0) return -sms;
  const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return ok();
  TO_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)));
  done.fetch_or(bit, std::memory_order_relaxed);
  return ok();
}

inline int dtype_bytes(int32_t dtype) { return dtype == TO_BF16 ? 2 : 4; }

// Checks of one rows argument; `tokens` == 0 needs no data.
inline int check_rows(const char* who, const char* name, const to_rows* r, int64_t tokens,
                      int32_t heads, int32_t width, int32_t dtype) {
  if (!r) return set_error(TO_ERR_INVALID_ARGUMENT, "%s: %s is null", who, name);
  if (tokens == 0 || heads == 0) return ok();
  if (!r->data) return set_error(TO_ERR_INVALID_ARGUMENT, "%s: %s.data is null", who, name);
  if (!aligned(r->data, size_t(dtype_bytes(dtype))))
    return set_error(TO_ERR_ALIGNMENT, "%s: %s.data is not aligned to its type", who, name);
  if ((tokens > 1 && r->token_stride < width) || (heads > 1 && r->head_stride < width))
    return set_error(TO_ERR_INVALID_ARGUMENT, "%s: %s strides (%lld, %lld) are below the width %d",
                     who, name, (long long)r->token_stride, (long long)r->head_stride, int(width));
  if (r->token_stride < 0 || r->head_stride < 0 || r->token_stride > (1ll << 40) ||
      r->head_stride > (1ll << 40))
    return set_error(TO_ERR_INVALID_ARGUMENT, "%s: %s strides are out of range", who, name);
  return ok();
}

// Whether rows can be read and written `bytes` at a time.
inline bool rows_aligned(const to_rows* r, int64_t tokens, int32_t heads, int32_t dtype, int bytes) {
  const int64_t e = dtype_bytes(dtype);
  return aligned(r->data, size_t(bytes)) && (tokens <= 1 || r->token_stride * e % bytes == 0) &&
         (heads <= 1 || r->head_stride * e % bytes == 0);
}

// ---- outputs apart from what a call still reads -----------------------------------

// Rows as they lie in memory, in bytes.
struct Span {
  const char* name;
  const char* p;
  long long ts, hs, width;
  long long tokens;
  int heads;
  long long token_bytes() const { return (heads - 1) * hs + width; }  // a token's heads, first to last
  long long bytes() const { return (tokens - 1) * ts + token_bytes(); }
};

inline Span span_of(const char* name, const to_rows* r, int64_t tokens, int32_t heads, int32_t width, int32_t dtype) {
  const long long e = dtype_bytes(dtype);
  return {name, static_cast<const char*>(r->data), tokens > 1 ? r->token_stride * e : 0,
          heads > 1 ? r->head_stride * e : 0, width * e, tokens, heads};
}

// Whether two different tokens or heads of the rows share memory.
inline bool meets_itself(const Span& a) {
  if (a.tokens <= 1 || a.heads <= 1 || a.ts >= a.token_bytes() || a.hs >= (a.tokens - 1) * a.ts + a.width) return false;
  for (long long h = 1; h < a.heads; ++h) {  // head h of one token and head 0 of a later one
    const long long t = h * a.hs / a.ts;
    if ((t < a.tokens && h * a.hs - t * a.ts < a.width) || (t + 1 < a.tokens && (t + 1) * a.ts - h * a.hs < a.width))
      return true;
  }
  return false;
}

// Whether one token of a and one of b, `shift` bytes on, share memory.
inline bool tokens_meet(const Span& a, const Span& b, long long shift) {
  for (int i = 0, j = 0; i < a.heads && j < b.heads;) {
    const long long x = i * a.hs, y = shift + j * b.hs;
    if (x + a.width <= y) ++i;
    else if (y + b.width <= x) ++j;
    else return true;
  }
  return false;
}

// Whether rows of a and of b share memory.  Exact where both have one token stride that holds a
// token's heads (views into the same packed rows); other layouts whose ranges cross, without
// beginning at the same place, are taken for apart.
inline bool meet(const Span& a, const Span& b) {
  if (!a.heads || !b.heads || !a.tokens) return false;
  const long long d = b.p - a.p;
  if (d >= a.bytes() || -d >= b.bytes()) return false;
  if (d == 0) return true;
  if (a.tokens == 1) return tokens_meet(a, b, d);
  if (a.ts != b.ts || a.ts < a.token_bytes() || b.ts < b.token_bytes()) return false;
  const long long t = d / a.ts - (d % a.ts < 0);  // b begins in a's token t
  return (t < a.tokens && -t < a.tokens && tokens_meet(a, b, d - t * a.ts)) ||
         (t + 1 < a.tokens && tokens_meet(a, b, d - (t + 1) * a.ts));
}

inline int refuse_overlap(const char* who, const char* a, const char* b) {
  return set_error(TO_ERR_INVALID_ARGUMENT, "%s: %s and %s share memory", who, a, b);
}

// The first `outs` of n row arguments are written by CTAs that run while others read the rest.
inline int check_apart(const char* who, const Span* s, int n, int outs) {
  for (int i = 0; i < outs; ++i) {
    if (meets_itself(s[i]))
      return set_error(TO_ERR_INVALID_ARGUMENT, "%s: rows of %s share memory", who, s[i].name);
    for (int j = i + 1; j < n; ++j)
      if (meet(s[i], s[j])) return refuse_overlap(who, s[i].name, s[j].name);
  }
  return ok();
}

// Two arrays of n bytes, either of which may be null.
inline bool arrays_meet(const void* a, const void* b, size_t n) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return a && b && (x < y ? y - x : x - y) < n;
}

}  // namespace seq
}  // namespace to_b200

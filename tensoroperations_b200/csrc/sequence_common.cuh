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

}  // namespace seq
}  // namespace to_b200

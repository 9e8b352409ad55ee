// rows8.cu -- rows of values into 8 bits and back (rows8.cuh), one pass each.
//
// Memory bound: a value is read once and its code written once (3.03 bytes for
// bf16), with about 5 instructions a value.  A thread takes 16 values, two threads a
// group; they exchange nothing but their maxima.  Measured on B200, each behind an L2
// flush: 16384 x 4096 bf16 in 41 us, 5.0 TB/s (0.76 of the copy rate), and back in 39 us,
// 5.2 TB/s; 8192 x 4096 f32 33 and 45 us; single-value accesses, 16384 x 4093 bf16, 184 and
// 358 us.
#include <algorithm>

#include "rows8.cuh"

namespace to_b200 {
namespace {

using seq::Packed;
using seq::Rows;

constexpr int kUnit = 16;  // values of a thread

struct Rows8Args {
  Rows x;
  Packed p;
  long long units;  // of all tokens: an even number a row
  int per_row, width;
  int wide;  // rows of x and codes can be read and written 16 bytes at a time
};

// (a division of 64 bits costs as much as the sixteen values)
__device__ __forceinline__ long long token_of(const Rows8Args& A, long long unit) {
  return A.units <= 0xffffffffll ? static_cast<uint32_t>(unit) / static_cast<uint32_t>(A.per_row) : unit / A.per_row;
}

template <typename T>
__device__ __forceinline__ void load_some(const T* p, int n, float (&x)[kUnit]) {
#pragma unroll
  for (int k = 0; k < kUnit; ++k) x[k] = k < n ? seq::to_f32(p[k]) : 0.f;
}

template <typename T>
__global__ void __launch_bounds__(256) pack_kernel(const __grid_constant__ Rows8Args A) {
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i - (threadIdx.x & 31) < A.units; i += gridDim.x * 256ll) {
    const long long token = token_of(A, i);
    const int c = static_cast<int>(i - token * A.per_row) * kUnit;
    const int n = i < A.units ? min(kUnit, A.width - c) : 0;  // (none in the second half of a short last group)
    const T* from = seq::row_ptr<const T>(A.x, token, 0) + c;
    float x[kUnit];
    if (A.wide && n == kUnit) seq::load_vec<T, kUnit>(from, x);
    else load_some<T>(from, n, x);
    uint32_t most = 0;
#pragma unroll
    for (int k = 0; k < kUnit; ++k) most = max(most, seq::abs_bits(x[k]));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    const int byte = seq::scale_byte(most);
    const float inverse = seq::inverse_scale(byte);
    union { uint4 v; uint32_t w[4]; } u;
#pragma unroll
    for (int k = 0; k < 4; ++k) u.w[k] = seq::codes_of(x + 4 * k, inverse, byte != 255);
    if (n <= 0) continue;
    int8_t* to = A.p.codes + token * A.p.code_stride + c;
    if (A.wide && n == kUnit) {
      *reinterpret_cast<uint4*>(to) = u.v;
    } else {
#pragma unroll
      for (int k = 0; k < kUnit; ++k)
        if (k < n) to[k] = static_cast<int8_t>(u.w[k / 4] >> (8 * (k % 4)));
    }
    if (c % seq::kGroup8 == 0) A.p.scales[token * A.p.scale_stride + c / seq::kGroup8] = static_cast<uint8_t>(byte);
  }
}

template <typename T>
__global__ void __launch_bounds__(256) unpack_kernel(const __grid_constant__ Rows8Args A) {
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < A.units; i += gridDim.x * 256ll) {
    const long long token = token_of(A, i);
    const int c = static_cast<int>(i - token * A.per_row) * kUnit, n = min(kUnit, A.width - c);
    if (n <= 0) continue;
    const float scale = seq::scale_of(A.p.scales[token * A.p.scale_stride + c / seq::kGroup8]);
    const int8_t* from = A.p.codes + token * A.p.code_stride + c;
    T* to = seq::row_ptr<T>(A.x, token, 0) + c;
    if (A.wide && n == kUnit) {
      union { uint4 v; uint32_t w[4]; } u;
      u.v = *reinterpret_cast<const uint4*>(from);
      float x[kUnit];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float y[4];
        seq::codes_to_f32(u.w[k], scale, y);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[4 * k + j] = y[j];
      }
      seq::store_vec<T, kUnit>(to, x);
    } else {
      for (int k = 0; k < n; ++k) to[k] = seq::from_f32<T>(seq::code_to_f32(from[k], scale));
    }
  }
}

// `rows_out`: the rows are written, the codes read.
int run(const char* who, int32_t dtype, int32_t width, int64_t tokens, const to_rows* x, const to_rows8* p,
        bool rows_out, cudaStream_t s) {
  if (dtype != TO_F32 && dtype != TO_BF16)
    return set_error(TO_ERR_UNSUPPORTED, "%s: dtype %d (built: f32, bf16)", who, dtype);
  if (width < 1 || width > (1 << 24)) return set_error(TO_ERR_UNSUPPORTED, "%s: width %d (1 .. 2^24)", who, width);
  if (tokens < 0 || tokens > INT32_MAX)
    return set_error(TO_ERR_INVALID_ARGUMENT, "%s: %lld tokens", who, (long long)tokens);
  if (!x || !p) return set_error(TO_ERR_INVALID_ARGUMENT, "%s: null", who);
  if (tokens == 0) return ok();
  int st = seq::check_rows(who, "x", x, tokens, 1, width, dtype);
  if (!st) st = seq::check_rows8(who, "codes", *p, tokens, width);
  if (st) return st;
  const seq::Span rows = seq::span_of("x", x, tokens, 1, width, dtype);
  const seq::Span codes = seq::codes_span("codes", *p, tokens, width), scales = seq::scales_span("scales", *p, tokens, width);
  const seq::Span packing[] = {codes, scales, rows}, unpacking[] = {rows, codes, scales};
  if ((st = seq::check_apart(who, rows_out ? unpacking : packing, 3, rows_out ? 1 : 2))) return st;
  Rows8Args A{};
  A.x = seq::rows_of(*x);
  A.p = seq::packed_of(*p);
  A.width = width;
  A.per_row = (width + seq::kGroup8 - 1) / seq::kGroup8 * 2;
  A.units = tokens * A.per_row;
  A.wide = seq::rows_aligned(x, tokens, 1, dtype, 16) && aligned(p->codes, 16) && (tokens <= 1 || p->code_stride % 16 == 0);
  int dev = 0;
  const int sms = device_sm_count(&dev);
  if (sms <= 0) return -sms;
  const unsigned grid = static_cast<unsigned>(std::min<long long>((A.units + 255) / 256, 16ll * sms));
  if (rows_out) {
    if (dtype == TO_BF16) unpack_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(A);
    else unpack_kernel<float><<<grid, 256, 0, s>>>(A);
  } else {
    if (dtype == TO_BF16) pack_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(A);
    else pack_kernel<float><<<grid, 256, 0, s>>>(A);
  }
  TO_CUDA_TRY(cudaGetLastError());
  return ok();
}

}  // namespace
}  // namespace to_b200

using namespace to_b200;

extern "C" {

int to_rows8_pack(int32_t dtype, int32_t width, int64_t tokens, const to_rows* x, const to_rows8* out, void* stream) {
  return run("to_rows8_pack", dtype, width, tokens, x, out, false, static_cast<cudaStream_t>(stream));
}

int to_rows8_unpack(int32_t dtype, int32_t width, int64_t tokens, const to_rows8* in, const to_rows* x, void* stream) {
  return run("to_rows8_unpack", dtype, width, tokens, x, in, true, static_cast<cudaStream_t>(stream));
}

}  // extern "C"

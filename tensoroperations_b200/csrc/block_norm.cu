// block_norm.cu -- what lies between two blocks: the norm of a block's output, its
// gate, the scaled sum with the residual stream and the next block's norm, in one
// pass over the rows; and the pass's gradients.
//
//   forward   u = w_post y / rms(y),  r' = r + scale u act(g),  n = w_pre r' / rms(r')
//   backward  e = w_pre dn,  t = dr' + (e - r^ mean(e r^)) / rms(r') = dr,
//             q = scale t,  dg = q u act'(g),  d = w_post q act(g),
//             dy = (d - y^ mean(d y^)) / rms(y)     (x^ = x / rms(x))
//             dw_pre = sum dn r^,  dw_post = sum q act(g) y^
//
// Memory bound: 15 to 40 flops a value, of which each is read once and written
// once.  A row lies in the registers of one warp, or of all warps of a CTA: sixteen
// values a thread (eight up to 256 values a row), each eight of them one 16-byte access
// of bf16; where addresses or widths do not allow that, neighbouring threads take
// neighbouring values.  (With eight values a thread the sums over a row took as many
// instructions as the values.)  The two sums of the forward pass follow one another, the
// gradients' three first ones are taken together.
//
// Measured on B200: 16384 x 4096 bf16 with a silu gate and an f32 stream in 164 us, 5.7 TB/s
// (0.88 of the copy rate), 8192 x 4096 f32 119 us (0.87), bf16 with 8-bit copies 109 us, 4.0
// TB/s.  Gradients of 8192 x 4096 bf16 in 145 us, 3.7 TB/s, from 8 bits 157 us, 2.8 TB/s: two
// rows an SM, whose loads, sums and 85 instructions a value follow one another; f32 199 us, 5.4
// TB/s.  6137 x 1003 f32 without a gate 242 us (registers of the single-value form are spilled),
// gradients 65 us.
#include <algorithm>
#include <cmath>

#include "rows8.cuh"
#include "sm100_primitives.cuh"

namespace to_b200 {
namespace {

using seq::Packed;
using seq::Rows;

constexpr int kVals = 8;  // values of a unit
constexpr int kMaxWarps = 32;

// A unit of a row as it lies in memory, and which of its values there are.
template <typename T>
struct Unit {
  static constexpr int kWords = kVals * int(sizeof(T)) / 4;
  uint32_t raw[kWords];

  __device__ __forceinline__ float operator[](int k) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(raw[k]);
    else return __uint_as_float(k & 1 ? raw[k / 2] & 0xffff0000u : raw[k / 2] << 16);
  }
  __device__ __forceinline__ V2<float> pair(int k) const {  // values 2 k, 2 k + 1
    if constexpr (sizeof(T) == 4) return mk2(__uint_as_float(raw[2 * k]), __uint_as_float(raw[2 * k + 1]));
    else return mk2(__uint_as_float(raw[k] << 16), __uint_as_float(raw[k] & 0xffff0000u));
  }
  __device__ __forceinline__ void set(const float (&x)[kVals]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int k = 0; k < kVals; ++k) raw[k] = __float_as_uint(x[k]);
    } else {
#pragma unroll
      for (int k = 0; k < kWords; ++k) {
        const __nv_bfloat162 p = __floats2bfloat162_rn(x[2 * k], x[2 * k + 1]);
        raw[k] = *reinterpret_cast<const uint32_t*>(&p);
      }
    }
  }
};

// Where a thread's unit lies in a row: WIDE, eight neighbouring columns; otherwise
// every `step`-th one.
template <bool WIDE>
struct Place {
  int first, step, width;
  __device__ __forceinline__ Place(int u, int width_) : width(width_) {
    first = WIDE ? (u * blockDim.x + threadIdx.x) * kVals : u * blockDim.x * kVals + threadIdx.x;
    step = WIDE ? 1 : blockDim.x;
  }
  __device__ __forceinline__ int col(int k) const { return first + k * step; }
  __device__ __forceinline__ bool on(int k) const { return WIDE ? first < width : col(k) < width; }
};

template <typename T, bool WIDE>
__device__ __forceinline__ void load_unit(const T* row, const Place<WIDE>& pl, Unit<T>& x) {
  if constexpr (WIDE) {
    constexpr int kSteps = Unit<T>::kWords / 4;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (pl.on(0)) v = *(reinterpret_cast<const uint4*>(row + pl.first) + i);
      x.raw[4 * i] = v.x, x.raw[4 * i + 1] = v.y, x.raw[4 * i + 2] = v.z, x.raw[4 * i + 3] = v.w;
    }
  } else {
    float v[kVals];
#pragma unroll
    for (int k = 0; k < kVals; ++k) v[k] = pl.on(k) ? seq::to_f32(row[pl.col(k)]) : 0.f;
    x.set(v);
  }
}

template <typename T, bool WIDE>
__device__ __forceinline__ void store_unit(T* row, const Place<WIDE>& pl, const float (&x)[kVals]) {
  if constexpr (WIDE) {
    if (pl.on(0)) seq::store_vec<T, kVals>(row + pl.first, x);
  } else {
#pragma unroll
    for (int k = 0; k < kVals; ++k)
      if (pl.on(k)) row[pl.col(k)] = seq::from_f32<T>(x[k]);
  }
}

// f32 values of the whole row, or 1 where there are none.
template <bool WIDE>
__device__ __forceinline__ void load_weights(const float* w, const Place<WIDE>& pl, float (&x)[kVals]) {
#pragma unroll
  for (int k = 0; k < kVals; ++k) x[k] = 1.f;
  if (!w) return;
  if constexpr (WIDE) {
    if (!pl.on(0)) return;
    const float4 a = __ldg(reinterpret_cast<const float4*>(w + pl.first)), b = __ldg(reinterpret_cast<const float4*>(w + pl.first) + 1);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
#pragma unroll
    for (int k = 0; k < kVals; ++k)
      if (pl.on(k)) x[k] = __ldg(w + pl.col(k));
  }
}

// A unit into 8 bits.  A group of 32 columns is held by four lanes (WIDE), or
// each of its values by one lane.  Whole warps.
template <bool WIDE>
__device__ __forceinline__ void keep_unit(const Packed& out, long long token, const Place<WIDE>& pl, const float (&x)[kVals]) {
  int8_t* codes = out.codes + token * out.code_stride;
  uint8_t* scales = out.scales + token * out.scale_stride;
  if constexpr (WIDE) {
    uint32_t most = 0;
#pragma unroll
    for (int k = 0; k < kVals; ++k) most = max(most, seq::abs_bits(x[k]));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
    const int byte = seq::scale_byte(most);
    const float inverse = seq::inverse_scale(byte);
    if (!pl.on(0)) return;
    *reinterpret_cast<uint2*>(codes + pl.first) =
        make_uint2(seq::codes_of(x, inverse, byte != 255), seq::codes_of(x + 4, inverse, byte != 255));
    if (threadIdx.x % 4 == 0) scales[pl.first / seq::kGroup8] = static_cast<uint8_t>(byte);
  } else {
#pragma unroll
    for (int k = 0; k < kVals; ++k) {
      const int byte = seq::scale_byte(__reduce_max_sync(0xffffffffu, seq::abs_bits(x[k])));
      const uint32_t code = seq::code_of(x[k], seq::inverse_scale(byte), byte != 255);
      if (pl.on(k)) {
        codes[pl.col(k)] = static_cast<int8_t>(code);
        if (threadIdx.x % 32 == 0) scales[pl.col(k) / seq::kGroup8] = static_cast<uint8_t>(byte);
      }
    }
  }
}

// A unit's codes (WIDE: in its first two words) and its scale, and their values afterwards: the
// codes of all rows are on their way before the first of them is waited for.
template <typename T, bool WIDE>
__device__ __forceinline__ int load_kept(const Packed& in, long long token, const Place<WIDE>& pl, Unit<T>& x) {
  const int8_t* codes = in.codes + token * in.code_stride;
  const uint8_t* scales = in.scales + token * in.scale_stride;
  if constexpr (WIDE) {
    x.raw[0] = x.raw[1] = 0;
    if (!pl.on(0)) return 0;
    const uint2 w = *reinterpret_cast<const uint2*>(codes + pl.first);
    x.raw[0] = w.x, x.raw[1] = w.y;
    return scales[pl.first / seq::kGroup8];
  } else {
    float v[kVals];
#pragma unroll
    for (int k = 0; k < kVals; ++k)
      v[k] = pl.on(k) ? seq::code_to_f32(codes[pl.col(k)], seq::scale_of(scales[pl.col(k) / seq::kGroup8])) : 0.f;
    x.set(v);  // (7 bits and a sign: exact in either type)
    return 0;
  }
}
template <bool WIDE, typename T>
__device__ __forceinline__ void expand(Unit<T>& x, int byte) {
  if constexpr (WIDE) {
    const float scale = seq::scale_of(byte);
    float a[4], b[4], v[kVals];
    seq::codes_to_f32(x.raw[0], scale, a);
    seq::codes_to_f32(x.raw[1], scale, b);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = a[k], v[4 + k] = b[k];
    x.set(v);
  }
}

// Sums over a row: of the warp, then of the CTA's warps in order.  `turn` picks one
// of two buffers, so that one barrier a sum is enough.
template <int N>
struct RowSums {
  float (*part)[N][kMaxWarps];
  int turn = 0;
  __device__ __forceinline__ void operator()(float (&v)[N]) {
#pragma unroll
    for (int o = 16; o; o >>= 1)
#pragma unroll
      for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
    const int warps = blockDim.x / 32;
    if (warps == 1) return;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    if (lane == 0) {
#pragma unroll
      for (int n = 0; n < N; ++n) part[turn][n][warp] = v[n];
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {
      v[n] = 0.f;
      const float4* from = reinterpret_cast<const float4*>(part[turn][n]);
      for (int w = 0; w < warps; w += 4) {  // (the rest of a four is zero)
        const float4 x = from[w / 4];
        v[n] += (x.x + x.y) + (x.z + x.w);
      }
    }
    turn ^= 1;
  }
  __device__ __forceinline__ void clear() {
    for (int i = threadIdx.x; i < 2 * N * kMaxWarps; i += blockDim.x) (&part[0][0][0])[i] = 0.f;
    __syncthreads();
  }
};

// The gate's factors and, for the gradients, their slopes.  (One branch for eight values.)
template <bool SLOPES, typename T>
__device__ __forceinline__ void gate_of(int kind, const Unit<T>& g, float (&factor)[kVals], float (&slope)[kVals]) {
  if (kind == TO_GATE_NONE) {
#pragma unroll
    for (int k = 0; k < kVals; ++k) factor[k] = 1.f;
  } else if (kind == TO_GATE_LINEAR) {
#pragma unroll
    for (int k = 0; k < kVals; ++k) {
      factor[k] = g[k];
      if (SLOPES) slope[k] = 1.f;
    }
  } else {
#pragma unroll
    for (int k = 0; k < kVals; ++k) {
      float t = -1.4426950408889634f * g[k];
      asm("min.NaN.f32 %0, %1, 0f42FC0000;" : "=f"(t) : "f"(t));  // 126: sigmoid(g) is 2^-126 at least
      const float e = seq::exp2_fast(t);
      const float p = seq::reciprocal(1.f + e);               // sigmoid(g); 1 - sigmoid(g) is e p
      factor[k] = kind == TO_GATE_SIGMOID ? p : g[k] * p;
      if (SLOPES) slope[k] = kind == TO_GATE_SIGMOID ? p * (e * p) : fmaf(factor[k], e * p, p);
    }
  }
}

// ---- forward -----------------------------------------------------------------------

struct ForwardArgs {
  Rows r, y, g, r_out, n;  // p null: not there
  Packed keep_r, keep_y, keep_g;
  const float* w_post;
  const float* w_pre;
  long long tokens;
  int width, gate, post_norm;
  float scale, eps;
};

template <typename T, typename R, int U, bool WIDE, int MOST>
__global__ void __launch_bounds__(MOST, MOST == 256 ? 3 : MOST == 512 ? 2 : 1) forward_kernel(const __grid_constant__ ForwardArgs A) {
  __shared__ alignas(16) float part[2][1][kMaxWarps];
  RowSums<1> sums{part};
  const float inv = 1.f / static_cast<float>(A.width);
  const bool has_y = A.y.p, keeps = A.keep_r.codes || A.keep_y.codes || A.keep_g.codes;
  const int gate = A.g.p ? A.gate : TO_GATE_NONE;
  if (blockDim.x > 32) sums.clear();
  for (long long t = blockIdx.x * static_cast<long long>(blockDim.y) + threadIdx.y; t < A.tokens;
       t += gridDim.x * static_cast<long long>(blockDim.y)) {
    Unit<R> r[U];
    Unit<T> y[U], g[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const Place<WIDE> pl(u, A.width);
      load_unit<R>(seq::row_ptr<const R>(A.r, t, 0), pl, r[u]);
      if (has_y) load_unit<T>(seq::row_ptr<const T>(A.y, t, 0), pl, y[u]);
      if (gate != TO_GATE_NONE) load_unit<T>(seq::row_ptr<const T>(A.g, t, 0), pl, g[u]);
    }
    float x[U][kVals], s[1] = {0.f};
    if (has_y) {
      float f = A.scale;
      if (A.post_norm) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int k = 0; k < kVals; ++k) s[0] = fmaf(y[u][k], y[u][k], s[0]);
        sums(s);
        f *= rsqrtf(fmaf(s[0], inv, A.eps));
        s[0] = 0.f;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float w[kVals], a[kVals], none[kVals];
        load_weights<WIDE>(A.w_post, Place<WIDE>(u, A.width), w);
        gate_of<false>(gate, g[u], a, none);
#pragma unroll
        for (int k = 0; k < kVals; ++k) x[u][k] = fmaf(f * w[k] * a[k], y[u][k], r[u][k]);
      }
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < kVals; ++k) x[u][k] = r[u][k];
    }
    if (A.r_out.p) {
#pragma unroll
      for (int u = 0; u < U; ++u) store_unit<R>(seq::row_ptr<R>(A.r_out, t, 0), Place<WIDE>(u, A.width), x[u]);
    }
    if (keeps) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const Place<WIDE> pl(u, A.width);
        float v[kVals];
        if (A.keep_r.codes) keep_unit<WIDE>(A.keep_r, t, pl, x[u]);
        if (A.keep_y.codes) {
#pragma unroll
          for (int k = 0; k < kVals; ++k) v[k] = y[u][k];
          keep_unit<WIDE>(A.keep_y, t, pl, v);
        }
        if (A.keep_g.codes) {
#pragma unroll
          for (int k = 0; k < kVals; ++k) v[k] = g[u][k];
          keep_unit<WIDE>(A.keep_g, t, pl, v);
        }
      }
    }
    if (!A.n.p) continue;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int k = 0; k < kVals; ++k) s[0] = fmaf(x[u][k], x[u][k], s[0]);
    sums(s);
    const float m = rsqrtf(fmaf(s[0], inv, A.eps));
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const Place<WIDE> pl(u, A.width);
      float w[kVals];
      load_weights<WIDE>(A.w_pre, pl, w);
#pragma unroll
      for (int k = 0; k < kVals; ++k) x[u][k] = m * w[k] * x[u][k];
      store_unit<T>(seq::row_ptr<T>(A.n, t, 0), pl, x[u]);
    }
  }
}

// ---- backward ----------------------------------------------------------------------

struct BackwardArgs {
  Rows r, y, g, dr_out, dn, dr, dy, dg;
  Packed r8, y8, g8;
  const float* w_post;
  const float* w_pre;
  float* partial;  // [CTAs][2][width]: sums for dw_pre and dw_post
  long long tokens;
  int width, gate, post_norm, has_y;
  float scale, eps;
};

template <typename T, typename R, int U, bool WIDE, int MOST>
__global__ void __launch_bounds__(MOST, MOST == 256 ? 2 : 1) backward_kernel(const __grid_constant__ BackwardArgs A) {
  __shared__ alignas(16) float part[2][3][kMaxWarps], part_d[2][1][kMaxWarps];
  // this thread's columns of dw_pre and dw_post, four at a time: in registers they would take the
  // room of values that would be unpacked again at each use (a quarter of all instructions)
  extern __shared__ __align__(16) char shared[];
  constexpr int kPairs = kVals / 2;
  RowSums<3> sums{part};
  RowSums<1> sum_d{part_d};
  const float inv = 1.f / static_cast<float>(A.width);
  const int gate = A.has_y ? A.gate : TO_GATE_NONE;
  if (blockDim.x > 32) {
    sums.clear();
    sum_d.clear();
  }
  const int threads = blockDim.x * blockDim.y, thread = threadIdx.y * blockDim.x + threadIdx.x;
  auto columns = [&](int which, int u, int half) -> float4& {
    return reinterpret_cast<float4*>(shared)[((which * U + u) * 2 + half) * threads + thread];
  };
#pragma unroll
  for (int u = 0; u < 2 * U; ++u)
#pragma unroll
    for (int h = 0; h < 2; ++h) columns(u / U, u % U, h) = make_float4(0.f, 0.f, 0.f, 0.f);
  auto gather = [&](int which, int u, const V2<float> (&x)[kPairs]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float4 c = columns(which, u, h);
      const V2<float> a = add2(mk2(c.x, c.y), x[2 * h]), b = add2(mk2(c.z, c.w), x[2 * h + 1]);
      columns(which, u, h) = make_float4(a.v.x, a.v.y, b.v.x, b.v.y);
    }
  };
  const long long stride = gridDim.x * static_cast<long long>(blockDim.y);
  for (long long t = blockIdx.x * static_cast<long long>(blockDim.y) + threadIdx.y; t < A.tokens; t += stride) {
    Unit<R> r_[U], dr_[U];
    Unit<T> y_[U], g[U], dn_[U];
    int bytes[U][3];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const Place<WIDE> pl(u, A.width);
      const float zero[kVals] = {};
      if (A.r8.codes) bytes[u][0] = load_kept<R>(A.r8, t, pl, r_[u]);
      else load_unit<R>(seq::row_ptr<const R>(A.r, t, 0), pl, r_[u]);
      if (A.dn.p) load_unit<T>(seq::row_ptr<const T>(A.dn, t, 0), pl, dn_[u]);
      else dn_[u].set(zero);
      if (A.dr_out.p) load_unit<R>(seq::row_ptr<const R>(A.dr_out, t, 0), pl, dr_[u]);
      else dr_[u].set(zero);
      if (A.y8.codes) bytes[u][1] = load_kept<T>(A.y8, t, pl, y_[u]);
      else if (A.y.p) load_unit<T>(seq::row_ptr<const T>(A.y, t, 0), pl, y_[u]);
      else y_[u].set(zero);
      if (A.g8.codes) bytes[u][2] = load_kept<T>(A.g8, t, pl, g[u]);
      else if (A.g.p) load_unit<T>(seq::row_ptr<const T>(A.g, t, 0), pl, g[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (A.r8.codes) expand<WIDE>(r_[u], bytes[u][0]);
      if (A.y8.codes) expand<WIDE>(y_[u], bytes[u][1]);
      if (A.g8.codes) expand<WIDE>(g[u], bytes[u][2]);
    }
    V2<float> r[U][kPairs], y[U][kPairs], dn[U][kPairs];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int k = 0; k < kPairs; ++k) r[u][k] = r_[u].pair(k), y[u][k] = y_[u].pair(k), dn[u][k] = dn_[u].pair(k);
    V2<float> s0 = mk2(0.f, 0.f), s1 = s0, s2 = s0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float w[kVals];
      load_weights<WIDE>(A.w_pre, Place<WIDE>(u, A.width), w);
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {
        s0 = fma2(r[u][k], r[u][k], s0);
        s1 = fma2(y[u][k], y[u][k], s1);
        s2 = fma2(mul2(mk2(w[2 * k], w[2 * k + 1]), dn[u][k]), r[u][k], s2);
      }
    }
    float s[3] = {s0.v.x + s0.v.y, s1.v.x + s1.v.y, s2.v.x + s2.v.y};
    sums(s);
    const float mr = rsqrtf(fmaf(s[0], inv, A.eps)), my = A.post_norm ? rsqrtf(fmaf(s[1], inv, A.eps)) : 1.f;
    // -mean(e r^) / rms: made of mean(e r) / rms, so that no power of 1 / rms leaves f32 before dr does
    // (1 / rms^3 is infinite below an rms of 1.4e-13 and zero above 1e15)
    const float back = -(mr * s[2] * inv) * mr;
    const V2<float> mr2 = mk2(mr, mr), my2 = mk2(my, my), back2 = mk2(back, back), scale2 = mk2(A.scale, A.scale);
    V2<float> d2 = mk2(0.f, 0.f);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const Place<WIDE> pl(u, A.width);
      float w[kVals], out[kVals];
      load_weights<WIDE>(A.w_pre, pl, w);
      V2<float> q[kPairs], add[kPairs];
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {
        const V2<float> m = mul2(mr2, dn[u][k]), rh = mul2(mr2, r[u][k]);  // rh: r^
        q[k] = fma2(mk2(w[2 * k], w[2 * k + 1]), m, fma2(back2, rh, dr_[u].pair(k)));
        add[k] = mul2(dn[u][k], rh);
        out[2 * k] = q[k].v.x, out[2 * k + 1] = q[k].v.y;
      }
      if (A.partial) gather(0, u, add);
      store_unit<R>(seq::row_ptr<R>(A.dr, t, 0), pl, out);
      if (!A.has_y) continue;
      load_weights<WIDE>(A.w_post, pl, w);
      float a[kVals], slope[kVals];
      gate_of<true>(gate, g[u], a, slope);
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {
        const V2<float> sq = mul2(scale2, q[k]), du = mul2(sq, mk2(a[2 * k], a[2 * k + 1]));
        const V2<float> wk = mk2(w[2 * k], w[2 * k + 1]);
        y[u][k] = mul2(my2, y[u][k]);  // y^
        if (gate != TO_GATE_NONE) {
          const V2<float> o = mul2(mul2(sq, mk2(slope[2 * k], slope[2 * k + 1])), mul2(wk, y[u][k]));
          out[2 * k] = o.v.x, out[2 * k + 1] = o.v.y;
        }
        add[k] = mul2(du, y[u][k]);
        dn[u][k] = mul2(wk, du);
        d2 = fma2(dn[u][k], y[u][k], d2);
      }
      if (A.partial) gather(1, u, add);
      if (gate != TO_GATE_NONE) store_unit<T>(seq::row_ptr<T>(A.dg, t, 0), pl, out);
    }
    if (!A.has_y) continue;
    float m = 0.f;
    if (A.post_norm) {
      float d[1] = {d2.v.x + d2.v.y};
      sum_d(d);
      m = -d[0] * inv;
    }
    const V2<float> m2 = mk2(m, m);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float out[kVals];
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {
        const V2<float> o = mul2(my2, fma2(m2, y[u][k], dn[u][k]));
        out[2 * k] = o.v.x, out[2 * k + 1] = o.v.y;
      }
      store_unit<T>(seq::row_ptr<T>(A.dy, t, 0), Place<WIDE>(u, A.width), out);
    }
  }
  if (!A.partial) return;
  // the CTA's rows in order
  __syncthreads();
  float* to = A.partial + blockIdx.x * 2ll * A.width;
  if (threadIdx.y) return;
#pragma unroll
  for (int u = 0; u < 2 * U; ++u) {
    float x[kVals] = {};
    for (int row = 0; row < static_cast<int>(blockDim.y); ++row)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float4 c = (&columns(u / U, u % U, h))[row * blockDim.x];
        x[4 * h] += c.x, x[4 * h + 1] += c.y, x[4 * h + 2] += c.z, x[4 * h + 3] += c.w;
      }
    store_unit<float>(to + (u / U) * A.width, Place<WIDE>(u % U, A.width), x);
  }
}

// dw = sum over CTAs of their partial sums, in a fixed order, in f64.  blockIdx.y: dw_pre or dw_post.
__global__ void __launch_bounds__(1024) weight_sum_kernel(const float* __restrict__ partial, int ctas, int width,
                                                          float* dw_pre, float* dw_post) {
  __shared__ double part[32][33];
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5, x = blockIdx.x * 32 + lane;
  double v = 0;
  if (x < width) {
#pragma unroll 8
    for (int c = row; c < ctas; c += 32) v += partial[(2ll * c + blockIdx.y) * width + x];
  }
  part[row][lane] = v;
  __syncthreads();
  float* dst = blockIdx.y ? dw_post : dw_pre;
  if (row == 0 && x < width && dst) {
    for (int k = 1; k < 32; ++k) v += part[k][lane];
    dst[x] = static_cast<float>(v);
  }
}

// ---- host --------------------------------------------------------------------------

int check_desc(const char* who, const to_block_norm_desc* desc) {
  if (!desc) return set_error(TO_ERR_INVALID_ARGUMENT, "%s: null descriptor", who);
  const to_block_norm_desc& d = *desc;
  if (d.dtype != TO_F32 && d.dtype != TO_BF16)
    return set_error(TO_ERR_UNSUPPORTED, "%s: dtype %d (built: f32, bf16)", who, d.dtype);
  if (d.residual != TO_F32 && d.residual != d.dtype)
    return set_error(TO_ERR_UNSUPPORTED, "%s: residual %d with dtype %d (built: f32, or the same)", who, d.residual, d.dtype);
  if (d.width < 1 || d.width > 16384) return set_error(TO_ERR_UNSUPPORTED, "%s: width %d (1 .. 16384)", who, d.width);
  if (d.gate < TO_GATE_NONE || d.gate > TO_GATE_SILU) return set_error(TO_ERR_INVALID_ARGUMENT, "%s: gate %d", who, d.gate);
  if (d.post_norm != 0 && d.post_norm != 1)
    return set_error(TO_ERR_INVALID_ARGUMENT, "%s: post_norm %d", who, d.post_norm);
  // (the kernels hold both in f32: one that is infinite there, or an eps that becomes zero, is refused too)
  if (!std::isfinite(static_cast<float>(d.scale)) || !(d.eps >= 0) || !std::isfinite(static_cast<float>(d.eps)) ||
      (d.eps > 0 && static_cast<float>(d.eps) == 0))
    return set_error(TO_ERR_INVALID_ARGUMENT, "%s: scale %g, eps %g", who, d.scale, d.eps);
  return ok();
}

// Threads of a row, rows of a CTA and units of a thread.
struct Shape {
  int threads, rows, units;
};
Shape shape_of(int width) {
  const int units = width > 256 ? 2 : 1;
  const int per = (width + kVals * units - 1) / (kVals * units);  // threads
  const int threads = (per + 31) / 32 * 32;
  return {threads, threads == 32 ? 8 : 1, units};
}

// CTAs of the gradients: what fits the SMs at once (their sums are added up afterwards).
int backward_ctas(int width, long long tokens, int sms) {
  const Shape s = shape_of(width);
  const long long per_sm = std::max(1, 512 / (s.threads * s.rows));
  return static_cast<int>(std::max<long long>(1, std::min(per_sm * sms, (tokens + s.rows - 1) / s.rows)));
}

// launch(T, R, units, wide, threads of the largest CTA)
template <typename F>
int each_kernel(const to_block_norm_desc& d, bool wide, const Shape& shape, F&& launch) {
  auto sized = [&](auto t, auto r, auto w) {
    using One = std::integral_constant<int, 1>;
    using Two = std::integral_constant<int, 2>;
    if (shape.units == 1) return launch(t, r, One{}, w, std::integral_constant<int, 256>{});
    if (shape.threads * shape.rows <= 256) return launch(t, r, Two{}, w, std::integral_constant<int, 256>{});
    if (shape.threads <= 512) return launch(t, r, Two{}, w, std::integral_constant<int, 512>{});
    return launch(t, r, Two{}, w, std::integral_constant<int, 1024>{});
  };
  auto with = [&](auto t, auto r) { return wide ? sized(t, r, std::true_type{}) : sized(t, r, std::false_type{}); };
  if (d.dtype == TO_F32) return with(float{}, float{});
  return d.residual == TO_F32 ? with(__nv_bfloat16{}, float{}) : with(__nv_bfloat16{}, __nv_bfloat16{});
}

// The rows of a call: their checks, whether they can be read eight values at a time, and where they lie.
struct RowSet {
  const char* who;
  const to_block_norm_desc& d;
  int64_t tokens;
  bool wide;
  seq::Span spans[20];
  int count = 0;

  RowSet(const char* w, const to_block_norm_desc& desc, int64_t t) : who(w), d(desc), tokens(t), wide(desc.width % kVals == 0) {}
  int rows(const char* name, const to_rows& r, int32_t dtype) {
    if (int st = seq::check_rows(who, name, &r, tokens, 1, d.width, dtype)) return st;
    wide = wide && seq::rows_aligned(&r, tokens, 1, dtype, 16);
    spans[count++] = seq::span_of(name, &r, tokens, 1, d.width, dtype);
    return ok();
  }
  int kept(const char* codes, const char* scales, const to_rows8& r) {
    if (int st = seq::check_rows8(who, codes, r, tokens, d.width)) return st;
    wide = wide && aligned(r.codes, 8) && (tokens <= 1 || r.code_stride % 8 == 0);
    spans[count++] = seq::codes_span(codes, r, tokens, d.width);
    spans[count++] = seq::scales_span(scales, r, tokens, d.width);
    return ok();
  }
  int weight(const char* name, const float* w) {
    if (w && !aligned(w, 4)) return set_error(TO_ERR_ALIGNMENT, "%s: %s is not 4-byte aligned", who, name);
    wide = wide && aligned(w, 16);
    return ok();
  }
  // The first `outs` share no memory with the others, but for a row that is read where it is written.
  int apart(int outs, const char* written, const char* read) const {
    for (int i = 0; i < outs; ++i) {
      if (seq::meets_itself(spans[i])) return set_error(TO_ERR_INVALID_ARGUMENT, "%s: rows of %s share memory", who, spans[i].name);
      for (int j = i + 1; j < count; ++j) {
        const bool own = spans[i].name == written && spans[j].name == read && spans[i].p == spans[j].p && spans[i].ts == spans[j].ts;
        if (!own && seq::meet(spans[i], spans[j])) return seq::refuse_overlap(who, spans[i].name, spans[j].name);
      }
    }
    return ok();
  }
};

}  // namespace
}  // namespace to_b200

using namespace to_b200;

extern "C" {

int to_block_norm(const to_block_norm_desc* desc, int64_t tokens, const to_block_norm_args* args, void* stream) {
  const char* who = "to_block_norm";
  if (int st = check_desc(who, desc)) return st;
  if (!args) return set_error(TO_ERR_INVALID_ARGUMENT, "%s: null arguments", who);
  if (tokens < 0 || tokens > INT32_MAX)
    return set_error(TO_ERR_INVALID_ARGUMENT, "%s: %lld tokens", who, (long long)tokens);
  if (tokens == 0) return ok();
  const to_block_norm_desc& d = *desc;
  const to_block_norm_args& a = *args;
  const bool y = a.y.data, g = d.gate != TO_GATE_NONE && y;
  if (!y && (a.r_out.data || a.keep_y.codes || a.keep_g.codes || a.g.data))
    return set_error(TO_ERR_INVALID_ARGUMENT, "%s: r_out, g, keep_y or keep_g without y", who);
  if (y && !a.r_out.data) return set_error(TO_ERR_INVALID_ARGUMENT, "%s: r_out.data is null", who);
  if (!y && !a.n.data) return set_error(TO_ERR_INVALID_ARGUMENT, "%s: neither y nor n", who);
  if (d.gate == TO_GATE_NONE && (a.g.data || a.keep_g.codes))
    return set_error(TO_ERR_INVALID_ARGUMENT, "%s: g or keep_g without a gate", who);
  static const char kIn[] = "r", kOut[] = "r_out";
  RowSet S(who, d, tokens);
  int st = ok();
  if (y) st = S.rows(kOut, a.r_out, d.residual);
  if (!st && a.n.data) st = S.rows("n", a.n, d.dtype);
  if (!st && a.keep_r.codes) st = S.kept("keep_r.codes", "keep_r.scales", a.keep_r);
  if (!st && a.keep_y.codes) st = S.kept("keep_y.codes", "keep_y.scales", a.keep_y);
  if (!st && a.keep_g.codes) st = S.kept("keep_g.codes", "keep_g.scales", a.keep_g);
  const int outs = S.count;
  if (!st) st = S.rows(kIn, a.r, d.residual);
  if (!st && y) st = S.rows("y", a.y, d.dtype);
  if (!st && g) st = S.rows("g", a.g, d.dtype);
  if (!st) st = S.weight("w_post", a.w_post);
  if (!st) st = S.weight("w_pre", a.w_pre);
  if (!st) st = S.apart(outs, kOut, kIn);
  if (st) return st;
  ForwardArgs A{};
  A.r = seq::rows_of(a.r);
  A.y = seq::rows_of(a.y);
  A.g = seq::rows_of(a.g);
  A.r_out = seq::rows_of(a.r_out);
  A.n = seq::rows_of(a.n);
  A.keep_r = seq::packed_of(a.keep_r);
  A.keep_y = seq::packed_of(a.keep_y);
  A.keep_g = seq::packed_of(a.keep_g);
  A.w_post = a.w_post;
  A.w_pre = a.w_pre;
  A.tokens = tokens;
  A.width = d.width;
  A.gate = d.gate;
  A.post_norm = d.post_norm;
  A.scale = static_cast<float>(d.scale);
  A.eps = static_cast<float>(d.eps);
  int dev = 0;
  const int sms = device_sm_count(&dev);
  if (sms <= 0) return -sms;
  const Shape shape = shape_of(d.width);
  const unsigned grid = static_cast<unsigned>(std::min<long long>((tokens + shape.rows - 1) / shape.rows, 64ll * sms));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return each_kernel(d, S.wide, shape, [&](auto t, auto r, auto units, auto wide, auto most) {
    forward_kernel<decltype(t), decltype(r), decltype(units)::value, decltype(wide)::value, decltype(most)::value>
        <<<grid, dim3(shape.threads, shape.rows), 0, s>>>(A);
    TO_CUDA_TRY(cudaGetLastError());
    return ok();
  });
}

size_t to_block_norm_workspace_bytes(const to_block_norm_desc* desc, int64_t tokens) {
  if (check_desc("to_block_norm_workspace_bytes", desc) || tokens < 0) return 0;
  int dev = 0;
  const int sms = device_sm_count(&dev);
  return size_t(backward_ctas(desc->width, tokens, sms > 0 ? sms : 148)) * 2 * desc->width * sizeof(float);
}

int to_block_norm_backward(const to_block_norm_desc* desc, int64_t tokens, const to_block_norm_grad_args* args,
                           void* stream) {
  const char* who = "to_block_norm_backward";
  if (int st = check_desc(who, desc)) return st;
  if (!args) return set_error(TO_ERR_INVALID_ARGUMENT, "%s: null arguments", who);
  if (tokens < 0 || tokens > INT32_MAX)
    return set_error(TO_ERR_INVALID_ARGUMENT, "%s: %lld tokens", who, (long long)tokens);
  const to_block_norm_desc& d = *desc;
  const to_block_norm_grad_args& a = *args;
  const bool y = a.y.data || a.y8.codes, g = d.gate != TO_GATE_NONE && y;
  static const char kIn[] = "dr_out", kOut[] = "dr";
  RowSet S(who, d, tokens);
  if (!y && (a.g.data || a.g8.codes || a.dy.data || a.dg.data || a.dw_post) && tokens)
    return set_error(TO_ERR_INVALID_ARGUMENT, "%s: g, dy, dg or dw_post without y", who);
  if (d.gate == TO_GATE_NONE && (a.g.data || a.g8.codes || a.dg.data))
    return set_error(TO_ERR_INVALID_ARGUMENT, "%s: g or dg without a gate", who);
  int st = S.rows(kOut, a.dr, d.residual);
  if (!st && y) st = S.rows("dy", a.dy, d.dtype);
  if (!st && g) st = S.rows("dg", a.dg, d.dtype);
  const int outs = S.count;
  if (!st) st = a.r8.codes ? S.kept("r8.codes", "r8.scales", a.r8) : S.rows("r_out", a.r_out, d.residual);
  if (!st && y) st = a.y8.codes ? S.kept("y8.codes", "y8.scales", a.y8) : S.rows("y", a.y, d.dtype);
  if (!st && g) st = a.g8.codes ? S.kept("g8.codes", "g8.scales", a.g8) : S.rows("g", a.g, d.dtype);
  if (!st && a.dn.data) st = S.rows("dn", a.dn, d.dtype);
  if (!st && a.dr_out.data) st = S.rows(kIn, a.dr_out, d.residual);
  if (!st) st = S.weight("w_post", a.w_post);
  if (!st) st = S.weight("w_pre", a.w_pre);
  for (float* p : {a.dw_post, a.dw_pre})
    if (!st && p && !aligned(p, 4)) st = set_error(TO_ERR_ALIGNMENT, "%s: dw_post / dw_pre is not 4-byte aligned", who);
  if (!st && seq::arrays_meet(a.dw_post, a.dw_pre, d.width * sizeof(float))) st = seq::refuse_overlap(who, "dw_post", "dw_pre");
  if (!st && tokens) st = S.apart(outs, kOut, kIn);
  if (st) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int dev = 0;
  const int sms = device_sm_count(&dev);
  const int ctas = backward_ctas(d.width, tokens, sms > 0 ? sms : 148);
  const bool sums = a.dw_post || a.dw_pre;
  if (sums) {
    const size_t need = size_t(ctas) * 2 * d.width * sizeof(float);
    if (!a.workspace || a.workspace_bytes < need)
      return set_error(TO_ERR_INVALID_ARGUMENT, "%s: workspace %zu < %zu bytes", who, a.workspace ? a.workspace_bytes : 0, need);
    if (!aligned(a.workspace, 16)) return set_error(TO_ERR_ALIGNMENT, "%s: workspace is not 16-byte aligned", who);
  }
  if (sms <= 0) return -sms;
  BackwardArgs A{};
  A.r = seq::rows_of(a.r_out);
  A.y = seq::rows_of(a.y);
  A.g = seq::rows_of(a.g);
  A.dr_out = seq::rows_of(a.dr_out);
  A.dn = seq::rows_of(a.dn);
  A.dr = seq::rows_of(a.dr);
  A.dy = seq::rows_of(a.dy);
  A.dg = seq::rows_of(a.dg);
  A.r8 = seq::packed_of(a.r8);
  A.y8 = seq::packed_of(a.y8);
  A.g8 = seq::packed_of(a.g8);
  A.w_post = a.w_post;
  A.w_pre = a.w_pre;
  A.partial = sums ? static_cast<float*>(a.workspace) : nullptr;
  A.tokens = tokens;
  A.width = d.width;
  A.gate = d.gate;
  A.post_norm = d.post_norm;
  A.has_y = y;
  A.scale = static_cast<float>(d.scale);
  A.eps = static_cast<float>(d.eps);
  const Shape shape = shape_of(d.width);
  st = each_kernel(d, S.wide, shape, [&](auto t, auto r, auto units, auto wide, auto most) {
    constexpr int kUnits = decltype(units)::value, kMost = decltype(most)::value;
    constexpr size_t kColumns = size_t(2) * kUnits * kVals * sizeof(float);  // of a thread
    auto* kernel = backward_kernel<decltype(t), decltype(r), kUnits, decltype(wide)::value, kMost>;
    static std::atomic<uint64_t> done;
    if (int bad = seq::allow_shared(kernel, kColumns * kMost, done)) return bad;
    kernel<<<ctas, dim3(shape.threads, shape.rows), kColumns * shape.threads * shape.rows, s>>>(A);
    TO_CUDA_TRY(cudaGetLastError());
    return ok();
  });
  if (st || !sums) return st;
  weight_sum_kernel<<<dim3((d.width + 31) / 32, 2), 1024, 0, s>>>(A.partial, ctas, d.width, a.dw_pre, a.dw_post);
  TO_CUDA_TRY(cudaGetLastError());
  return ok();
}

}  // extern "C"

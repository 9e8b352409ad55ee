// qk_norm_rotary.cu -- norm of every query and key head and its rotation by
// position, one pass over the rows; and the pass's gradients.
//
//   forward   n = x r,  r = (mean x^2 + eps)^(-1/2),  y = R (w n)
//   backward  u = R^T g,  dw = sum u n,  d = w u,  dx = r (d - n mean(d n))
// R turns pair j of a row by positions[axis(j)] * theta^(-2j / rotary_dim).
//
// Memory bound: 8-16 flops for each value, which is read once and written
// once.  A pair's two values sit in one lane, so the rotation needs no
// exchange; `lanes` lanes hold a row (VP pairs a unit, 16-byte accesses where
// widths and addresses allow) and exchange only the row's sum.  A lane keeps
// its pairs (and their weights) over all the heads that it visits of one token,
// so their sines are computed once a token, by the warp's lanes together.
//
// Angles: a pair's frequency is a 64-bit fixed-point number of turns F =
// theta^(-2j/R) / 2 pi * 2^64, so position * F modulo 2^64 is the angle's
// fraction of a turn, exact but for F's own rounding (|position| * 2^-64
// turns).  Its top 32 bits go to sincospif.  A product of f32 values would
// lose the fraction at large positions (2^-24 * 100000 radians).
#include <cmath>
#include <cstring>
#include <new>

#include "sequence_common.cuh"

struct to_qk_plan {
  to_qk_desc desc;
  uint64_t turns[128];  // frequency of each pair, 2^-64 turns a position
};

namespace to_b200 {
namespace {

using seq::Rows;

constexpr int kMaxPairs = 128;
constexpr int kWarps = 8;  // warps a CTA

struct QkArgs {
  Rows in[2], g[2], out[2];  // q, k: x; gradients of y (backward); y or dx
  const float* w[2];
  float* partial;  // backward: [CTAs][dim] sums of u n
  const int32_t* positions;
  long long tokens;
  int heads[2];
  int dim, rotary, interleaved;
  float eps;
  int lanes;       // lanes that hold a row: a power of two
  int splits[2];   // warps that share a token's heads
  int units;       // pairs / VP
  int q_ctas;      // CTAs [0, q_ctas) take q, the others k
  int axis_end[4]; // first pair past each axis
  uint64_t turns[kMaxPairs];
};

// First elements of the two halves of the VP pairs that start at pair p (b is
// not used for neighbours).
struct Place {
  int a, b;
};

__device__ __forceinline__ Place place_of(const QkArgs& A, int p) {
  const int rot = A.rotary >> 1;
  if (A.interleaved) return {2 * p, 0};
  if (p < rot) return {p, p + rot};
  const int rest = (A.dim - A.rotary) >> 1;  // the part that does not turn, halved the same way
  return {A.rotary + p - rot, A.rotary + p - rot + rest};
}

template <typename T, int VP>
__device__ __forceinline__ void load_pairs(const T* row, const Place& pl, int interleaved,
                                           float (&a)[VP], float (&b)[VP]) {
  if (interleaved) {
    float t[2 * VP];
    seq::load_vec<T, 2 * VP>(row + pl.a, t);
#pragma unroll
    for (int i = 0; i < VP; ++i) {
      a[i] = t[2 * i];
      b[i] = t[2 * i + 1];
    }
  } else {
    seq::load_vec<T, VP>(row + pl.a, a);
    seq::load_vec<T, VP>(row + pl.b, b);
  }
}

template <typename T, int VP>
__device__ __forceinline__ void store_pairs(T* row, const Place& pl, int interleaved,
                                            const float (&a)[VP], const float (&b)[VP]) {
  if (interleaved) {
    float t[2 * VP];
#pragma unroll
    for (int i = 0; i < VP; ++i) {
      t[2 * i] = a[i];
      t[2 * i + 1] = b[i];
    }
    seq::store_vec<T, 2 * VP>(row + pl.a, t);
  } else {
    seq::store_vec<T, VP>(row + pl.a, a);
    seq::store_vec<T, VP>(row + pl.b, b);
  }
}

__device__ __forceinline__ float sum_over(float x, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// One warp takes a token's heads, or one of `splits` equal parts of them; in
// each step its 32 / lanes groups of lanes take HEADS heads each.  UPL units of
// VP pairs a lane.  SHARE groups (of those that there are) compute a token's
// sines together, VP / SHARE pairs each, and hand them round.
template <typename T, int VP, int UPL, int SHARE, int HEADS, bool BACKWARD>
__global__ void __launch_bounds__(32 * kWarps) qk_kernel(const __grid_constant__ QkArgs A) {
  extern __shared__ float sums[];  // backward: [kWarps][dim]
  constexpr int kOwn = VP / SHARE;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int groups = 32 / A.lanes, group = lane / A.lanes, gl = lane & (A.lanes - 1);
  const int t = static_cast<int>(blockIdx.x) >= A.q_ctas;  // q or k
  const int first_cta = t ? A.q_ctas : 0, ctas = t ? gridDim.x - A.q_ctas : A.q_ctas;
  const int heads = A.heads[t], splits = A.splits[t], rot = A.rotary >> 1, interleaved = A.interleaved;
  const float inv_dim = 1.f / static_cast<float>(A.dim), eps = A.eps;
  const Rows in = A.in[t], gr = A.g[t], out = A.out[t];
  bool on[UPL];
  Place pl[UPL];
  float wa[UPL][VP], wb[UPL][VP];
  uint64_t turn[UPL][kOwn];
  const int32_t* pos[UPL][kOwn];
  float dwa[BACKWARD ? UPL : 1][VP], dwb[BACKWARD ? UPL : 1][VP];
#pragma unroll
  for (int u = 0; u < UPL; ++u) {
    const int unit = gl + u * A.lanes;
    on[u] = unit < A.units;
    const int p0 = on[u] ? unit * VP : 0;
    pl[u] = place_of(A, p0);
#pragma unroll
    for (int i = 0; i < VP; ++i) {
      const int ia = pl[u].a + (interleaved ? 2 * i : i), ib = interleaved ? ia + 1 : pl[u].b + i;
      wa[u][i] = A.w[t] ? __ldg(A.w[t] + ia) : 1.f;
      wb[u][i] = A.w[t] ? __ldg(A.w[t] + ib) : 1.f;
      if (BACKWARD) dwa[BACKWARD ? u : 0][i] = dwb[BACKWARD ? u : 0][i] = 0.f;
    }
#pragma unroll
    for (int k = 0; k < kOwn; ++k) {
      const int p = p0 + k * SHARE + (group & (SHARE - 1));
      const int axis = (p >= A.axis_end[0]) + (p >= A.axis_end[1]) + (p >= A.axis_end[2]);
      const bool turns = on[u] && p < rot;  // the others stay: no position, no angle
      turn[u][k] = turns ? A.turns[p] : 0;
      pos[u][k] = turns ? A.positions + axis * A.tokens : nullptr;
    }
  }
  const long long items = A.tokens * splits, stride = static_cast<long long>(ctas) * kWarps;
  for (long long item = static_cast<long long>(blockIdx.x - first_cta) * kWarps + warp; item < items; item += stride) {
    const long long token = splits == 1 ? item : item / splits;
    const int part = splits == 1 ? 0 : static_cast<int>(item - token * splits);
    float c[UPL][VP], s[UPL][VP];
#pragma unroll
    for (int u = 0; u < UPL; ++u) {
      float oc[kOwn], os[kOwn];
#pragma unroll
      for (int k = 0; k < kOwn; ++k) {
        const long long x = pos[u][k] ? __ldg(pos[u][k] + token) : 0;
        const int top = static_cast<int>((static_cast<uint64_t>(x) * turn[u][k]) >> 32);  // [-1/2, 1/2) turns
        sincospif(static_cast<float>(top) * 4.656612873077393e-10f, &os[k], &oc[k]);
      }
#pragma unroll
      for (int i = 0; i < VP; ++i) {
        if (SHARE == 1) {
          c[u][i] = oc[i];
          s[u][i] = os[i];
        } else {  // pair i is made by the groups whose number is i modulo SHARE
          const int from = (i & (SHARE - 1)) * A.lanes + gl;
          c[u][i] = __shfl_sync(0xffffffffu, oc[i / SHARE], from);
          s[u][i] = __shfl_sync(0xffffffffu, os[i / SHARE], from);
        }
      }
    }
    // every lane of the warp takes every step (the sums are warp-wide)
    for (int h0 = part * groups * HEADS; h0 < heads; h0 += splits * groups * HEADS) {
      bool live[HEADS];
      float xa[HEADS][UPL][VP], xb[HEADS][UPL][VP];
      float ga[BACKWARD ? HEADS : 1][UPL][VP], gb[BACKWARD ? HEADS : 1][UPL][VP];
#pragma unroll
      for (int e = 0; e < HEADS; ++e) {
        const int h = h0 + e * groups + group;
        live[e] = h < heads;
        const T* xr = seq::row_ptr<const T>(in, token, live[e] ? h : 0);
        const T* gp = BACKWARD ? seq::row_ptr<const T>(gr, token, live[e] ? h : 0) : nullptr;
#pragma unroll
        for (int u = 0; u < UPL; ++u)
          if (on[u] && live[e]) {
            load_pairs<T, VP>(xr, pl[u], interleaved, xa[e][u], xb[e][u]);
            if (BACKWARD) load_pairs<T, VP>(gp, pl[u], interleaved, ga[BACKWARD ? e : 0][u], gb[BACKWARD ? e : 0][u]);
          } else {
#pragma unroll
            for (int i = 0; i < VP; ++i) {
              xa[e][u][i] = xb[e][u][i] = 0.f;
              if (BACKWARD) ga[BACKWARD ? e : 0][u][i] = gb[BACKWARD ? e : 0][u][i] = 0.f;
            }
          }
      }
#pragma unroll
      for (int e = 0; e < HEADS; ++e) {
        const int h = h0 + e * groups + group;
        float ss = 0.f;
#pragma unroll
        for (int u = 0; u < UPL; ++u)
#pragma unroll
          for (int i = 0; i < VP; ++i) ss = fmaf(xa[e][u][i], xa[e][u][i], fmaf(xb[e][u][i], xb[e][u][i], ss));
        ss = sum_over(ss, A.lanes);
        const float r = rsqrtf(ss * inv_dim + eps);
        T* row = seq::row_ptr<T>(out, token, live[e] ? h : 0);
        if (!BACKWARD) {
#pragma unroll
          for (int u = 0; u < UPL; ++u) {
            float ya[VP], yb[VP];
#pragma unroll
            for (int i = 0; i < VP; ++i) {
              const float a = xa[e][u][i] * (r * wa[u][i]), b = xb[e][u][i] * (r * wb[u][i]);
              ya[i] = a * c[u][i] - b * s[u][i];
              yb[i] = b * c[u][i] + a * s[u][i];
            }
            if (on[u] && live[e]) store_pairs<T, VP>(row, pl[u], interleaved, ya, yb);
          }
        } else {
          constexpr int kB = BACKWARD ? 1 : 0;
          float dot = 0.f;
#pragma unroll
          for (int u = 0; u < UPL; ++u)
#pragma unroll
            for (int i = 0; i < VP; ++i) {
              const float gx = ga[kB * e][u][i], gy = gb[kB * e][u][i];
              const float ua = gx * c[u][i] + gy * s[u][i], ub = gy * c[u][i] - gx * s[u][i];
              const float na = xa[e][u][i] * r, nb = xb[e][u][i] * r;
              dwa[kB * u][i] = fmaf(ua, na, dwa[kB * u][i]);
              dwb[kB * u][i] = fmaf(ub, nb, dwb[kB * u][i]);
              xa[e][u][i] = na;
              xb[e][u][i] = nb;
              ga[kB * e][u][i] = ua * wa[u][i];
              gb[kB * e][u][i] = ub * wb[u][i];
              dot = fmaf(ga[kB * e][u][i], na, fmaf(gb[kB * e][u][i], nb, dot));
            }
          const float m = sum_over(dot, A.lanes) * inv_dim;
#pragma unroll
          for (int u = 0; u < UPL; ++u) {
            float da[VP], db[VP];
#pragma unroll
            for (int i = 0; i < VP; ++i) {
              da[i] = r * (ga[kB * e][u][i] - xa[e][u][i] * m);
              db[i] = r * (gb[kB * e][u][i] - xb[e][u][i] * m);
            }
            if (on[u] && live[e]) store_pairs<T, VP>(row, pl[u], interleaved, da, db);
          }
        }
      }
    }
  }
  if (BACKWARD) {
    // groups of a warp, then warps of the CTA, in a fixed order
#pragma unroll
    for (int u = 0; u < UPL; ++u)
#pragma unroll
      for (int i = 0; i < VP; ++i) {
        float a = dwa[BACKWARD ? u : 0][i], b = dwb[BACKWARD ? u : 0][i];
        for (int o = A.lanes; o < 32; o <<= 1) {
          a += __shfl_xor_sync(0xffffffffu, a, o);
          b += __shfl_xor_sync(0xffffffffu, b, o);
        }
        if (group == 0 && on[u]) {
          float* row = sums + warp * A.dim;
          row[pl[u].a + (interleaved ? 2 * i : i)] = a;
          row[interleaved ? pl[u].a + 2 * i + 1 : pl[u].b + i] = b;
        }
      }
    __syncthreads();
    for (int e = threadIdx.x; e < A.dim; e += 32 * kWarps) {
      float v = 0.f;
      for (int w = 0; w < kWarps; ++w) v += sums[w * A.dim + e];
      A.partial[static_cast<long long>(blockIdx.x) * A.dim + e] = v;
    }
  }
}

// dw[e] = sum over CTAs of their partial sums, in a fixed order, in f64 (a few
// hundred terms: f32 would add as much rounding again as the terms have).  A
// warp takes one value of dwq or dwk, its lanes every 32nd CTA.
__global__ void __launch_bounds__(256) qk_sum_kernel(const float* __restrict__ partial, int q_ctas, int ctas,
                                                     int dim, float* dwq, float* dwk) {
  const int e = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (e >= 2 * dim) return;
  const bool q = e < dim;
  const int x = q ? e : e - dim, first = q ? 0 : q_ctas, last = q ? q_ctas : ctas;
  double v = 0;
#pragma unroll 8
  for (int c = first + lane; c < last; c += 32) v += partial[static_cast<long long>(c) * dim + x];
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  float* dst = q ? dwq : dwk;
  if (lane == 0 && dst) dst[x] = static_cast<float>(v);
}

// CTAs for q and for k, in proportion to their heads: `cap` CTAs in all, fewer
// where the warps would have no token.
struct QkGrid {
  int q, k;
};
QkGrid grid_of(const to_qk_desc& d, long long items_q, long long items_k, long long cap) {
  auto part = [&](long long heads, long long items) {
    if (!heads) return 0;
    const long long share = (cap * heads + d.q_heads + d.k_heads - 1) / (d.q_heads + d.k_heads);
    const long long want = (items + kWarps - 1) / kWarps;
    return static_cast<int>(want < 1 ? 1 : want < share ? want : share);
  };
  return {part(d.q_heads, items_q), part(d.k_heads, items_k)};
}

// Two CTAs of eight warps an SM hold the gradients' registers.
QkGrid backward_grid(const to_qk_desc& d, long long tokens, int sms) { return grid_of(d, tokens, tokens, 2ll * sms); }

template <typename T, int VP, int UPL, int SHARE>
int launch(QkArgs& A, const to_qk_desc& d, bool backward, int sms, cudaStream_t s) {
  if (backward) {
    const QkGrid g = backward_grid(d, A.tokens, sms);
    A.q_ctas = g.q;
    qk_kernel<T, VP, UPL, SHARE, 1, true><<<g.q + g.k, 32 * kWarps, size_t(kWarps) * A.dim * sizeof(float), s>>>(A);
  } else {
    const QkGrid g = grid_of(d, A.tokens * A.splits[0], A.tokens * A.splits[1], 32ll * sms);
    A.q_ctas = g.q;
    // two heads a step (more loads in flight) where a lane holds one unit
    qk_kernel<T, VP, UPL, SHARE, UPL == 1 ? 2 : 1, false><<<g.q + g.k, 32 * kWarps, 0, s>>>(A);
  }
  TO_CUDA_TRY(cudaGetLastError());
  return ok();
}

// VP: pairs of a unit.  16-byte accesses are VP 8 (bf16 halves), 4 (bf16
// neighbours, f32 halves) and 2 (f32 neighbours); widths or addresses that do
// not allow them go down to single pairs.
template <typename T>
int dispatch(QkArgs& A, const to_qk_desc& d, int vp, bool backward, int sms, cudaStream_t s) {
  const int pairs = A.dim / 2;
  A.units = pairs / vp;
  A.lanes = 1;
  while (A.lanes < 32 && A.lanes < A.units) A.lanes *= 2;
  const int upl = (A.units + A.lanes - 1) / A.lanes, groups = 32 / A.lanes;
  // warps that share a token's heads: one, unless the tokens are too few to give
  // every SM sixteen warps; then at most one a step of heads
  for (int t = 0; t < 2; ++t) {
    const long long steps = (A.heads[t] + groups - 1) / groups;
    long long n = backward || A.tokens == 0 ? 1 : (16ll * sms + A.tokens - 1) / A.tokens;
    A.splits[t] = static_cast<int>(n > steps ? (steps > 0 ? steps : 1) : n);
  }
  if (vp == 8 && sizeof(T) == 2)
    return groups >= 4 ? launch<__nv_bfloat16, 8, 1, 4>(A, d, backward, sms, s)
                       : launch<__nv_bfloat16, 8, 1, 2>(A, d, backward, sms, s);
  if (vp == 4)
    return groups >= 4   ? launch<T, 4, 1, 4>(A, d, backward, sms, s)
           : groups >= 2 ? launch<T, 4, 1, 2>(A, d, backward, sms, s)
                         : launch<T, 4, 1, 1>(A, d, backward, sms, s);
  if (vp == 2) {
    if (upl == 1) return launch<T, 2, 1, 1>(A, d, backward, sms, s);
    return launch<T, 2, 2, 1>(A, d, backward, sms, s);
  }
  if (upl == 1) return launch<T, 1, 1, 1>(A, d, backward, sms, s);
  if (upl == 2) return launch<T, 1, 2, 1>(A, d, backward, sms, s);
  return launch<T, 1, 4, 1>(A, d, backward, sms, s);
}

int run(const char* who, const to_qk_plan* plan, int64_t tokens, const to_rows* q, const to_rows* k,
        const int32_t* positions, const float* wq, const float* wk, const to_rows* gq,
        const to_rows* gk, const to_rows* oq, const to_rows* ok_, float* partial, cudaStream_t s) {
  const to_qk_desc& d = plan->desc;
  const bool backward = partial != nullptr;
  QkArgs A;
  const to_rows* in[2] = {q, k};
  const to_rows* gr[2] = {gq, gk};
  const to_rows* out[2] = {oq, ok_};
  const char* names[3][2] = {{"q", "k"}, {"gq", "gk"}, {"q_out", "k_out"}};
  if (backward) names[2][0] = "dq", names[2][1] = "dk";
  A.heads[0] = d.q_heads;
  A.heads[1] = d.k_heads;
  const int width = d.head_dim, half = d.rotary_dim / 2, rest = width / 2 - half;
  int vp = d.dtype == TO_BF16 ? (d.interleaved ? 4 : 8) : (d.interleaved ? 2 : 4);
  const to_rows none{nullptr, 0, 0};
  for (int t = 0; t < 2; ++t) {
    if (!A.heads[t]) {
      A.in[t] = A.g[t] = A.out[t] = seq::rows_of(none);
      continue;
    }
    int st = seq::check_rows(who, names[0][t], in[t], tokens, A.heads[t], width, d.dtype);
    if (!st && backward) st = seq::check_rows(who, names[1][t], gr[t], tokens, A.heads[t], width, d.dtype);
    if (!st) st = seq::check_rows(who, names[2][t], out[t], tokens, A.heads[t], width, d.dtype);
    if (st) return st;
    A.in[t] = seq::rows_of(*in[t]);
    A.g[t] = seq::rows_of(backward ? *gr[t] : none);
    A.out[t] = seq::rows_of(*out[t]);
  }
  A.w[0] = wq;
  A.w[1] = wk;
  for (const float* w : A.w)
    if (w && !aligned(w, 4)) return set_error(TO_ERR_ALIGNMENT, "%s: a weight is not 4-byte aligned", who);
  if (tokens > 0 && d.rotary_dim > 0 && !positions)
    return set_error(TO_ERR_INVALID_ARGUMENT, "%s: positions is null", who);
  if (positions && !aligned(positions, 4))
    return set_error(TO_ERR_ALIGNMENT, "%s: positions is not 4-byte aligned", who);
  if (tokens == 0 && !backward) return ok();
  // the widest unit that divides both parts of a row and that every address allows
  const int e = seq::dtype_bytes(d.dtype);
  auto fits = [&](int v) {
    if (d.interleaved ? (half % v || rest % v) : (half % v || rest % v || (2 * half) % v)) return false;
    const int bytes = (d.interleaved ? 2 : 1) * v * e > 16 ? 16 : (d.interleaved ? 2 : 1) * v * e;
    for (int t = 0; t < 2; ++t) {
      if (!A.heads[t] || tokens == 0) continue;
      if (!seq::rows_aligned(in[t], tokens, A.heads[t], d.dtype, bytes) ||
          !seq::rows_aligned(out[t], tokens, A.heads[t], d.dtype, bytes) ||
          (backward && !seq::rows_aligned(gr[t], tokens, A.heads[t], d.dtype, bytes)))
        return false;
    }
    return true;
  };
  while (vp > 1 && !fits(vp)) vp /= 2;
  if (vp == 1 && d.interleaved && !fits(1))
    return set_error(TO_ERR_ALIGNMENT, "%s: interleaved pairs must be aligned to a pair (%d bytes)", who, 2 * e);
  A.partial = partial;
  A.positions = positions;
  A.tokens = tokens;
  A.dim = width;
  A.rotary = d.rotary_dim;
  A.interleaved = d.interleaved;
  A.eps = static_cast<float>(d.eps);
  int end = 0;
  for (int a = 0; a < 4; ++a) {
    end += a < d.axes ? d.section[a] : 0;
    A.axis_end[a] = a < d.axes - 1 ? end : kMaxPairs + 1;
  }
  std::memcpy(A.turns, plan->turns, sizeof(A.turns));
  int dev = 0;
  const int sms = device_sm_count(&dev);
  if (sms <= 0) return -sms;
  return d.dtype == TO_BF16 ? dispatch<__nv_bfloat16>(A, d, vp, backward, sms, s)
                            : dispatch<float>(A, d, vp, backward, sms, s);
}

}  // namespace
}  // namespace to_b200

using namespace to_b200;

extern "C" {

int to_qk_plan_create(const to_qk_desc* desc, to_qk_plan** out) {
  if (!desc || !out) return set_error(TO_ERR_INVALID_ARGUMENT, "to_qk_plan_create: null");
  *out = nullptr;
  const to_qk_desc& d = *desc;
  if (d.dtype != TO_F32 && d.dtype != TO_BF16)
    return set_error(TO_ERR_UNSUPPORTED, "to_qk_plan_create: dtype %d (built: f32, bf16)", d.dtype);
  if (d.q_heads <= 0 || d.k_heads < 0 || d.q_heads > 65536 || d.k_heads > 65536)
    return set_error(TO_ERR_INVALID_ARGUMENT, "to_qk_plan_create: %d query and %d key heads", d.q_heads, d.k_heads);
  if (d.head_dim < 2 || d.head_dim > 2 * kMaxPairs || d.head_dim % 2)
    return set_error(TO_ERR_UNSUPPORTED, "to_qk_plan_create: head_dim %d (even, 2 .. 256)", d.head_dim);
  if (d.rotary_dim < 0 || d.rotary_dim > d.head_dim || d.rotary_dim % 2)
    return set_error(TO_ERR_INVALID_ARGUMENT, "to_qk_plan_create: rotary_dim %d of head_dim %d", d.rotary_dim, d.head_dim);
  if (d.interleaved != 0 && d.interleaved != 1)
    return set_error(TO_ERR_INVALID_ARGUMENT, "to_qk_plan_create: interleaved %d", d.interleaved);
  if (d.axes < 1 || d.axes > 4)
    return set_error(TO_ERR_INVALID_ARGUMENT, "to_qk_plan_create: %d axes (1 .. 4)", d.axes);
  long long pairs = 0;
  for (int a = 0; a < d.axes; ++a) {
    if (d.section[a] < 0) return set_error(TO_ERR_INVALID_ARGUMENT, "to_qk_plan_create: section %d is negative", a);
    pairs += d.section[a];
  }
  if (pairs != d.rotary_dim / 2)
    return set_error(TO_ERR_INVALID_ARGUMENT, "to_qk_plan_create: sections sum to %lld of %d pairs", pairs, d.rotary_dim / 2);
  if (!(d.theta > 0) || !std::isfinite(d.theta) || !(d.eps >= 0) || !std::isfinite(d.eps))
    return set_error(TO_ERR_INVALID_ARGUMENT, "to_qk_plan_create: theta %g, eps %g", d.theta, d.eps);
  to_qk_plan* p = new (std::nothrow) to_qk_plan{};
  if (!p) return set_error(TO_ERR_INVALID_ARGUMENT, "to_qk_plan_create: out of host memory");
  p->desc = d;
  const long double two_pi = 6.283185307179586476925286766559005768L;
  for (int j = 0; j < d.rotary_dim / 2; ++j) {
    const long double f = powl(static_cast<long double>(d.theta), -2.0L * j / d.rotary_dim) / two_pi;
    const long double frac = f - floorl(f);  // whole turns do not show at integer positions
    const long double scaled = frac * 18446744073709551616.0L;
    p->turns[j] = scaled >= 18446744073709551615.0L ? 0 : static_cast<uint64_t>(scaled + 0.5L);
  }
  *out = p;
  return ok();
}

int to_qk_plan_destroy(to_qk_plan* plan) {
  delete plan;
  return ok();
}

int to_qk_norm_rotary(const to_qk_plan* plan, int64_t tokens, const to_rows* q, const to_rows* k,
                      const int32_t* positions, const float* wq, const float* wk,
                      const to_rows* q_out, const to_rows* k_out, void* stream) {
  if (!plan) return set_error(TO_ERR_INVALID_ARGUMENT, "to_qk_norm_rotary: null plan");
  if (tokens < 0 || tokens > INT32_MAX)
    return set_error(TO_ERR_INVALID_ARGUMENT, "to_qk_norm_rotary: %lld tokens", (long long)tokens);
  return run("to_qk_norm_rotary", plan, tokens, q, k, positions, wq, wk, nullptr, nullptr, q_out, k_out,
             nullptr, static_cast<cudaStream_t>(stream));
}

size_t to_qk_norm_rotary_workspace_bytes(const to_qk_plan* plan, int64_t tokens) {
  if (!plan || tokens < 0) return 0;
  int dev = 0;
  const int sms = device_sm_count(&dev);
  const QkGrid g = backward_grid(plan->desc, tokens, sms > 0 ? sms : 148);
  return size_t(g.q + g.k) * plan->desc.head_dim * sizeof(float);
}

int to_qk_norm_rotary_backward(const to_qk_plan* plan, int64_t tokens, const to_rows* q,
                               const to_rows* k, const int32_t* positions, const float* wq,
                               const float* wk, const to_rows* gq, const to_rows* gk,
                               const to_rows* dq, const to_rows* dk, float* dwq, float* dwk,
                               void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "to_qk_norm_rotary_backward";
  if (!plan) return set_error(TO_ERR_INVALID_ARGUMENT, "%s: null plan", who);
  if (tokens < 0 || tokens > INT32_MAX)
    return set_error(TO_ERR_INVALID_ARGUMENT, "%s: %lld tokens", who, (long long)tokens);
  const size_t need = to_qk_norm_rotary_workspace_bytes(plan, tokens);
  if (!workspace || workspace_bytes < need)
    return set_error(TO_ERR_INVALID_ARGUMENT, "%s: workspace %zu < %zu bytes", who, workspace ? workspace_bytes : 0, need);
  if (!aligned(workspace, 16)) return set_error(TO_ERR_ALIGNMENT, "%s: workspace is not 16-byte aligned", who);
  for (float* p : {dwq, dwk})
    if (p && !aligned(p, 4)) return set_error(TO_ERR_ALIGNMENT, "%s: dwq / dwk is not 4-byte aligned", who);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  float* partial = static_cast<float*>(workspace);
  if (int st = run(who, plan, tokens, q, k, positions, wq, wk, gq, gk, dq, dk, partial, s)) return st;
  if (!dwq && !dwk) return ok();
  int dev = 0;
  const int sms = device_sm_count(&dev);
  if (sms <= 0) return -sms;
  const int dim = plan->desc.head_dim;
  const QkGrid g = backward_grid(plan->desc, tokens, sms);
  qk_sum_kernel<<<(2 * dim + 7) / 8, 256, 0, s>>>(partial, g.q, g.q + g.k, dim, dwq, dwk);
  TO_CUDA_TRY(cudaGetLastError());
  return ok();
}

}  // extern "C"

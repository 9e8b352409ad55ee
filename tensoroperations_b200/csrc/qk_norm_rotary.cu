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
// so their sines are computed once a token, by the warp's lanes together, and
// the next rows are on their way while it works (without that, 112 us for the
// first figure).
//
// Measured on B200: 16384 tokens x 40 heads x 128 bf16 in 65.6 us, 5.1 TB/s (0.79
// of the copy rate); 6137 x 24 x 96 f32, three axes, 26 us, 4.4 TB/s; gradients of
// 8192 x 40 x 128 bf16 in 69 us and 6 us for the weights' sums, 3.4 TB/s: two
// sums over a row, taken one after the other, which sixteen warps an SM do not hide.
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

// A unit of a row as it lies in memory, and as f32 values two to a register
// pair (the packed f32x2 instructions).  N pairs of halves or neighbours; where
// VP is odd (1) the second lane of a register pair is unused.
template <typename T, int VP>
struct Unit {
  static constexpr int kBytes = VP * int(sizeof(T));  // of one half
  static constexpr int kWords = kBytes < 4 ? 1 : kBytes / 4;
  static constexpr int kPacked = (VP + 1) / 2;
  uint32_t raw[2 * kWords];

  __device__ __forceinline__ void load(const T* row, const Place& pl, int interleaved) {
    if (interleaved) {
      read<2 * kBytes>(row + pl.a, raw);
    } else {
      read<kBytes>(row + pl.a, raw);
      read<kBytes>(row + pl.b, raw + kWords);
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 2 * kWords; ++i) raw[i] = 0;
  }
  // a: the pairs' first values, b: their second ones
  __device__ __forceinline__ void unpack(int interleaved, float2 (&a)[kPacked], float2 (&b)[kPacked]) const {
    float x[2 * VP];
#pragma unroll
    for (int i = 0; i < 2 * VP; ++i) {
      if (sizeof(T) == 4) {
        x[i] = __uint_as_float(raw[i % (2 * kWords)]);
      } else {
        // one value a half: each half has a word of its own (neighbours share the first)
        const uint32_t w = VP == 1 ? (interleaved ? raw[0] : raw[i]) : raw[i / 2];
        const bool high = VP == 1 ? interleaved && i == 1 : i & 1;
        x[i] = __uint_as_float(high ? w & 0xffff0000u : w << 16);
      }
    }
#pragma unroll
    for (int i = 0; i < kPacked; ++i) {
      const int j = 2 * i + 1 < VP ? 2 * i + 1 : 2 * i;
      a[i] = interleaved ? make_float2(x[4 * i], x[2 * j]) : make_float2(x[2 * i], x[j]);
      b[i] = interleaved ? make_float2(x[4 * i + 1], x[2 * j + 1]) : make_float2(x[VP + 2 * i], x[VP + j]);
    }
  }
  __device__ __forceinline__ static void store(T* row, const Place& pl, int interleaved, const float2 (&a)[kPacked],
                                               const float2 (&b)[kPacked]) {
    float x[VP], y[VP], t[2 * VP];
#pragma unroll
    for (int i = 0; i < VP; ++i) {
      x[i] = i & 1 ? a[i / 2].y : a[i / 2].x;
      y[i] = i & 1 ? b[i / 2].y : b[i / 2].x;
      t[2 * i] = x[i];
      t[2 * i + 1] = y[i];
    }
    if (interleaved) {
      seq::store_vec<T, 2 * VP>(row + pl.a, t);
    } else {
      seq::store_vec<T, VP>(row + pl.a, x);
      seq::store_vec<T, VP>(row + pl.b, y);
    }
  }

 private:
  template <int BYTES>
  __device__ __forceinline__ static void read(const T* p, uint32_t* dst) {
    if (BYTES == 2) {
      dst[0] = *reinterpret_cast<const uint16_t*>(p);
    } else if (BYTES == 4) {
      dst[0] = *reinterpret_cast<const uint32_t*>(p);
    } else if (BYTES == 8) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      dst[0] = v.x, dst[1] = v.y;
    } else {
#pragma unroll
      for (int i = 0; i < BYTES / 16; ++i) {
        const uint4 v = *(reinterpret_cast<const uint4*>(p) + i);
        dst[4 * i] = v.x, dst[4 * i + 1] = v.y, dst[4 * i + 2] = v.z, dst[4 * i + 3] = v.w;
      }
    }
  }
};

__device__ __forceinline__ float sum_over(float x, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// One warp takes a token's heads, or one of `splits` equal parts of them; in
// each step its 32 / lanes groups of lanes take HEADS heads each, and the next
// step's rows (the next token's, at the end) are on their way meanwhile.  UPL
// units of VP pairs a lane.  SHARE groups (of those that there are) compute a
// token's sines together, VP / SHARE pairs each, and hand them round.
// Forwards with four pairs a lane three CTAs fit an SM, with 80 registers a thread, of which
// some instantiations spill a few: with two it takes 104 us against 92 (16384 tokens x 40 heads x
// 128 bf16 neighbours) and 79 against 76 (16384 x 40 x 64 f32), as long at 128 f32, and 70
// against 73 at 4000 x 40 x 192 f32.
template <typename T, int VP, int UPL, int SHARE, int HEADS, bool BACKWARD>
__global__ void __launch_bounds__(32 * kWarps, VP == 4 && !BACKWARD ? 3 : 2) qk_kernel(const __grid_constant__ QkArgs A) {
  extern __shared__ float sums[];  // backward: [kWarps][dim]
  using U = Unit<T, VP>;
  constexpr int kOwn = VP / SHARE, kP = U::kPacked, kB = BACKWARD ? 1 : 0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int groups = 32 / A.lanes, group = lane / A.lanes, gl = lane & (A.lanes - 1);
  const int t = static_cast<int>(blockIdx.x) >= A.q_ctas;  // q or k
  const int first_cta = t ? A.q_ctas : 0, ctas = t ? gridDim.x - A.q_ctas : A.q_ctas;
  const int heads = A.heads[t], splits = A.splits[t], rot = A.rotary >> 1, interleaved = A.interleaved;
  const float inv_dim = 1.f / static_cast<float>(A.dim), eps = A.eps;
  const Rows in = A.in[t], gr = A.g[t], out = A.out[t];
  bool on[UPL];
  Place pl[UPL];
  float2 wa[UPL][kP], wb[UPL][kP];
  uint64_t turn[UPL][kOwn];
  const int32_t* pos[UPL][kOwn];
  float2 dwa[kB * (UPL - 1) + 1][kP], dwb[kB * (UPL - 1) + 1][kP];
#pragma unroll
  for (int u = 0; u < UPL; ++u) {
    const int unit = gl + u * A.lanes;
    on[u] = unit < A.units;
    const int p0 = on[u] ? unit * VP : 0;
    pl[u] = place_of(A, p0);
#pragma unroll
    for (int i = 0; i < kP; ++i) {
      const int j = 2 * i + 1 < VP ? 2 * i + 1 : 2 * i;
      auto weight = [&](int first, int k) {
        return A.w[t] ? __ldg(A.w[t] + first + (interleaved ? 2 * k : k)) : 1.f;
      };
      const int second = interleaved ? pl[u].a + 1 : pl[u].b;
      wa[u][i] = make_float2(weight(pl[u].a, 2 * i), weight(pl[u].a, j));
      wb[u][i] = make_float2(weight(second, 2 * i), weight(second, j));
      if (BACKWARD) dwa[kB * u][i] = dwb[kB * u][i] = make_float2(0.f, 0.f);
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
  long long item = static_cast<long long>(blockIdx.x - first_cta) * kWarps + warp;
  auto token_of = [&](long long i) { return splits == 1 ? i : i / splits; };
  auto first_of = [&](long long i) {  // first head of an item
    return splits == 1 ? 0 : static_cast<int>(i - i / splits * splits) * groups * HEADS;
  };
  U x[HEADS][UPL], g[kB * (HEADS - 1) + 1][UPL], nx[HEADS][UPL], ng[kB * (HEADS - 1) + 1][UPL];
  auto fetch = [&](U (&fx)[HEADS][UPL], U (&fg)[kB * (HEADS - 1) + 1][UPL], long long token, int h0) {
#pragma unroll
    for (int e = 0; e < HEADS; ++e) {
      const int h = h0 + e * groups + group;
      const T* xr = seq::row_ptr<const T>(in, token, h < heads ? h : 0);
      const T* gp = BACKWARD ? seq::row_ptr<const T>(gr, token, h < heads ? h : 0) : nullptr;
#pragma unroll
      for (int u = 0; u < UPL; ++u) {
        if (on[u] && h < heads) {
          fx[e][u].load(xr, pl[u], interleaved);
          if (BACKWARD) fg[kB * e][u].load(gp, pl[u], interleaved);
        } else {
          fx[e][u].clear();
          if (BACKWARD) fg[kB * e][u].clear();
        }
      }
    }
  };
  if (item < items) fetch(x, g, token_of(item), first_of(item));
  while (item < items) {
    const long long token = token_of(item), next = item + stride;
    float2 c[UPL][kP], s[UPL][kP];
#pragma unroll
    for (int u = 0; u < UPL; ++u) {
      float oc[kOwn], os[kOwn], cc[2 * kP], ss[2 * kP];
#pragma unroll
      for (int k = 0; k < kOwn; ++k) {
        const long long at = pos[u][k] ? __ldg(pos[u][k] + token) : 0;
        const int top = static_cast<int>((static_cast<uint64_t>(at) * turn[u][k]) >> 32);  // [-1/2, 1/2) turns
        sincospif(static_cast<float>(top) * 4.656612873077393e-10f, &os[k], &oc[k]);
      }
#pragma unroll
      for (int i = 0; i < 2 * kP; ++i) {
        if (SHARE == 1 || VP == 1) {
          cc[i] = oc[i % kOwn];
          ss[i] = os[i % kOwn];
        } else {  // pair i is made by the groups whose number is i modulo SHARE
          const int from = (i & (SHARE - 1)) * A.lanes + gl;
          cc[i] = __shfl_sync(0xffffffffu, oc[i / SHARE], from);
          ss[i] = __shfl_sync(0xffffffffu, os[i / SHARE], from);
        }
      }
#pragma unroll
      for (int i = 0; i < kP; ++i) {
        c[u][i] = make_float2(cc[2 * i], cc[2 * i + 1]);
        s[u][i] = make_float2(ss[2 * i], ss[2 * i + 1]);
      }
    }
    // every lane of the warp takes every step (the sums are warp-wide)
    const int step = splits * groups * HEADS;
    for (int h0 = first_of(item); h0 < heads; h0 += step) {
      if (h0 + step < heads) fetch(nx, ng, token, h0 + step);
      else if (next < items) fetch(nx, ng, token_of(next), first_of(next));
#pragma unroll
      for (int e = 0; e < HEADS; ++e) {
        const int h = h0 + e * groups + group;
        float2 xa[UPL][kP], xb[UPL][kP], sq = make_float2(0.f, 0.f);
#pragma unroll
        for (int u = 0; u < UPL; ++u) {
          x[e][u].unpack(interleaved, xa[u], xb[u]);
#pragma unroll
          for (int i = 0; i < kP; ++i) {
            if (VP == 1) xa[u][i].y = xb[u][i].y = 0.f;
            sq = __ffma2_rn(xa[u][i], xa[u][i], __ffma2_rn(xb[u][i], xb[u][i], sq));
          }
        }
        const float sum = sum_over(sq.x + sq.y, A.lanes);
        // (a group past the heads holds zeros, which without eps have no norm: they count as nothing)
        const float r = h < heads ? rsqrtf(sum * inv_dim + eps) : 0.f;
        const float2 r2 = make_float2(r, r);
        T* row = seq::row_ptr<T>(out, token, h < heads ? h : 0);
        if (!BACKWARD) {
#pragma unroll
          for (int u = 0; u < UPL; ++u) {
            float2 ya[kP], yb[kP];
#pragma unroll
            for (int i = 0; i < kP; ++i) {
              const float2 a = __fmul2_rn(xa[u][i], __fmul2_rn(r2, wa[u][i]));
              const float2 b = __fmul2_rn(xb[u][i], __fmul2_rn(r2, wb[u][i]));
              const float2 m = __fmul2_rn(b, s[u][i]);
              ya[i] = __ffma2_rn(a, c[u][i], make_float2(-m.x, -m.y));
              yb[i] = __ffma2_rn(b, c[u][i], __fmul2_rn(a, s[u][i]));
            }
            if (on[u] && h < heads) U::store(row, pl[u], interleaved, ya, yb);
          }
        } else {
          float2 da[UPL][kP], db[UPL][kP], dot = make_float2(0.f, 0.f);
#pragma unroll
          for (int u = 0; u < UPL; ++u) {
            float2 ga[kP], gb[kP];
            g[kB * e][u].unpack(interleaved, ga, gb);
#pragma unroll
            for (int i = 0; i < kP; ++i) {
              const float2 m = __fmul2_rn(ga[i], s[u][i]);
              const float2 ua = __ffma2_rn(ga[i], c[u][i], __fmul2_rn(gb[i], s[u][i]));
              const float2 ub = __ffma2_rn(gb[i], c[u][i], make_float2(-m.x, -m.y));
              xa[u][i] = __fmul2_rn(xa[u][i], r2);  // n
              xb[u][i] = __fmul2_rn(xb[u][i], r2);
              dwa[kB * u][i] = __ffma2_rn(ua, xa[u][i], dwa[kB * u][i]);
              dwb[kB * u][i] = __ffma2_rn(ub, xb[u][i], dwb[kB * u][i]);
              da[u][i] = __fmul2_rn(ua, wa[u][i]);
              db[u][i] = __fmul2_rn(ub, wb[u][i]);
              dot = __ffma2_rn(da[u][i], xa[u][i], __ffma2_rn(db[u][i], xb[u][i], dot));
            }
          }
          const float m = -sum_over(dot.x + dot.y, A.lanes) * inv_dim;
          const float2 m2 = make_float2(m, m);
#pragma unroll
          for (int u = 0; u < UPL; ++u) {
#pragma unroll
            for (int i = 0; i < kP; ++i) {
              da[u][i] = __fmul2_rn(r2, __ffma2_rn(xa[u][i], m2, da[u][i]));
              db[u][i] = __fmul2_rn(r2, __ffma2_rn(xb[u][i], m2, db[u][i]));
            }
            if (on[u] && h < heads) U::store(row, pl[u], interleaved, da[u], db[u]);
          }
        }
      }
#pragma unroll
      for (int e = 0; e < HEADS; ++e)
#pragma unroll
        for (int u = 0; u < UPL; ++u) {
          x[e][u] = nx[e][u];
          if (BACKWARD) g[kB * e][u] = ng[kB * e][u];
        }
    }
    item = next;
  }
  if (BACKWARD) {
    // groups of a warp, then warps of the CTA, in a fixed order
#pragma unroll
    for (int u = 0; u < UPL; ++u)
#pragma unroll
      for (int i = 0; i < VP; ++i) {
        float a = i & 1 ? dwa[kB * u][i / 2].y : dwa[kB * u][i / 2].x;
        float b = i & 1 ? dwb[kB * u][i / 2].y : dwb[kB * u][i / 2].x;
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
// hundred terms: f32 would add as much rounding again as the terms have).
// blockIdx.y: dwq or dwk; 32 values a CTA, every 32nd partial row a warp.
__global__ void __launch_bounds__(1024) qk_sum_kernel(const float* __restrict__ partial, int q_ctas, int ctas, int dim,
                                                      float* dwq, float* dwk) {
  __shared__ double part[32][33];
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5, x = blockIdx.x * 32 + lane;
  const int first = blockIdx.y ? q_ctas : 0, last = blockIdx.y ? ctas : q_ctas;
  double v = 0;
  if (x < dim) {
#pragma unroll 8
    for (int c = first + row; c < last; c += 32) v += partial[static_cast<long long>(c) * dim + x];
  }
  part[row][lane] = v;
  __syncthreads();
  float* dst = blockIdx.y ? dwk : dwq;
  if (row == 0 && x < dim && dst) {
    for (int k = 1; k < 32; ++k) v += part[k][lane];
    dst[x] = static_cast<float>(v);
  }
}

// CTAs for q and for k: `cap` CTAs in all, shared by the time that a token takes
// (its steps over four heads, and about two steps more for its sines), fewer
// where the warps would have no token.
struct QkGrid {
  int q, k;
};
QkGrid grid_of(const to_qk_desc& d, long long items_q, long long items_k, long long cap) {
  const long long cost_q = (d.q_heads + 3) / 4 + 2, cost_k = d.k_heads ? (d.k_heads + 3) / 4 + 2 : 0;
  auto part = [&](long long cost, long long items) {
    if (!cost) return 0;
    const long long share = (cap * cost + cost_q + cost_k - 1) / (cost_q + cost_k);
    const long long want = (items + kWarps - 1) / kWarps;
    return static_cast<int>(want < 1 ? 1 : want < share ? want : share);
  };
  return {part(cost_q, items_q), part(cost_k, items_k)};
}

// Heads that a group of lanes takes in one step of the forward pass: two (more loads in flight)
// where a lane holds one unit.
constexpr int forward_heads(int upl) { return upl == 1 ? 2 : 1; }

// Two CTAs of eight warps fit an SM; three rounds of them even out their lengths.
QkGrid backward_grid(const to_qk_desc& d, long long tokens, int sms) { return grid_of(d, tokens, tokens, 6ll * sms); }

template <typename T, int VP, int UPL, int SHARE>
int launch(QkArgs& A, const to_qk_desc& d, bool backward, int sms, cudaStream_t s) {
  if (backward) {
    const QkGrid g = backward_grid(d, A.tokens, sms);
    A.q_ctas = g.q;
    if constexpr (VP < 8)  // (gradients take four pairs at most)
      qk_kernel<T, VP, UPL, SHARE, VP == 4 ? 2 : 1, true>
          <<<g.q + g.k, 32 * kWarps, size_t(kWarps) * A.dim * sizeof(float), s>>>(A);
  } else {
    // eight CTAs an SM: a warp takes several tokens (its weights are read once, and the next
    // token's rows while it works), and the last ones still even out (72 us with 32, 87 with 2,
    // at 16384 tokens of 40 heads)
    const QkGrid g = grid_of(d, A.tokens * A.splits[0], A.tokens * A.splits[1], 8ll * sms);
    A.q_ctas = g.q;
    qk_kernel<T, VP, UPL, SHARE, forward_heads(UPL), false><<<g.q + g.k, 32 * kWarps, 0, s>>>(A);
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
  // every SM sixteen warps; then at most one a step of heads, so that each has a first
  // step (in its last one a warp fetches the rows of its next item)
  for (int t = 0; t < 2; ++t) {
    const int a_step = groups * forward_heads(upl);
    const long long steps = (A.heads[t] + a_step - 1) / a_step;
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
  int vp = d.dtype == TO_BF16 ? (d.interleaved ? 4 : 8) : 4;
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
  // a row is read by the lanes that write it: an output may be its own input, row for row, and
  // shares memory with nothing else
  seq::Span spans[6];
  int n = 0;
  for (const to_rows* const* set : {out, in, gr}) {
    if (set == gr && !backward) continue;
    for (int t = 0; t < 2; ++t, ++n)
      spans[n] = A.heads[t] ? seq::span_of(names[set == out ? 2 : set == in ? 0 : 1][t], set[t], tokens, A.heads[t],
                                           width, d.dtype)
                            : seq::Span{};
  }
  for (int t = 0; t < 2 && tokens > 0; ++t) {
    const seq::Span& o = spans[t];
    if (!o.heads) continue;
    if (seq::meets_itself(o)) return set_error(TO_ERR_INVALID_ARGUMENT, "%s: rows of %s share memory", who, o.name);
    for (int j = t + 1; j < n; ++j) {
      const seq::Span& x = spans[j];
      const bool own = j > 1 && j % 2 == t && x.p == o.p && x.ts == o.ts && x.hs == o.hs;
      if (!own && seq::meet(o, x)) return seq::refuse_overlap(who, o.name, x.name);
    }
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
  // (gradients hold twice the rows: four pairs a lane and two heads a step, 68 us against 77
  // with eight pairs and one head at 8192 tokens of 40 heads)
  if (backward && vp == 8) vp = 4;
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
  qk_sum_kernel<<<dim3((dim + 31) / 32, 2), 1024, 0, s>>>(partial, g.q, g.q + g.k, dim, dwq, dwk);
  TO_CUDA_TRY(cudaGetLastError());
  return ok();
}

}  // extern "C"

// linear_attention.cu -- linear attention with a decay for each head: the
// chunked form and its gradients (one chain, linear_attention.cuh) on the CUDA
// cores, the segment scan, the single-token step, and the C-ABI entries.
#include <algorithm>
#include <cmath>

#include "linear_attention.cuh"

namespace to_b200 {
namespace {

using lin::Chain;
using lin::Segment;
using seq::Rows;

constexpr int kMaxDim = 256;

// ---- the chain on the CUDA cores ---------------------------------------------------
// f32 rows, and bf16 rows whose widths or addresses the tensor-core form does
// not take.  One CTA: one segment, one head, DCB columns of c.  Chunks of 64
// tokens: P = (a b^T) masked and decayed, out = P c + decay (a X), then X, all
// in f32 in shared memory, 4 x 4 results a thread.  At most 128 flops come
// from 8 16-byte shared loads, so the shared-memory pipe bounds it at about
// half of the f32 rate.  Measured on B200: 2500 tokens x 12 heads x 64 f32 in
// 74 us with its states' launch and scan (49 us the outputs).  Each segment is
// cut to about two chunks there, and waiting for rows, shared memory and the
// other warps takes as long as the sums.
constexpr int kRows = 64;  // tokens of a chunk
constexpr int kThreads = 256;

template <int DCB>
struct SimtShape {
  static constexpr int kColPad = DCB + 4;
  static size_t bytes(int dbp) {
    return sizeof(float) * (2 * size_t(kRows) * (dbp + 4) + size_t(kRows) * kColPad +
                            size_t(kRows) * (kRows + 4) + size_t(dbp) * kColPad + 2 * (kRows + 4));
  }
};

// Rows of a chunk into shared memory as f32, four columns a thread; rows past
// cnt and columns past width become zero.  `vec`: four columns are one access.
// Whether this thread met an infinity or a NaN.
template <typename T>
__device__ __forceinline__ bool load_rows(float* dst, int ld, const Rows& r, int head, int row0, int step, int cnt,
                                          int first, int width, int padded, bool vec) {
  int lanes = 8;  // threads of a row: a power of two
  while (lanes * 4 < padded) lanes *= 2;
  const int x = (threadIdx.x & (lanes - 1)) * 4;
  if (x >= padded) return false;
  float odd = 0.f;  // 0 times each value: 0 while all are finite
  const T* src = seq::row_ptr<const T>(r, row0, head) + first + x;
  const long long hop = static_cast<long long>(step) * r.ts;
#pragma unroll 4
  for (int i = threadIdx.x / lanes; i < kRows; i += kThreads / lanes) {
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (i < cnt) {
      const T* p = src + i * hop;
      if (vec && x + 4 <= width) {
        seq::load_vec<T, 4>(p, v);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (x + e < width) v[e] = seq::to_f32(p[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) odd = fmaf(0.f, v[e], odd);
    *reinterpret_cast<float4*>(dst + i * ld + x) = make_float4(v[0], v[1], v[2], v[3]);
  }
  return !(odd == 0.f);
}

template <typename T, int DCB, bool STATES, int N>
__global__ void __launch_bounds__(kThreads) chain_simt_kernel(const __grid_constant__ lin::Batch<N> batch) {
  const Chain& C = batch.c[blockIdx.y % N];
  constexpr int kColPad = SimtShape<DCB>::kColPad;
  constexpr int VC = DCB / 16;  // columns of a thread
  const Segment g = lin::segment_of(C, blockIdx.x);
  if (g.idx < 0 || (STATES && g.idx == g.count - 1)) return;
  const int head = blockIdx.z, col0 = blockIdx.y / N * DCB;
  if (col0 >= C.dc) return;
  const int dbp = (C.db + 3) & ~3, lda = dbp + 4;
  extern __shared__ __align__(16) float sm[];
  float* A = sm;
  float* B = A + kRows * lda;
  float* V = B + kRows * lda;
  float* P = V + kRows * kColPad;
  float* X = P + kRows * (kRows + 4);
  float* dec = X + dbp * kColPad;  // l^n, n = 0 .. kRows
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  const int ncols = min(DCB, C.dc - col0);
  const float gl = lin::log_decay_of(C, head);
  if (tid <= kRows) dec[tid] = expf(gl * static_cast<float>(tid));

  // entering X
  const long long slot = lin::state_slot(C, g.seq);
  const float* src = nullptr;
  int src_t = 0;
  if (!STATES) {
    if (g.count > 1) {
      src = C.seg_state + (static_cast<long long>(blockIdx.x) * C.heads + head) * C.db * C.dc;
    } else if (C.init && slot >= 0) {
      src = C.init + (slot * C.heads + head) * C.db * C.dc;
      src_t = C.init_t;
    }
  }
  for (int e = tid; e < dbp * DCB; e += kThreads) {
    const int b = e / DCB, c = e - b * DCB;
    X[b * kColPad + c] =
        src && b < C.db && c < ncols ? src[lin::state_index(C, src_t, b, col0 + c)] : 0.f;
  }

  const int s0 = g.idx * C.seg, len = min(C.seg, g.tokens - s0);
  const int step = C.rev ? -1 : 1;
  for (int done = 0; done < len; done += kRows) {
    const int cnt = min(kRows, len - done), t = s0 + done;
    const int row0 = C.rev ? g.first + g.tokens - 1 - t : g.first + t;
    __syncthreads();  // the last chunk's readers are done
    if (!STATES) load_rows<T>(A, lda, C.a, head / C.a_div, row0, step, cnt, 0, C.db, dbp, C.vec & 1);
    load_rows<T>(B, lda, C.b, head / C.b_div, row0, step, cnt, 0, C.db, dbp, C.vec & 2);
    const bool met = load_rows<T>(V, kColPad, C.c, head / C.c_div, row0, step, cnt, col0, ncols, DCB, C.vec & 4);
    // a value of V that is not finite may not meet the zeros of P: 0 * inf is not 0
    const bool masked = STATES ? (__syncthreads(), false) : __syncthreads_or(met);
    if (!STATES) {
      float acc[4][4] = {};
      for (int k = 0; k < dbp; k += 4) {
        float4 x[4], y[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          x[r] = *reinterpret_cast<const float4*>(A + (ty + 16 * r) * lda + k);
          y[r] = *reinterpret_cast<const float4*>(B + (tx + 16 * r) * lda + k);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int q = 0; q <= r; ++q)  // (rows 16 r .. see no columns past 16 r + 15)
            acc[r][q] = fmaf(x[r].w, y[q].w, fmaf(x[r].z, y[q].z, fmaf(x[r].y, y[q].y, fmaf(x[r].x, y[q].x, acc[r][q]))));
      }
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int i = ty + 16 * r, j = tx + 16 * q;
          P[i * (kRows + 4) + j] = j <= i && j < cnt ? acc[r][q] * dec[i - j] * C.intra : 0.f;
        }
      __syncthreads();
      // out = P V + inter * l^(i+1-rev) A X
      float o[4][VC] = {}, w[4][VC] = {};
      if (masked) {
        for (int j = 0; j < cnt; ++j) {
          float v[VC];
          seq::load_vec<float, VC>(V + j * kColPad + tx * VC, v);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if (ty + 16 * r < j) continue;
            const float pv = P[(ty + 16 * r) * (kRows + 4) + j];
#pragma unroll
            for (int c = 0; c < VC; ++c) o[r][c] = fmaf(pv, v[c], o[r][c]);
          }
        }
      } else {
#pragma unroll
        for (int block = 0; block < 4; ++block)  // 16 columns of P: rows from 16 block on see them
#pragma unroll 1
          for (int j = 16 * block; j < 16 * block + 16; j += 4) {
            float4 p[4];
#pragma unroll
            for (int r = block; r < 4; ++r)
              p[r] = *reinterpret_cast<const float4*>(P + (ty + 16 * r) * (kRows + 4) + j);
#pragma unroll
            for (int jj = 0; jj < 4; ++jj) {
              float v[VC];
              seq::load_vec<float, VC>(V + (j + jj) * kColPad + tx * VC, v);
#pragma unroll
              for (int r = block; r < 4; ++r) {
                const float pv = jj == 0 ? p[r].x : jj == 1 ? p[r].y : jj == 2 ? p[r].z : p[r].w;
#pragma unroll
                for (int c = 0; c < VC; ++c) o[r][c] = fmaf(pv, v[c], o[r][c]);
              }
            }
          }
      }
      for (int k = 0; k < dbp; k += 4) {
        float4 p[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) p[r] = *reinterpret_cast<const float4*>(A + (ty + 16 * r) * lda + k);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          float v[VC];
          seq::load_vec<float, VC>(X + (k + kk) * kColPad + tx * VC, v);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float pv = kk == 0 ? p[r].x : kk == 1 ? p[r].y : kk == 2 ? p[r].z : p[r].w;
#pragma unroll
            for (int c = 0; c < VC; ++c) w[r][c] = fmaf(pv, v[c], w[r][c]);
          }
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = ty + 16 * r;
        if (i >= cnt) continue;
        const long long token = row0 + static_cast<long long>(step) * i;
        const float f = C.inter * dec[i + 1 - C.rev];
#pragma unroll
        for (int c = 0; c < VC; ++c) {
          const int x = tx * VC + c;
          const float v = fmaf(f, w[r][c], o[r][c]);
          if (x >= ncols) continue;
          if (C.out_f32) seq::row_ptr<float>(C.out, token, head)[col0 + x] = v;
          else seq::row_ptr<T>(C.out, token, head)[col0 + x] = seq::from_f32<T>(v);
        }
      }
      __syncthreads();  // X has been read
    }
    // X = l^cnt X + upd * sum_j l^(cnt-1+rev-j) b_j c_j
    const float keep = dec[cnt];
    // (a thread: rows k .. k+3 and k+64 .. k+67 at a time, so V is read half as often)
    for (int k0 = 0; k0 < dbp; k0 += 128) {
      const int k[2] = {k0 + ty * 4, k0 + 64 + ty * 4};
      const bool on[2] = {k[0] < dbp, k[1] < dbp};
      if (!on[0]) continue;
      float u[2][4][VC] = {};
#pragma unroll 4
      for (int j = 0; j < cnt; ++j) {
        const float d = C.upd * dec[cnt - 1 + C.rev - j];
        float v[VC];
        seq::load_vec<float, VC>(V + j * kColPad + tx * VC, v);
#pragma unroll
        for (int c = 0; c < VC; ++c) v[c] *= d;
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          if (!on[z]) continue;
          float b[4];
          seq::load_vec<float, 4>(B + j * lda + k[z], b);
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int c = 0; c < VC; ++c) u[z][r][c] = fmaf(b[r], v[c], u[z][r][c]);
        }
      }
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        if (!on[z]) continue;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int c = 0; c < VC; ++c) {
            float* x = X + (k[z] + r) * kColPad + tx * VC + c;
            *x = fmaf(keep, *x, u[z][r][c]);
          }
      }
    }
  }
  __syncthreads();
  float* dst = nullptr;
  if (STATES) {
    dst = C.seg_state + (static_cast<long long>(blockIdx.x) * C.heads + head) * C.db * C.dc;
  } else if (C.fin && slot >= 0 && g.idx == g.count - 1) {
    dst = C.fin + (slot * C.heads + head) * C.db * C.dc;
  }
  if (dst)
    for (int e = tid; e < C.db * DCB; e += kThreads) {
      const int b = e / DCB, c = e - b * DCB;
      if (c < ncols) dst[lin::state_index(C, 0, b, col0 + c)] = X[b * kColPad + c];
    }
}

// ---- scan over the segments ---------------------------------------------------------
// In place: slot s holds segment s's own X (the last one's is not read) and
// gets the X that enters it.  Sequences of one segment have nothing to scan.
// A thread follows VEC values; the next kAhead segments are on their way while
// one group is written, so a long sequence is not one memory latency a segment.
template <int VEC, int N>
__global__ void __launch_bounds__(256) chain_scan_kernel(const __grid_constant__ lin::Batch<N> batch) {
  const Chain& C = batch.c[blockIdx.x % N];
  constexpr int kAhead = 8;
  const int s = blockIdx.z, head = blockIdx.y;
  const Segment g = lin::sequence_of(C, s);
  const int w0 = lin::first_slot(C, s);
  const int n = C.db * C.dc, e = (blockIdx.x / N * 256 + threadIdx.x) * VEC;
  const int slots = lin::segment_slots(C.tokens, C.nseq, C.seg);
  const int count = min(g.count, slots - w0);
  if (count < 2 || e >= n) return;
  const long long slot = lin::state_slot(C, s);
  float x[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    x[v] = 0.f;
    if (C.init && slot >= 0)
      x[v] = C.init[(slot * C.heads + head) * n + lin::state_index(C, C.init_t, (e + v) / C.dc, (e + v) % C.dc)];
  }
  const float keep = expf(lin::log_decay_of(C, head) * static_cast<float>(C.seg));
  const long long hop = static_cast<long long>(C.heads) * n;
  float* p = C.seg_state + (static_cast<long long>(w0) * C.heads + head) * n + e;
  float own[kAhead][VEC];
#pragma unroll
  for (int j = 0; j < kAhead; ++j)
    if (j < count - 1) seq::load_vec<float, VEC>(p + j * hop, own[j]);
  for (int i = 0; i < count; i += kAhead)
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (i + j >= count) break;
      seq::store_vec<float, VEC>(p + (i + j) * hop, x);
#pragma unroll
      for (int v = 0; v < VEC; ++v) x[v] = fmaf(keep, x[v], own[j][v]);
      if (i + j + kAhead < count - 1) seq::load_vec<float, VEC>(p + (i + j + kAhead) * hop, own[j]);
    }
}

// ---- shared heads: sum the gradients of the heads of a group ---------------------------
// blockIdx.y: dk or dv.  Packed sequences lie between the first and the last of their bounds;
// the chains have written no other rows, and none are summed.
struct GroupSum {
  const float* part[2];
  Rows out[2];
  int width[2];
  const int32_t* cu;
  int nseq, tokens;
  int kv_heads, group;
};

template <typename T>
__global__ void __launch_bounds__(256) group_sum_kernel(const __grid_constant__ GroupSum G) {
  const int y = blockIdx.y, width = G.width[y];
  const long long per = static_cast<long long>(G.kv_heads) * width;
  const int first = min(max(__ldg(G.cu), 0), G.tokens), last = min(max(__ldg(G.cu + G.nseq), 0), G.tokens);
  for (long long e = first * per + blockIdx.x * 256ll + threadIdx.x; e < last * per; e += gridDim.x * 256ll) {
    const long long t = e / per;
    const int r = static_cast<int>(e - t * per), h = r / width, x = r - h * width;
    const float* p = G.part[y] + ((t * G.kv_heads + h) * G.group) * width + x;
    float v = 0.f;
    for (int i = 0; i < G.group; ++i) v += p[static_cast<long long>(i) * width];
    seq::row_ptr<T>(G.out[y], t, h)[x] = seq::from_f32<T>(v);
  }
}

// ---- one token of each request ------------------------------------------------------------
// Memory bound: the state is read and written once, 8 bytes a value, for 4
// flops.  A CTA takes `cols` columns of one request's head; a lane holds VEC
// consecutive columns and walks the rows of the state, kUnroll of them in flight.
// Measured on B200: 192 requests x 32 heads x 128 x 128 in 129 us, 6.3 TB/s (0.97
// of the copy rate).
struct StepArgs {
  Rows q, k, v, o;
  const float* log_decay;
  const int32_t* slots;
  float* state;
  long long num_slots;
  int heads, group, dk, dv, cols;
  float scale;
};

constexpr int kStepThreads = 128;
constexpr int kUnroll = 8;

template <typename T, int VEC>
__global__ void __launch_bounds__(kStepThreads) step_kernel(const __grid_constant__ StepArgs A) {
  __shared__ float sq[kMaxDim], sk[kMaxDim];
  __shared__ float part[kStepThreads * VEC];
  const int head = blockIdx.y, col0 = blockIdx.z * A.cols;
  const long long req = blockIdx.x;
  const int lanes = A.cols / VEC;  // a power of two, at most the CTA
  const int row = threadIdx.x / lanes, cl = threadIdx.x - row * lanes, rows = kStepThreads / lanes;
  const int c = col0 + cl * VEC;
  long long slot = A.slots ? static_cast<long long>(__ldg(A.slots + req)) : req;
  if (slot < 0 || slot >= A.num_slots) slot = -1;
  const T* q = seq::row_ptr<const T>(A.q, req, head);
  const T* k = seq::row_ptr<const T>(A.k, req, head / A.group);
  for (int i = threadIdx.x; i < A.dk; i += kStepThreads) {
    sq[i] = seq::to_f32(q[i]);
    sk[i] = seq::to_f32(k[i]);
  }
  const bool on = c < A.dv;
  float v[VEC], acc[VEC];
#pragma unroll
  for (int x = 0; x < VEC; ++x) v[x] = acc[x] = 0.f;
  if (on) {
    const T* vr = seq::row_ptr<const T>(A.v, req, head / A.group) + c;
#pragma unroll
    for (int x = 0; x < VEC; ++x) v[x] = seq::to_f32(vr[x]);
  }
  const float g = __ldg(A.log_decay + head);
  const float l = expf(g > 0.f ? 0.f : g);
  __syncthreads();
  if (on && slot >= 0) {
    float* S = A.state + (slot * A.heads + head) * static_cast<long long>(A.dk) * A.dv + c;
    for (int r0 = row; r0 < A.dk; r0 += rows * kUnroll) {
      float s[kUnroll][VEC];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int r = r0 + u * rows;
        if (r < A.dk) seq::load_vec<float, VEC>(S + static_cast<long long>(r) * A.dv, s[u]);
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int r = r0 + u * rows;
        if (r < A.dk) {
#pragma unroll
          for (int x = 0; x < VEC; ++x) {
            s[u][x] = fmaf(l, s[u][x], sk[r] * v[x]);
            acc[x] = fmaf(sq[r], s[u][x], acc[x]);
          }
          seq::store_vec<float, VEC>(S + static_cast<long long>(r) * A.dv, s[u]);
        }
      }
    }
  }
#pragma unroll
  for (int x = 0; x < VEC; ++x) part[threadIdx.x * VEC + x] = acc[x];
  __syncthreads();
  for (int x = threadIdx.x; x < A.cols; x += kStepThreads)
    if (col0 + x < A.dv) {
      float o = 0.f;
      for (int r = 0; r < rows; ++r) o += part[r * A.cols + x];
      seq::row_ptr<T>(A.o, req, head)[col0 + x] = seq::from_f32<T>(A.scale * o);
    }
}

// ---- host ------------------------------------------------------------------------------------

int check_desc(const char* who, const to_linear_attention_desc* d) {
  if (!d) return set_error(TO_ERR_INVALID_ARGUMENT, "%s: null descriptor", who);
  if (d->dtype != TO_F32 && d->dtype != TO_BF16)
    return set_error(TO_ERR_UNSUPPORTED, "%s: dtype %d (built: f32, bf16)", who, d->dtype);
  if (d->q_heads <= 0 || d->kv_heads <= 0 || d->q_heads > 65535 || d->q_heads % d->kv_heads)
    return set_error(TO_ERR_INVALID_ARGUMENT, "%s: %d query heads on %d key heads", who, d->q_heads, d->kv_heads);
  if (d->key_dim < 1 || d->key_dim > kMaxDim || d->value_dim < 1 || d->value_dim > kMaxDim)
    return set_error(TO_ERR_UNSUPPORTED, "%s: key_dim %d, value_dim %d (1 .. 256)", who, d->key_dim, d->value_dim);
  if (d->tokens < 0 || d->tokens > INT32_MAX || d->nseq < 0 || d->nseq > 65535 || d->num_slots < 0)
    return set_error(TO_ERR_INVALID_ARGUMENT, "%s: %lld tokens, %d sequences, %lld slots", who,
                     (long long)d->tokens, d->nseq, (long long)d->num_slots);
  if (!std::isfinite(d->scale)) return set_error(TO_ERR_INVALID_ARGUMENT, "%s: scale %g", who, d->scale);
  return ok();
}

int check_state(const char* who, const char* name, const void* p) {
  if (p && !aligned(p, 16)) return set_error(TO_ERR_ALIGNMENT, "%s: %s is not 16-byte aligned", who, name);
  return ok();
}

int check_list(const char* who, const char* name, const void* p, bool need) {
  if (need && !p) return set_error(TO_ERR_INVALID_ARGUMENT, "%s: %s is null", who, name);
  if (p && !aligned(p, 4)) return set_error(TO_ERR_ALIGNMENT, "%s: %s is not 4-byte aligned", who, name);
  return ok();
}

// Tokens of a segment, from what the host knows: the tokens, the sequences and
// the heads (taken for sequences of equal length).  Among cuts of a sequence
// into k segments, the one with the least estimated time, in quarters of what a
// chunk's outputs take: rounds of items over the CTAs that run at a time, a chunk
// 4 in the outputs' launch and `states` in the states', an item `begin` to begin,
// the scan and its launch 6 and what its bytes cost, and a quarter of an item
// for SMs that come out late.  Real lengths differ, so a segment is also at most
// an SM's share of all chunks (half of it on the CUDA cores, where a chunk takes
// long): one long sequence among short ones is cut too.  One segment for all
// where no sequence can be longer than one.
// Tensor cores: chunks of 128 tokens (about 4 us), one CTA an SM.  CUDA cores:
// chunks of 64 (about 20 us), one CTA for each 64 or 32 columns; narrow rows
// leave shared memory for two an SM.
constexpr int kOneSegment = 1 << 30;

int plan_segment(const to_linear_attention_desc& d, bool tc, int chains) {
  const int db = chains > 1 ? std::max(d.key_dim, d.value_dim) : d.key_dim;
  const int dc = chains > 1 ? db : d.value_dim;
  const long long chunk = tc ? 128 : kRows, states = tc ? 2 : 1, begin = tc ? 3 : 2;
  const long long at_once = 148 * (!tc && db <= 64 ? 2 : 1);
  const long long blocks = chains * (tc ? 1ll : db <= 128 ? (dc + 63) / 64 : (dc + 31) / 32);
  const long long chunks = (d.tokens + chunk - 1) / chunk, pairs = d.nseq * blocks * d.q_heads;
  if (chunks <= 2 || pairs == 0) return kOneSegment;
  const long long mean = std::max(1ll, (chunks + d.nseq - 1) / d.nseq);
  long long best = mean, least = INT64_MAX;
  for (long long k = 1; k <= 64 && k <= mean; ++k) {
    const long long per = (mean + k - 1) / k;
    long long cost = at_once * (((pairs * k + at_once - 1) / at_once) * (4 * per + begin) + per);
    if (k > 1)
      cost += at_once * (((pairs * (k - 1) + at_once - 1) / at_once) * (states * per + begin) + 6) + 4 * pairs * k;
    if (cost < least) least = cost, best = per;
  }
  const long long load = (chunks * blocks * d.q_heads + at_once - 1) / at_once;
  const long long share = std::max(tc ? 4ll : 2ll, tc ? load : (load + 1) / 2);
  if (tc && best == mean) best = std::max(best, std::min(chunks, 2 * mean));  // ragged ones stay whole too
  best = std::min(best, std::max(share, mean / 64 + 1));
  return best >= chunks ? kOneSegment : static_cast<int>(best * chunk);
}

// The rows of a prompt or of single tokens: o is written while others read q, k and v.
int check_outputs(const char* who, const to_linear_attention_desc& d, const to_linear_attention_args& a) {
  auto span = [&](const char* name, const to_rows& r, int heads, int width) {
    return seq::span_of(name, &r, d.tokens, heads, width, d.dtype);
  };
  const seq::Span rows[] = {span("o", a.o, d.q_heads, d.value_dim), span("q", a.q, d.q_heads, d.key_dim),
                            span("k", a.k, d.kv_heads, d.key_dim), span("v", a.v, d.kv_heads, d.value_dim)};
  return seq::check_apart(who, rows, 4, 1);
}

// Bytes of `slots` states.
size_t states_bytes(const to_linear_attention_desc& d, long long slots) {
  return size_t(slots) * d.q_heads * d.key_dim * d.value_dim * 4;
}

constexpr size_t kAlign = 256;
size_t rounded(size_t n) { return (n + kAlign - 1) / kAlign * kAlign; }

// Bytes of the segments' states of one of `chains` chains, on either kind of cores.
size_t state_bytes(const to_linear_attention_desc& d, int chains) {
  size_t most = 0;
  for (const bool tc : {false, true}) {
    const int seg = plan_segment(d, tc, chains);
    if (seg == kOneSegment || (tc && d.dtype == TO_F32)) continue;
    const size_t slots = size_t(lin::segment_slots(static_cast<int>(d.tokens), d.nseq, seg));
    most = std::max(most, rounded(slots * d.q_heads * d.key_dim * d.value_dim * 4));
  }
  return most;
}

// f32 gradients of every query head, before the heads of a group are summed.
size_t part_bytes(const to_linear_attention_desc& d, int width) {
  return d.q_heads == d.kv_heads ? 0 : rounded(size_t(d.tokens) * d.q_heads * width * 4);
}

template <typename T, int DCB, bool STATES, int N>
int launch_simt(const lin::Batch<N>& B, cudaStream_t s) {
  static std::atomic<uint64_t> done{0};
  const size_t most = SimtShape<DCB>::bytes(DCB == 64 ? 128 : 256);
  if (int st = seq::allow_shared(chain_simt_kernel<T, DCB, STATES, N>, most, done)) return st;
  const Chain& C = B.c[0];
  int db = 0, dc = 0;
  for (const Chain& x : B.c) db = std::max(db, x.db), dc = std::max(dc, x.dc);
  const int slots = C.seg_state ? lin::segment_slots(C.tokens, C.nseq, C.seg) : C.nseq;
  const dim3 grid(static_cast<unsigned>(slots), (dc + DCB - 1) / DCB * N, C.heads);
  chain_simt_kernel<T, DCB, STATES, N><<<grid, kThreads, SimtShape<DCB>::bytes((db + 3) & ~3), s>>>(B);
  TO_CUDA_TRY(cudaGetLastError());
  return ok();
}

template <typename T, bool STATES, int N>
int launch_width(const lin::Batch<N>& B, cudaStream_t s) {
  // wider b takes narrower columns: both operands and X share 227 KB
  for (const Chain& C : B.c)
    if (C.db > 128) return launch_simt<T, 32, STATES, N>(B, s);
  return launch_simt<T, 64, STATES, N>(B, s);
}

template <int N>
int launch_scan(const lin::Batch<N>& B, cudaStream_t s) {
  const Chain& C = B.c[0];  // (db dc is the same for all)
  const int n = C.db * C.dc;
  const dim3 grid((n % 4 ? (n + 255) / 256 : (n / 4 + 255) / 256) * N, C.heads, C.nseq);
  if (n % 4) chain_scan_kernel<1, N><<<grid, 256, 0, s>>>(B);
  else chain_scan_kernel<4, N><<<grid, 256, 0, s>>>(B);
  TO_CUDA_TRY(cudaGetLastError());
  return ok();
}

template <typename T, int N>
int run_simt(const lin::Batch<N>& B, cudaStream_t s) {
  if (B.c[0].seg_state) {
    if (int st = launch_width<T, true, N>(B, s)) return st;
    if (int st = launch_scan<N>(B, s)) return st;
  }
  return launch_width<T, false, N>(B, s);
}

// `states`: workspace for the segments' states, state_bytes(d, N) for each chain.
template <int N>
int run_chains(lin::Batch<N>& B, const to_linear_attention_desc& d, void* states, cudaStream_t s) {
  auto cut = [&](bool tc) {
    const int seg = plan_segment(d, tc, N);
    const size_t each = state_bytes(d, N);
    for (int n = 0; n < N; ++n) {
      B.c[n].seg = seg;
      B.c[n].seg_state =
          seg == kOneSegment ? nullptr : reinterpret_cast<float*>(static_cast<char*>(states) + n * each);
    }
  };
  if (d.dtype == TO_BF16) {
    cut(true);
    bool all = true;
    for (const Chain& C : B.c) all = all && lin::tc_takes(C);
    if (all) {
      if (B.c[0].seg_state) {
        if (int st = lin::tc_states<N>(B, s)) return st;
        if (int st = launch_scan<N>(B, s)) return st;
      }
      return lin::tc_outputs<N>(B, s);
    }
  }
  cut(false);
  const int bytes = 4 * seq::dtype_bytes(d.dtype);
  for (Chain& C : B.c) {
    const Rows* rows[3] = {&C.a, &C.b, &C.c};
    for (int i = 0; i < 3; ++i)
      if (aligned(rows[i]->p, size_t(bytes)) && rows[i]->ts % 4 == 0 && rows[i]->hs % 4 == 0) C.vec |= 1 << i;
  }
  return d.dtype == TO_F32 ? run_simt<float, N>(B, s) : run_simt<__nv_bfloat16, N>(B, s);
}

Chain base_chain(const to_linear_attention_desc& d, const int32_t* cu, const float* log_decay) {
  Chain C{};
  C.heads = d.q_heads;
  C.nseq = d.nseq;
  C.tokens = static_cast<int>(d.tokens);
  C.cu = cu;
  C.log_decay = log_decay;
  C.a_div = C.b_div = C.c_div = 1;
  return C;
}

}  // namespace
}  // namespace to_b200

using namespace to_b200;

extern "C" {

size_t to_linear_attention_workspace_bytes(const to_linear_attention_desc* desc) {
  if (check_desc("to_linear_attention_workspace_bytes", desc)) return 0;
  return state_bytes(*desc, 1);
}

size_t to_linear_attention_backward_workspace_bytes(const to_linear_attention_desc* desc) {
  if (check_desc("to_linear_attention_backward_workspace_bytes", desc)) return 0;
  const to_linear_attention_desc& d = *desc;
  return 3 * state_bytes(d, 3) + part_bytes(d, d.key_dim) + part_bytes(d, d.value_dim);
}

int to_linear_attention(const to_linear_attention_desc* desc, const to_linear_attention_args* args,
                        void* stream) {
  const char* who = "to_linear_attention";
  if (int st = check_desc(who, desc)) return st;
  if (!args) return set_error(TO_ERR_INVALID_ARGUMENT, "%s: null arguments", who);
  const to_linear_attention_desc& d = *desc;
  const to_linear_attention_args& a = *args;
  if (d.nseq == 0) return ok();
  int st = seq::check_rows(who, "q", &a.q, d.tokens, d.q_heads, d.key_dim, d.dtype);
  if (!st) st = seq::check_rows(who, "k", &a.k, d.tokens, d.kv_heads, d.key_dim, d.dtype);
  if (!st) st = seq::check_rows(who, "v", &a.v, d.tokens, d.kv_heads, d.value_dim, d.dtype);
  if (!st) st = seq::check_rows(who, "o", &a.o, d.tokens, d.q_heads, d.value_dim, d.dtype);
  if (!st) st = check_list(who, "log_decay", a.log_decay, true);
  if (!st) st = check_list(who, "cu_seqlens", a.cu_seqlens, true);
  if (!st) st = check_list(who, "slots", a.slots, false);
  if (!st) st = check_state(who, "state_in", a.state_in);
  if (!st) st = check_state(who, "state_out", a.state_out);
  if (st) return st;
  const size_t need = state_bytes(d, 1);
  if (need && (!a.workspace || a.workspace_bytes < need))
    return set_error(TO_ERR_INVALID_ARGUMENT, "%s: workspace %zu < %zu bytes", who,
                     a.workspace ? a.workspace_bytes : 0, need);
  if (need && !aligned(a.workspace, kAlign))
    return set_error(TO_ERR_ALIGNMENT, "%s: workspace is not 256-byte aligned", who);
  if ((st = check_outputs(who, d, a))) return st;
  if (a.state_in != a.state_out &&
      seq::arrays_meet(a.state_in, a.state_out, states_bytes(d, a.slots ? d.num_slots : d.nseq)))
    return set_error(TO_ERR_INVALID_ARGUMENT, "%s: state_in and state_out share memory in part", who);
  lin::Batch<1> B{{base_chain(d, a.cu_seqlens, a.log_decay)}};
  Chain& C = B.c[0];
  C.a = seq::rows_of(a.q);
  C.b = seq::rows_of(a.k);
  C.c = seq::rows_of(a.v);
  C.out = seq::rows_of(a.o);
  C.b_div = C.c_div = d.q_heads / d.kv_heads;
  C.db = d.key_dim;
  C.dc = d.value_dim;
  C.intra = C.inter = static_cast<float>(d.scale);
  C.upd = 1.f;
  C.init = a.state_in;
  C.fin = a.state_out;
  C.slots = a.slots;
  C.num_slots = d.num_slots;
  return run_chains<1>(B, d, a.workspace, static_cast<cudaStream_t>(stream));
}

int to_linear_attention_backward(const to_linear_attention_desc* desc,
                                 const to_linear_attention_grad_args* args, void* stream) {
  const char* who = "to_linear_attention_backward";
  if (int st = check_desc(who, desc)) return st;
  if (!args) return set_error(TO_ERR_INVALID_ARGUMENT, "%s: null arguments", who);
  const to_linear_attention_desc& d = *desc;
  const to_linear_attention_grad_args& a = *args;
  if (d.nseq == 0) return ok();
  int st = seq::check_rows(who, "q", &a.q, d.tokens, d.q_heads, d.key_dim, d.dtype);
  if (!st) st = seq::check_rows(who, "k", &a.k, d.tokens, d.kv_heads, d.key_dim, d.dtype);
  if (!st) st = seq::check_rows(who, "v", &a.v, d.tokens, d.kv_heads, d.value_dim, d.dtype);
  if (!st) st = seq::check_rows(who, "d_o", &a.d_o, d.tokens, d.q_heads, d.value_dim, d.dtype);
  if (!st) st = seq::check_rows(who, "dq", &a.dq, d.tokens, d.q_heads, d.key_dim, d.dtype);
  if (!st) st = seq::check_rows(who, "dk", &a.dk, d.tokens, d.kv_heads, d.key_dim, d.dtype);
  if (!st) st = seq::check_rows(who, "dv", &a.dv, d.tokens, d.kv_heads, d.value_dim, d.dtype);
  if (!st) st = check_list(who, "log_decay", a.log_decay, true);
  if (!st) st = check_list(who, "cu_seqlens", a.cu_seqlens, true);
  if (!st) st = check_state(who, "state_in", a.state_in);
  if (!st) st = check_state(who, "dstate_out", a.dstate_out);
  if (!st) st = check_state(who, "dstate_in", a.dstate_in);
  if (st) return st;
  // the three chains run at the same time: none may write what another reads
  const size_t states = states_bytes(d, d.nseq);
  if (seq::arrays_meet(a.dstate_in, a.dstate_out, states)) return seq::refuse_overlap(who, "dstate_in", "dstate_out");
  if (seq::arrays_meet(a.dstate_in, a.state_in, states)) return seq::refuse_overlap(who, "dstate_in", "state_in");
  const size_t need = to_linear_attention_backward_workspace_bytes(desc);
  if (need && (!a.workspace || a.workspace_bytes < need))
    return set_error(TO_ERR_INVALID_ARGUMENT, "%s: workspace %zu < %zu bytes", who,
                     a.workspace ? a.workspace_bytes : 0, need);
  if (need && !aligned(a.workspace, kAlign))
    return set_error(TO_ERR_ALIGNMENT, "%s: workspace is not 256-byte aligned", who);
  const int group = d.q_heads / d.kv_heads;
  auto span = [&](const char* name, const to_rows& r, int heads, int width) {
    return seq::span_of(name, &r, d.tokens, heads, width, d.dtype);
  };
  const seq::Span rows[] = {span("dq", a.dq, d.q_heads, d.key_dim), span("dk", a.dk, d.kv_heads, d.key_dim),
                            span("dv", a.dv, d.kv_heads, d.value_dim), span("q", a.q, d.q_heads, d.key_dim),
                            span("k", a.k, d.kv_heads, d.key_dim), span("v", a.v, d.kv_heads, d.value_dim),
                            span("d_o", a.d_o, d.q_heads, d.value_dim)};
  if ((st = seq::check_apart(who, rows, 7, 3))) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const float scale = static_cast<float>(d.scale);
  // the gradients of shared heads go through f32 rows of every query head
  char* part = static_cast<char*>(a.workspace) + 3 * state_bytes(d, 3);
  float* parts[2] = {reinterpret_cast<float*>(part), reinterpret_cast<float*>(part + part_bytes(d, d.key_dim))};
  auto target = [&](Chain& C, const to_rows& r, int n, int width) {
    C.out_f32 = group > 1;
    C.out = group == 1 ? seq::rows_of(r)
                       : Rows{reinterpret_cast<char*>(parts[n]), static_cast<long long>(d.q_heads) * width, width};
  };
  const Chain base = base_chain(d, a.cu_seqlens, a.log_decay);
  lin::Batch<3> B{{base, base, base}};
  // dq: forwards, a = do, b = v, c = k
  Chain& dq = B.c[0];
  dq.a = seq::rows_of(a.d_o);
  dq.b = seq::rows_of(a.v);
  dq.c = seq::rows_of(a.k);
  dq.out = seq::rows_of(a.dq);
  dq.b_div = dq.c_div = group;
  dq.db = d.value_dim;
  dq.dc = d.key_dim;
  dq.intra = dq.inter = scale;
  dq.upd = 1.f;
  dq.init = a.state_in;
  dq.init_t = 1;
  // dk: backwards, a = v, b = do, c = q
  Chain& dk = B.c[1];
  dk.a = seq::rows_of(a.v);
  dk.b = seq::rows_of(a.d_o);
  dk.c = seq::rows_of(a.q);
  target(dk, a.dk, 0, d.key_dim);
  dk.a_div = group;
  dk.db = d.value_dim;
  dk.dc = d.key_dim;
  dk.rev = 1;
  dk.intra = dk.upd = scale;
  dk.inter = 1.f;
  dk.init = a.dstate_out;
  dk.init_t = 1;
  // dv: backwards, a = k, b = q, c = do
  Chain& dv = B.c[2];
  dv.a = seq::rows_of(a.k);
  dv.b = seq::rows_of(a.q);
  dv.c = seq::rows_of(a.d_o);
  target(dv, a.dv, 1, d.value_dim);
  dv.a_div = group;
  dv.db = d.key_dim;
  dv.dc = d.value_dim;
  dv.rev = 1;
  dv.intra = dv.upd = scale;
  dv.inter = 1.f;
  dv.init = a.dstate_out;
  dv.fin = a.dstate_in;
  if ((st = run_chains<3>(B, d, a.workspace, s))) return st;
  if (group == 1 || d.tokens == 0) return ok();
  GroupSum G{{parts[0], parts[1]}, {seq::rows_of(a.dk), seq::rows_of(a.dv)}, {d.key_dim, d.value_dim},
             a.cu_seqlens, d.nseq, static_cast<int>(d.tokens), d.kv_heads, group};
  const long long want = (d.tokens * d.kv_heads * std::max(d.key_dim, d.value_dim) + 255) / 256;
  const dim3 grid(static_cast<unsigned>(std::min(want, 148ll * 16)), 2);
  if (d.dtype == TO_BF16) group_sum_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(G);
  else group_sum_kernel<float><<<grid, 256, 0, s>>>(G);
  TO_CUDA_TRY(cudaGetLastError());
  return ok();
}

int to_linear_attention_step(const to_linear_attention_desc* desc,
                             const to_linear_attention_args* args, void* stream) {
  const char* who = "to_linear_attention_step";
  if (int st = check_desc(who, desc)) return st;
  if (!args) return set_error(TO_ERR_INVALID_ARGUMENT, "%s: null arguments", who);
  const to_linear_attention_desc& d = *desc;
  const to_linear_attention_args& a = *args;
  if (d.tokens == 0) return ok();
  int st = seq::check_rows(who, "q", &a.q, d.tokens, d.q_heads, d.key_dim, d.dtype);
  if (!st) st = seq::check_rows(who, "k", &a.k, d.tokens, d.kv_heads, d.key_dim, d.dtype);
  if (!st) st = seq::check_rows(who, "v", &a.v, d.tokens, d.kv_heads, d.value_dim, d.dtype);
  if (!st) st = seq::check_rows(who, "o", &a.o, d.tokens, d.q_heads, d.value_dim, d.dtype);
  if (!st) st = check_list(who, "log_decay", a.log_decay, true);
  if (!st) st = check_list(who, "slots", a.slots, false);
  if (st) return st;
  if (!a.state_out) return set_error(TO_ERR_INVALID_ARGUMENT, "%s: state_out is null", who);
  if ((st = check_state(who, "state_out", a.state_out))) return st;
  if ((st = check_outputs(who, d, a))) return st;
  StepArgs A{};
  A.q = seq::rows_of(a.q);
  A.k = seq::rows_of(a.k);
  A.v = seq::rows_of(a.v);
  A.o = seq::rows_of(a.o);
  A.log_decay = a.log_decay;
  A.slots = a.slots;
  A.state = a.state_out;
  A.num_slots = d.num_slots;
  A.heads = d.q_heads;
  A.group = d.q_heads / d.kv_heads;
  A.dk = d.key_dim;
  A.dv = d.value_dim;
  A.scale = static_cast<float>(d.scale);
  const bool vec = d.value_dim % 4 == 0;  // rows of the state stay 16-byte aligned
  // columns of a CTA: up to 128, fewer (32 at least) while the CTAs are fewer than two an SM
  int cols = 128;
  const long long work = d.tokens * d.q_heads;
  while (cols > 32 && (cols / 2 >= d.value_dim || work * ((d.value_dim + cols - 1) / cols) < 2 * 148)) cols /= 2;
  A.cols = cols;
  const dim3 grid(static_cast<unsigned>(d.tokens), d.q_heads, (d.value_dim + cols - 1) / cols);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (d.dtype == TO_BF16) {
    if (vec) step_kernel<__nv_bfloat16, 4><<<grid, kStepThreads, 0, s>>>(A);
    else step_kernel<__nv_bfloat16, 1><<<grid, kStepThreads, 0, s>>>(A);
  } else {
    if (vec) step_kernel<float, 4><<<grid, kStepThreads, 0, s>>>(A);
    else step_kernel<float, 1><<<grid, kStepThreads, 0, s>>>(A);
  }
  TO_CUDA_TRY(cudaGetLastError());
  return ok();
}

}  // extern "C"

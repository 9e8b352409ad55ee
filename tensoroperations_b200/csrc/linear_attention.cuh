// linear_attention.cuh -- the decayed chain behind linear attention and its
// gradients, and how it is cut along the sequences.
//
// One chain serves all of them.  With rows a, b, c of a sequence in the
// chain's direction (forwards or backwards in time), i and j counting tokens
// in that direction, l = exp(log_decay[head]):
//   out_i = intra * sum_{j <= i} l^(i-j) (a_i . b_j) c_j  +  inter * l^(i+1-rev) a_i . X
//   X'    = l^n X + upd * sum_j l^(n-1+rev-j) b_j c_j^T     (n tokens later)
//   forward  a = q,  b = k,   c = v :  o,  X = S
//   dq       a = do, b = v,   c = k :  X = S^T
//   dv       a = k,  b = q,   c = do, backwards, X = l * gradient of S
//   dk       a = v,  b = do,  c = q,  backwards, X = l * gradient of S, transposed
// `rev` (1 backwards) shifts the decay by one token: a gradient state enters
// undecayed at the last token and has decayed once when it leaves the first.
//
// Along a sequence the chain is cut into segments of `seg` tokens (a multiple
// of the chunk).  Segment slots: sequence s owns slots floor(cu[s]/seg) + s
// and up, enough for its ceil(len/seg) (at least one), without any prefix sum
// over the lengths, so the grid needs nothing from the host.  Three launches:
// every segment's own X from zero (not the last one's), a scan that turns them
// into each segment's entering X, and the outputs.  Where one segment holds
// any sequence, the outputs' launch alone does it all.
#pragma once

#include "sequence_common.cuh"

namespace to_b200 {
namespace lin {

using seq::Rows;

struct Chain {
  Rows a, b, c, out;
  int a_div, b_div, c_div;  // head h reads head h / div
  int heads, nseq;
  int db, dc;  // widths of b (and a) and of c (and out)
  int tokens;
  const int32_t* cu;
  const float* log_decay;
  float intra, inter, upd;
  int rev;
  // entering and leaving X of whole sequences: [slot][heads] matrices [db][dc]
  // (the entering one [dc][db] when init_t)
  const float* init;
  float* fin;
  int init_t;
  const int32_t* slots;
  long long num_slots;
  float* seg_state;  // [segment slots][heads][db][dc]; null: one segment a sequence
  int seg;           // tokens of a segment
  int vec;           // bits 0, 1, 2: rows of a, b, c can be read four values at a time
  int out_f32;       // out is f32, not of the rows' type
};

// The chains of one call, run by the same launches: one forwards, three for the
// gradients.  Sequences and segments are the same for all.
template <int N>
struct Batch {
  Chain c[N];
};

// Where a segment lies.  idx < 0: an unused slot.
struct Segment {
  int seq, idx, count;  // its sequence, its place among the sequence's `count`
  int first, tokens;    // the sequence's first row, its length
};

__device__ __forceinline__ int clamped(const Chain& C, int s) {
  const int x = __ldg(C.cu + s);
  return x < 0 ? 0 : x > C.tokens ? C.tokens : x;
}

__device__ __forceinline__ Segment sequence_of(const Chain& C, int s) {
  Segment g;
  g.seq = s;
  g.first = clamped(C, s);
  const int end = clamped(C, s + 1);
  g.tokens = end > g.first ? end - g.first : 0;
  g.count = g.tokens ? (g.tokens - 1) / C.seg + 1 : 1;
  g.idx = 0;
  return g;
}

__device__ __forceinline__ int first_slot(const Chain& C, int s) {
  return clamped(C, s) / C.seg + s;
}

// The last sequence whose first slot is at most w, by bisection.
__device__ __forceinline__ Segment segment_of(const Chain& C, int w) {
  int lo = 0, hi = C.nseq - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first_slot(C, mid) <= w) lo = mid;
    else hi = mid - 1;
  }
  Segment g = sequence_of(C, lo);
  const int idx = w - first_slot(C, lo);
  g.idx = idx >= 0 && idx < g.count ? idx : -1;
  return g;
}

// At most 2^31 / 512 + 65535, or one a sequence and one more.
__host__ __device__ inline int segment_slots(int tokens, int nseq, int seg) {
  return tokens / seg + nseq;
}

__device__ __forceinline__ float log_decay_of(const Chain& C, int h) {
  // -1e30 stands for -inf (0 * -inf has no value): exp gives 1 at distance 0, else 0
  const float g = __ldg(C.log_decay + h);
  return g < -1e30f ? -1e30f : g > 0.f ? 0.f : g;
}

// State slot of a sequence; -1: none.
__device__ __forceinline__ long long state_slot(const Chain& C, int s) {
  if (!C.slots) return s;
  const long long x = __ldg(C.slots + s);
  return x >= 0 && x < C.num_slots ? x : -1;
}

__device__ __forceinline__ long long state_index(const Chain& C, int transposed, int b, int c) {
  return transposed ? static_cast<long long>(c) * C.db + b : static_cast<long long>(b) * C.dc + c;
}

// The tensor-core form (linear_attention_tc.cu): whether it takes a chain's
// rows, every segment's own X, and the outputs, N = 1 or 3.
bool tc_takes(const Chain& C);
template <int N>
int tc_states(const Batch<N>& B, cudaStream_t s);
template <int N>
int tc_outputs(const Batch<N>& B, cudaStream_t s);

}  // namespace lin
}  // namespace to_b200

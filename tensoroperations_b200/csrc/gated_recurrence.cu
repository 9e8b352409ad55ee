// gated_recurrence.cu -- the gated linear recurrence of every channel
//   a_t = sigmoid(f_t + bias),  h_t = a_t h_{t-1} + (1 - a_t) x_t  (or + x_t),
// over packed sequences in one pass, its gradients in another, and the
// single-token step.
//
// The maps h -> A h + H compose: (A, H) then (A', H') is (A' A, A' H + H'), so a
// sequence is cut into segments of 128 tokens that are reduced at the same time
// and joined afterwards.  A CTA takes a segment and 128 bytes of channels (64 bf16
// or 32 f32, two or one a lane).  Each of eight warps goes over 16 tokens once and
// keeps, in registers, the map of its first tokens up to every one of them; the
// maps of the warps are joined in shared memory, those of the segments through
// global memory while the CTAs run (below), and with the state that enters every
// output is one multiply-add.  So x and f are read once and h is written once; 8
// flops, two special functions a value (exp and a reciprocal) and three selections
// leave it memory bound in principle.  Gradients keep the gates and df_t / G_t instead,
// and walk back once what enters from behind is known.
//
// Measured on B200 (behind an L2 flush; gates do not change it): 49152 tokens x 4096 channels
// bf16, one sequence, in 262 us, 4.6 TB/s (0.71 of the copy rate): its 64 chains of segments
// keep 296 CTAs busy, so four or five segments of a chain are in work at once and wait for one
// another's maps (a form that took 261 us took 200 without those waits; eight more warps that
// only reduce, a tile ahead, and eight that walk needed half as many instructions again, and
// 277).  24576 x 4096 f32 215 us, 5.6 TB/s, its gradients 326 us, 6.2 TB/s.  4 x 4096 tokens x
// 4096 bf16 with 8-bit copies 128 us, 4.2 TB/s, 43 instructions a value, near what 20 warps an
// SM issue; gradients of these 174 us, 3.9 TB/s, from 8 bits 211 us, 2.6 TB/s, 57 instructions:
// they wait for tiles and for the slowest of eight warps.  Rows that TMA does not take are
// copied by the warps that compute: 16384 x 4091 bf16 279 us, gradients 514 us, with 8-bit
// copies 680 and 606 us.
//
// Gates: with u = exp(-|f|), u / (1 + u) is the smaller of a and 1 - a, accurate to
// f32 relative to itself.  It is kept with a sign ("c": a where positive, -(1 - a)
// where negative), and every step adds c times a difference to the larger term:
//   f >= 0:  h + (1 - a)(x - h)      f < 0:  x + a (h - x)
// so a memory of thousands of tokens does not take over a rounding of a near 1, and
// what is left of a state after a token that almost forgets it stays exact.  All gates
// take these steps: a path without the selections, for tiles whose gates all lie above
// -2.77 (a made of 1 - a, four tokens' reciprocals shared), was 2 to 4 % faster forwards, but
// lost up to 6 bits of a there, and a channel's digits went by its neighbours' gates.
//
// Joining the segments: a CTA takes segments in the order of a counter (so a
// segment's predecessors have been taken by CTAs that run), publishes its map as
// soon as it has reduced its tokens, and folds the maps of its predecessors from
// the nearest one whose number is a multiple of 8, whose entering state is
// published too.  One of its warps does that while others reduce.  What is folded, and in
// which order, goes by the segment's number alone: results do not depend on timing.  A
// published word is a value and its mark in 8 bytes, written and read at once, so
// no fence and no flag is waited for; the words are cleared before the launch.
//
// Waits are bounded.  Where a map does not come, what enters is NaN, and so is all that
// depends on it.  Where a barrier of a CTA's own warps does not, the CTA ends: the warp that
// has waited sets a flag which ends the other warps' waits, the eight that compute agree on
// it at their next barrier (which all of them reach), and the one that looks ahead leaves
// when its tiles have landed.  Both set the device status.
#include <algorithm>

#include "rows8.cuh"
#include "sm100_primitives.cuh"
#include "tensor_map.hpp"

namespace to_b200 {
namespace {

using seq::Packed;
using seq::Rows;

constexpr int kSegment = TO_RECURRENCE_SEGMENT;   // tokens of a tile; a state is saved at the head of each
constexpr int kWarps = 8, kThreads = 32 * kWarps;  // that compute
constexpr int kRowBytes = 128;                    // of a tile's row of values
constexpr int kChained = 1024;                    // tokens between published states
// How long a segment waits for others' maps, and a CTA's warps for one another and for tiles.
constexpr long long kMapsWait = 2000000, kTilesWait = 8000000;  // microseconds
constexpr uint32_t kDrain = 1u << 22;                            // polls for tiles in flight, at a CTA's end

__device__ int g_recurrence_status;

// A lane's channels: one 32-bit word of a row, as one f32 or two in a register pair
// (packed f32x2 instructions).
template <int V>
struct Vals;
template <>
struct Vals<1> {
  float v[1];
};
template <>
struct Vals<2> {
  float v[2];
};
template <int V>
__device__ __forceinline__ Vals<V> all(float x) {
  Vals<V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = x;
  return r;
}
__device__ __forceinline__ Vals<1> fma(Vals<1> a, Vals<1> b, Vals<1> c) { return {{fmaf(a.v[0], b.v[0], c.v[0])}}; }
__device__ __forceinline__ Vals<2> fma(Vals<2> a, Vals<2> b, Vals<2> c) {
  const float2 r = __ffma2_rn(make_float2(a.v[0], a.v[1]), make_float2(b.v[0], b.v[1]), make_float2(c.v[0], c.v[1]));
  return {{r.x, r.y}};
}
__device__ __forceinline__ Vals<1> mul(Vals<1> a, Vals<1> b) { return {{a.v[0] * b.v[0]}}; }
__device__ __forceinline__ Vals<2> mul(Vals<2> a, Vals<2> b) {
  const float2 r = __fmul2_rn(make_float2(a.v[0], a.v[1]), make_float2(b.v[0], b.v[1]));
  return {{r.x, r.y}};
}
__device__ __forceinline__ Vals<1> add(Vals<1> a, Vals<1> b) { return {{a.v[0] + b.v[0]}}; }
__device__ __forceinline__ Vals<2> add(Vals<2> a, Vals<2> b) {
  const float2 r = __fadd2_rn(make_float2(a.v[0], a.v[1]), make_float2(b.v[0], b.v[1]));
  return {{r.x, r.y}};
}
template <int V>
__device__ __forceinline__ Vals<V> sub(Vals<V> a, Vals<V> b) {
  return fma(b, all<V>(-1.f), a);
}

// The same values, which the compiler keeps in registers: packed instructions take no
// immediates, and made anew for each they cost two moves.
template <int V>
__device__ __forceinline__ Vals<V> kept(Vals<V> x) {
#pragma unroll
  for (int i = 0; i < V; ++i) asm volatile("" : "+f"(x.v[i]));
  return x;
}

template <typename T>
struct Lane {
  static constexpr int kVec = 4 / int(sizeof(T));
  static constexpr int kChannels = kRowBytes / int(sizeof(T));  // of a tile
  using P = Vals<kVec>;
  __device__ __forceinline__ static P unpack(uint32_t w) {
    if constexpr (kVec == 1) return {{__uint_as_float(w)}};
    else return {{__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)}};
  }
  __device__ __forceinline__ static uint32_t pack(const P& p) {
    if constexpr (kVec == 1) {
      return __float_as_uint(p.v[0]);
    } else {
      const __nv_bfloat162 b = __floats2bfloat162_rn(p.v[0], p.v[1]);
      return *reinterpret_cast<const uint32_t*>(&b);
    }
  }
};

// How a call's segments lie, and what they share (see the head of the file).
struct Chain {
  const int32_t* cu;
  int nseq, tokens, channels, slabs, slots;  // slabs: tiles of channels; slots: segments that there may be
  unsigned* ticket;                          // null: no sequence is longer than a segment
  int* gave_up;                              // set once a wait of this call has run out; null where ticket is
  long long maps_wait, tiles_wait;           // nanoseconds
  // [slots][slabs * kChannels] words of two f32, zero until they are published
  uint64_t* maps;    // (H, A with its sign bit set)
  uint64_t* states;  // (the entering state, 1)
};

struct Item {
  int slot, slab, idx, count, seq, row0, n;  // slot -1: no more
};

__device__ __forceinline__ int bound_of(const Chain& C, int s) {
  const int x = __ldg(C.cu + s);
  return x < 0 ? 0 : x > C.tokens ? C.tokens : x;
}

// The segment of slot w, by the warp together: sequence s owns the slots
// cu[s] / kSegment + s and up, enough for its segments (an empty sequence has one).
__device__ __forceinline__ void find_segment(const Chain& C, int w, int lane, Item& it) {
  int lo = 0, hi = C.nseq;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, probe = lo + lane * step;
    const bool below = probe < hi && bound_of(C, probe) / kSegment + probe <= w;
    const int found = __popc(__ballot_sync(0xffffffffu, below));
    lo += found > 1 ? (found - 1) * step : 0;
    hi = min(hi, lo + step);
  }
  const int first = bound_of(C, lo), end = bound_of(C, lo + 1);
  const int tokens = end > first ? end - first : 0;
  it.seq = lo;
  it.count = tokens ? (tokens - 1) / kSegment + 1 : 1;
  it.idx = w - (first / kSegment + lo);
  if (it.idx < 0 || it.idx >= it.count) it.idx = -1;
  it.row0 = first + it.idx * kSegment;
  it.n = min(kSegment, tokens - it.idx * kSegment);
  it.slot = w;
}

__device__ __forceinline__ void next_ticket(const Chain& C, unsigned& ticket, int lane) {
  // (as PTX: atomicAdd is turned into one for the warp, whose result is waited for at once)
  if (!C.ticket) ticket += gridDim.x;
  else if (lane == 0) asm volatile("atom.relaxed.gpu.global.add.u32 %0, [%1], 1;" : "=r"(ticket) : "l"(C.ticket) : "memory");
}

// The order of the segments.  Segments of one sequence that are in work at the same time wait
// for one another's maps, so sequences are taken side by side: the slots are cut into at most
// kSides parts, each at the beginning of a sequence, and every part in turn gives its next slot
// (backwards: from its end).  A sequence lies in one part, so its segments keep their order.
// (Four sequences of 4096 tokens, 4096 channels, forwards: 157 us one after the other, then 136.)
constexpr int kSides = 8;

struct Order {  // of a whole warp: lane g < kSides holds part g
  int begin = 0, size = 0;
  int round = 0, before = 0;  // before: upto(round)

  __device__ __forceinline__ Order(const Chain& C, int lane) {
    if (lane < kSides) {
      const int target = static_cast<int>(static_cast<long long>(C.slots) * lane / kSides);
      int lo = 0, hi = lane ? C.nseq : 1;  // the last sequence that begins at or before it
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (bound_of(C, mid) / kSegment + mid <= target) lo = mid;
        else hi = mid;
      }
      begin = lane ? min(bound_of(C, lo) / kSegment + lo, target) : 0;
    }
#pragma unroll
    for (int o = 1; o < kSides; o <<= 1) {  // (no part begins before another one, whatever cu holds)
      const int other = __shfl_up_sync(0xffffffffu, begin, o);
      if (lane >= o) begin = max(begin, other);
    }
    const int next = __shfl_down_sync(0xffffffffu, begin, 1);
    if (lane < kSides) size = max(0, (lane + 1 < kSides ? next : C.slots) - begin);
  }
  __device__ __forceinline__ int upto(int rounds) const {  // slots of the first rounds
    return __reduce_add_sync(0xffffffffu, min(size, rounds));
  }
  // The n-th slot; n never falls from one call to the next.
  template <bool BACKWARD>
  __device__ __forceinline__ int slot(int n, int lane) {
    for (int next; (next = upto(round + 1)) <= n; ++round) before = next;
    const uint32_t active = __ballot_sync(0xffffffffu, size > round);
    const bool mine = size > round && __popc(active & ((1u << lane) - 1)) == n - before;
    const int from = __ffs(__ballot_sync(0xffffffffu, mine)) - 1;
    return __shfl_sync(0xffffffffu, BACKWARD ? begin + size - 1 - round : begin + round, from);
  }
};

// The item of a warp's ticket (lane 0's); a slot that no segment has goes to `unused`,
// and the next ticket is taken.  `ticket`: the one that the item has.
template <bool BACKWARD, typename UNUSED>
__device__ __forceinline__ Item next_item(const Chain& C, Order& order, unsigned& ticket, int lane, UNUSED&& unused) {
  Item it;
  for (;;) {
    ticket = __shfl_sync(0xffffffffu, ticket, 0);
    const unsigned at = ticket / static_cast<unsigned>(C.slabs);
    if (at >= static_cast<unsigned>(C.slots)) {
      it.slot = -1;
      return it;
    }
    it.slab = static_cast<int>(ticket - at * C.slabs);
    find_segment(C, order.slot<BACKWARD>(static_cast<int>(at), lane), lane, it);
    if (it.idx >= 0) return it;
    unused(it);
    next_ticket(C, ticket, lane);
  }
}

// ---- tiles in shared memory ----------------------------------------------------------

// `rows` rows of ROWB bytes into shared memory, ACCESS bytes at a time; the
// columns from `valid` bytes on become zero.  By the eight warps; a thread keeps its column.
template <int ACCESS, int ROWB>
__device__ __forceinline__ void load_tile(char* dst, const char* src, long long pitch, int rows, int valid) {
  constexpr int kPer = ROWB / ACCESS, kStep = kThreads / kPer;  // threads of a row, rows of an iteration
  const int col = (threadIdx.x % kPer) * ACCESS, row0 = threadIdx.x / kPer;
  const int bytes = max(0, min(ACCESS, valid - col));
  const char* s = src + row0 * pitch + (bytes ? col : 0);
  dst += row0 * ROWB + col;
  const long long step = kStep * pitch;
#pragma unroll 4
  for (int row = row0; row < rows; row += kStep, s += step, dst += kStep * ROWB) {
    if constexpr (ACCESS >= 16) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(s), "r"(bytes) : "memory");
    } else if constexpr (ACCESS >= 4) {
      asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(smem_u32(dst)), "l"(s), "n"(ACCESS), "r"(bytes)
                   : "memory");
    } else if constexpr (ACCESS == 2) {
      *reinterpret_cast<uint16_t*>(dst) = bytes ? *reinterpret_cast<const uint16_t*>(s) : uint16_t(0);
    } else {
      *reinterpret_cast<uint8_t*>(dst) = bytes ? *reinterpret_cast<const uint8_t*>(s) : uint8_t(0);
    }
  }
}

template <int ROWB>
__device__ __forceinline__ void load_tile(int access, char* dst, const char* src, long long pitch, int rows, int valid) {
  if (access >= 16) load_tile<16, ROWB>(dst, src, pitch, rows, valid);
  else if (access == 8) load_tile<8, ROWB>(dst, src, pitch, rows, valid);
  else if (access == 4) load_tile<4, ROWB>(dst, src, pitch, rows, valid);
  else if (access == 2) load_tile<2, ROWB>(dst, src, pitch, rows, valid);
  else load_tile<1, ROWB>(dst, src, pitch, rows, valid);
}

__device__ __forceinline__ void close_tiles() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// until at most N of the closed groups are still on their way
template <int N>
__device__ __forceinline__ void wait_tiles() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

struct Source {  // x or f of a call: rows, or rows in 8 bits
  Rows rows;
  Packed packed;
  int access;  // bytes that one access may take
};

// A tile through TMA: `rows` of a tensor map of [tokens][channels] from (row, channel) on.
__device__ __forceinline__ void tma_tile(char* dst, const CUtensorMap* map, int channel, int row, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(channel), "r"(row), "r"(smem_u32(bar))
      : "memory");
}

// (without an arrival)
__device__ __forceinline__ void expect_bytes(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}

__device__ __forceinline__ long long nanoseconds() {
  long long t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t)::"memory");
  return t;
}

template <typename T>
__device__ __forceinline__ void load_rows(char* dst, const Rows& r, int access, const Item& it, int ch, int channels) {
  load_tile<kRowBytes>(access, dst, reinterpret_cast<const char*>(seq::row_ptr<const T>(r, it.row0, 0) + ch),
                       r.ts * static_cast<long long>(sizeof(T)), it.n, (channels - ch) * static_cast<int>(sizeof(T)));
}

// ---- the recurrence ------------------------------------------------------------------

using seq::exp2_fast;
using seq::reciprocal;

constexpr float kLog2e = 1.4426950408889634f;

// t = log2(e) (f + bias).  The sum comes first: its rounding is relative to f + bias, also where the two cancel.
template <int V>
__device__ __forceinline__ Vals<V> argument_of(Vals<V> f, Vals<V> bias, const Vals<V>& log2e) {
  return mul(add(f, bias), log2e);
}
// c of a gate, from its argument; below 2^-126 it counts as zero.
template <int V>
__device__ __forceinline__ Vals<V> gate_of(Vals<V> t) {
  Vals<V> u, r;
#pragma unroll
  for (int i = 0; i < V; ++i) u.v[i] = exp2_fast(-fabsf(t.v[i]));
  r = add(u, all<V>(1.f));
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = reciprocal(r.v[i]);
  r = mul(u, r);
#pragma unroll
  for (int i = 0; i < V; ++i)
    r.v[i] = __uint_as_float(__float_as_uint(r.v[i]) | (~__float_as_uint(t.v[i]) & 0x80000000u));
  return r;
}
// c is -(1 - a)
__device__ __forceinline__ bool is_rest(float c) { return __float_as_int(c) < 0; }
// a h
template <int V>
__device__ __forceinline__ Vals<V> decayed(Vals<V> c, Vals<V> h) {
  Vals<V> base;
#pragma unroll
  for (int i = 0; i < V; ++i) base.v[i] = is_rest(c.v[i]) ? h.v[i] : 0.f;
  return fma(c, h, base);
}
// one step of the recurrence
template <bool COMPLEMENT, int V>
__device__ __forceinline__ Vals<V> stepped(Vals<V> c, Vals<V> x, Vals<V> h) {
  const Vals<V> other = COMPLEMENT ? h : add(h, x);
  Vals<V> base;
#pragma unroll
  for (int i = 0; i < V; ++i) base.v[i] = is_rest(c.v[i]) ? other.v[i] : x.v[i];
  return fma(c, COMPLEMENT ? sub(h, x) : h, base);
}

// h -> a h + b of a lane's channels.
template <int V>
struct alignas(8 * V) Map {
  Vals<V> a, b;
  __device__ __forceinline__ Vals<V> operator()(Vals<V> h) const { return fma(a, h, b); }
  // this map, then m
  __device__ __forceinline__ Map then(const Map& m) const { return {mul(a, m.a), m(b)}; }
};

// ---- segments joined while the CTAs run ------------------------------------------------

__device__ __forceinline__ uint64_t word_of(float value, uint32_t mark) {
  return static_cast<uint64_t>(mark) << 32 | __float_as_uint(value);
}
__device__ __forceinline__ void publish(uint64_t* p, uint64_t w) {
  asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(p), "l"(w) : "memory");
}
__device__ __forceinline__ uint64_t published(const uint64_t* p) {
  uint64_t w;
  asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(w) : "l"(p) : "memory");
  return w;
}

__device__ __forceinline__ void give_up(const Chain& C) {
  if (C.gave_up) atomicExch(C.gave_up, 1);
  atomicExch(&g_recurrence_status, TO_ERR_TIMEOUT);
}

// What a CTA has to do with the other segments of its sequence: position p of
// `count` in the chain's direction, whose slots lie at origin + dir * position.
template <typename T>
struct Links {
  static constexpr int kChain = kChained / kSegment;
  static constexpr int V = Lane<T>::kVec, CH = Lane<T>::kChannels;
  const Chain& C;
  int lane, slab, origin, dir, p, count;

  __device__ __forceinline__ long long place(int at) const {
    return (static_cast<long long>(origin + dir * at) * C.slabs + slab) * CH + lane * V;
  }
  __device__ __forceinline__ int base() const { return (p - 1) / kChain * kChain; }  // of p > 0
  // The segment's own map, for those behind it.
  __device__ __forceinline__ void publish_map(const Map<V>& m) const {
    if (p + 1 >= count) return;
#pragma unroll
    for (int v = 0; v < V; ++v)
      publish(C.maps + place(p) + v, word_of(m.b.v[v], __float_as_uint(m.a.v[v]) | 0x80000000u));
  }
  __device__ __forceinline__ void publish_state(const Vals<V>& h) const {
    if (p + 1 >= count || p % kChain) return;
#pragma unroll
    for (int v = 0; v < V; ++v) publish(C.states + place(p) + v, word_of(h.v[v], 1u));
  }
  // The state that enters position p > 0, by one warp: the state at base() and the maps from
  // there on, applied in order.  NaN where they do not come.
  __device__ __forceinline__ Vals<V> entering() const {
    const int b = base(), n = p - b;
    long long since = 0;
    uint64_t w[kChain][V], state[V];
    uint32_t missing = (1u << n) - 1 | 1u << kChain;
    for (uint32_t polls = 0;; ++polls) {
#pragma unroll
      for (int k = 0; k <= kChain; ++k) {
        if (!(missing >> k & 1)) continue;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          if (k < kChain) w[k < kChain ? k : 0][v] = published(C.maps + place(b + k) + v);
          else state[v] = published(C.states + place(b) + v);
        }
      }
#pragma unroll
      for (int k = 0; k <= kChain; ++k) {
        if (!(missing >> k & 1)) continue;
        bool there = true;
#pragma unroll
        for (int v = 0; v < V; ++v) there = there && (k < kChain ? w[k < kChain ? k : 0][v] : state[v]) != 0;
        if (__all_sync(0xffffffffu, there)) missing &= ~(1u << k);
      }
      if (!missing) break;
      if (polls % 64 == 63 || !C.maps_wait) {  // (once a wait has run out, the others of the call need not)
        const long long now = nanoseconds();
        if (!since) since = now;
        bool out = now - since >= C.maps_wait;
        if (lane == 0 && !out) out = *reinterpret_cast<volatile int*>(C.gave_up) != 0;
        if (__any_sync(0xffffffffu, out)) {
          if (lane == 0) give_up(C);
          return all<V>(__int_as_float(0x7fc00000));
        }
      }
    }
    Vals<V> e;
#pragma unroll
    for (int v = 0; v < V; ++v) e.v[v] = __uint_as_float(static_cast<uint32_t>(state[v]));
#pragma unroll
    for (int k = 0; k < kChain; ++k) {
      if (k >= n) continue;
      Map<V> m;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        m.a.v[v] = __uint_as_float(static_cast<uint32_t>(w[k][v] >> 32) & 0x7fffffffu);
        m.b.v[v] = __uint_as_float(static_cast<uint32_t>(w[k][v]));
      }
      e = m(e);
    }
    return e;
  }
};

// ---- forward -----------------------------------------------------------------------

struct ForwardArgs {
  CUtensorMap x_map, f_map;  // (TMA)
  Chain C;
  Rows x, f, h;
  int x_access, f_access, pairs;  // pairs: a lane's word of h is one access
  Packed keep_x, keep_f;          // codes null: not kept
  int keep_access;
  const float* bias;
  const int32_t* slots;
  long long num_slots;
  const float* state_in;
  float* state_out;
  float* saved;
};

template <typename T>
__device__ __forceinline__ void store_word(T* p, uint32_t w, int n, bool whole) {
  if constexpr (sizeof(T) == 4) {
    if (n > 0) *reinterpret_cast<uint32_t*>(p) = w;
  } else {
    if (whole && n >= 2) {
      *reinterpret_cast<uint32_t*>(p) = w;
    } else {
      if (n > 0) *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(w);
      if (n > 1) *(reinterpret_cast<uint16_t*>(p) + 1) = static_cast<uint16_t>(w >> 16);
    }
  }
}

// A tile of values in shared memory into 8 bits: 16 values a thread, two threads a group.
template <typename T>
__device__ __forceinline__ void keep_tile(const char* tile, const Packed& out, int access, const Item& it, int ch,
                                          int channels) {
  constexpr int kParts = Lane<T>::kChannels / 16;
  for (int i = threadIdx.x; i < kSegment * kParts; i += kThreads) {  // (whole warps)
    const int row = i / kParts, part = i % kParts, c = ch + part * 16;
    float x[16];
    seq::load_vec<T, 16>(reinterpret_cast<const T*>(tile + row * kRowBytes) + part * 16, x);
    uint32_t most = 0;
    if constexpr (sizeof(T) == 2) {  // two at a time, as they lie
      const uint4* raw = reinterpret_cast<const uint4*>(tile + row * kRowBytes + part * 32);
      const uint4 a = raw[0], b = raw[1];
      for (const uint32_t w : {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}) most = __vmaxu2(most, w & 0x7fff7fffu);
      most = max(most << 16, most & 0xffff0000u);
    } else {
#pragma unroll
      for (int k = 0; k < 16; ++k) most = max(most, seq::abs_bits(x[k]));
    }
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    const int byte = seq::scale_byte(most);
    const float inverse = seq::inverse_scale(byte);
    union { uint4 v; uint32_t w[4]; uint8_t b[16]; } u;
#pragma unroll
    for (int k = 0; k < 4; ++k) u.w[k] = seq::codes_of(x + 4 * k, inverse, byte != 255);
    if (row >= it.n || c >= channels) continue;
    int8_t* to = out.codes + (it.row0 + static_cast<long long>(row)) * out.code_stride + c;
    const int n = min(16, channels - c);
    if (access >= 16 && n == 16) {
      *reinterpret_cast<uint4*>(to) = u.v;
    } else if (access >= 4 && n == 16) {
#pragma unroll
      for (int k = 0; k < 4; ++k) *(reinterpret_cast<uint32_t*>(to) + k) = u.w[k];
    } else {
#pragma unroll
      for (int k = 0; k < 16; ++k)
        if (k < n) to[k] = static_cast<int8_t>(u.w[k / 4] >> (8 * (k % 4)));
    }
    if (part % 2 == 0) out.scales[(it.row0 + static_cast<long long>(row)) * out.scale_stride + c / 32] = static_cast<uint8_t>(byte);
  }
}

// Ten warps: eight compute.  One looks ahead: it takes tickets, reads what a tile's
// channels need once (bias, and backwards the saved state) and, where TMA takes the
// rows, loads the tiles, two stages ahead.  One finds out what enters a tile while the
// eight reduce it; these join the maps of the warps before them (the last one so has the
// segment's, and publishes it).
constexpr int kAhead = kWarps, kEntering = kWarps + 1, kLaunched = kThreads + 64;

struct Stages {
  uint64_t known[2], full[2], empty[2];  // the item, its tile, its tile has been read
  uint64_t entered[4];                   // (a tile's is read after its stage is empty: twice as many)
  Item items[2];
  int lost;  // a wait for one of the barriers has run out
};

// Until a barrier's phase is complete; false: it does not come, or another warp has given up.
// By whole warps, which agree on the answer (no phase follows before its warp has gone on).
// The two warps that do not compute watch the time.
__device__ __forceinline__ bool wait_for(const Chain& C, Stages& S, uint64_t* bar, uint32_t parity) {
  volatile int* const lost = &S.lost;
  long long since = 0;
  for (uint32_t n = 1; C.tiles_wait; ++n) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    bool out = *lost != 0;
    if (n % 16 == 0) {  // (the clock is read seldom: it takes longer than a probe)
      const long long now = nanoseconds();
      if (!since) since = now;
      out = out || now - since >= C.tiles_wait;
    }
    if (__any_sync(0xffffffffu, out)) break;
  }
  *lost = 1;
  give_up(C);
  return false;
}
// Those that compute wait for these two, or for tiles that the first one will miss (kMost: at last).
__device__ __forceinline__ bool wait_here(Stages& S, uint64_t* bar, uint32_t parity) {
  constexpr uint32_t kMost = 1u << 28;
  volatile int* const lost = &S.lost;
  for (uint32_t n = 0; n < kMost; ++n) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    if (__any_sync(0xffffffffu, *lost)) return false;
  }
  *lost = 1;
  atomicExch(&g_recurrence_status, TO_ERR_TIMEOUT);
  return false;
}

// A barrier of the eight warps; whether any of them has lost a wait.
__device__ __forceinline__ bool any_lost(bool lost) {
  int any;
  asm volatile(
      "{\n.reg .pred p, q;\nsetp.ne.s32 p, %1, 0;\nbar.red.or.pred q, 1, %2, p;\nselp.s32 %0, 1, 0, q;\n}"
      : "=r"(any)
      : "r"(static_cast<int>(lost)), "n"(kThreads)
      : "memory");
  return any != 0;
}
__device__ __forceinline__ void compute_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory"); }

__device__ __forceinline__ void arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ void open_stages(Stages& S) {
  if (threadIdx.x == 0) {
    S.lost = 0;
    for (int k = 0; k < 2; ++k) {
      mbar_init(&S.known[k], 1);
      mbar_init(&S.full[k], 1);
      mbar_init(&S.empty[k], kWarps + 1);
    }
    for (uint64_t& b : S.entered) mbar_init(&b, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
}

// The warp that looks ahead.  load(item, stage): one lane; fill(item, stage): the whole warp.
// A ticket is taken when its stage is free: the segments of a chain are in work at the same time,
// and a tile that is held for later keeps those behind it waiting (a tile ahead, 49152 tokens x
// 4096 channels took 328 us for 266, 4 x 4096 with 8-bit copies 134 for 129, without them 86 for 90).
template <bool BACKWARD, typename UNUSED, typename FILL, typename LOAD>
__device__ __forceinline__ void look_ahead(const Chain& C, Stages& S, UNUSED&& unused, FILL&& fill, LOAD&& load) {
  const int lane = threadIdx.x & 31;
  Order order(C, lane);
  unsigned ticket = blockIdx.x;
  if (C.ticket) next_ticket(C, ticket, lane);
  for (uint32_t k = 0;; ++k) {
    const int stage = k & 1;
    auto free = [&] { return k < 2 || wait_for(C, S, &S.empty[stage], (k / 2 - 1) & 1); };
    auto drain = [&] {  // the tiles before this one have landed
      for (uint32_t j = k < 2 ? 0 : k - 2; j < k; ++j) {
        if (mbar_wait_bounded(&S.full[j & 1], j / 2 & 1, kDrain)) continue;
        *const_cast<volatile int*>(&S.lost) = 1;
        give_up(C);
      }
    };
    if (!free()) return drain();
    if (k) next_ticket(C, ticket, lane);
    const Item it = next_item<BACKWARD>(C, order, ticket, lane, unused);
    if (lane == 0) {
      S.items[stage] = it;
      arrive(&S.known[stage]);
      if (it.slot >= 0 && it.n > 0) load(it, stage);
    }
    if (it.slot >= 0) fill(it, stage);  // (while the tile is on its way)
    else drain();                       // (nor may the last tiles outlive a CTA that ends early)
    __syncwarp();
    if (lane == 0) arrive(&S.full[stage]);
    if (it.slot < 0) return;
  }
}

// The warp that finds what enters.  first(item): what enters a sequence; done(item, state).
template <typename T, bool BACKWARD, typename FIRST, typename DONE>
__device__ __forceinline__ void find_entering(const Chain& C, Stages& S, Vals<Lane<T>::kVec> (&enter)[4][32], FIRST&& first,
                                              DONE&& done) {
  const int lane = threadIdx.x & 31;
  for (uint32_t k = 0;; ++k) {
    const int stage = k & 1;
    if (!wait_for(C, S, &S.known[stage], k / 2 & 1)) return;
    const Item it = S.items[stage];
    __syncwarp();
    if (lane == 0) arrive(&S.empty[stage]);
    if (it.slot < 0) return;
    const int p = BACKWARD ? it.count - 1 - it.idx : it.idx;
    const Links<T> links{C, lane, it.slab, it.slot - (BACKWARD ? -p : p), BACKWARD ? -1 : 1, p, it.count};
    const Vals<Lane<T>::kVec> e = p > 0 ? links.entering() : first(it);
    links.publish_state(e);
    enter[k & 3][lane] = e;
    __syncwarp();
    if (lane == 0) arrive(&S.entered[k & 3]);
    done(it, e);
  }
}

template <typename T, bool KEEP, bool COMPLEMENT, bool TMA>
__global__ void __launch_bounds__(kLaunched, 2) forward_kernel(const __grid_constant__ ForwardArgs A) {
  using L = Lane<T>;
  using P = typename L::P;
  constexpr int V = L::kVec, CH = L::kChannels, kTok = kSegment / kWarps, kTile = kSegment * kRowBytes;
  extern __shared__ __align__(128) char tiles[];  // two stages of x and f
  __shared__ Map<V> all_maps[2][kWarps][32];
  __shared__ P enter[4][32], biases[2][32];
  __shared__ Stages S;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Chain& C = A.C;
  open_stages(S);
  if (warp == kAhead) {
    look_ahead<false>(
        C, S, [](const Item&) {},
        [&](const Item& it, int stage) {
          P b = all<V>(0.f);
#pragma unroll
          for (int v = 0; v < V; ++v)
            if (A.bias && it.slab * CH + lane * V + v < C.channels)
              b.v[v] = __ldg(A.bias + it.slab * CH + lane * V + v);
          biases[stage][lane] = b;
        },
        [&](const Item& it, int stage) {
          if (!TMA) return;
          char* to = tiles + stage * 2 * kTile;
          expect_bytes(&S.full[stage], 2 * kTile);
          tma_tile(to, &A.x_map, it.slab * CH, it.row0, &S.full[stage]);
          tma_tile(to + kTile, &A.f_map, it.slab * CH, it.row0, &S.full[stage]);
        });
    return;
  }
  auto state_of = [&](const Item& it) {  // the place of the sequence's state; -1: none
    const long long slot = A.slots ? __ldg(A.slots + it.seq) : it.seq;
    return slot >= 0 && slot < A.num_slots ? slot * C.channels + it.slab * CH + lane * V : -1;
  };
  if (warp == kEntering) {
    find_entering<T, false>(
        C, S, enter,
        [&](const Item& it) {
          P e = all<V>(0.f);
          const long long state = A.state_in ? state_of(it) : -1;
#pragma unroll
          for (int v = 0; v < V; ++v)
            if (state >= 0 && it.slab * CH + lane * V + v < C.channels) e.v[v] = A.state_in[state + v];
          return e;
        },
        [&](const Item& it, const P& e) {
          if (!A.saved) return;
          const int c = it.slab * CH + lane * V;
#pragma unroll
          for (int v = 0; v < V; ++v)
            if (c + v < C.channels) A.saved[static_cast<long long>(it.slot) * C.channels + c + v] = e.v[v];
        });
    return;
  }
  auto fetch = [&](int stage) {  // the next tile, by the warps that compute
    const Item& it = S.items[stage];
    char* to = tiles + stage * 2 * kTile;
    if (it.slot >= 0 && it.n > 0) {
      load_rows<T>(to, A.x, A.x_access, it, it.slab * CH, C.channels);
      load_rows<T>(to + kTile, A.f, A.f_access, it, it.slab * CH, C.channels);
    }
    close_tiles();
  };
  const P log2e = kept(all<V>(kLog2e));
  bool lost = false;
  auto next_tile = [&](uint32_t t) {  // (not TMA) asks for it
    lost = lost || !wait_here(S, &S.full[t & 1], t / 2 & 1);
    if (!lost) fetch(t & 1);
  };
  if (!TMA) next_tile(0);
  for (uint32_t turn = 0;; ++turn) {
    const int stage = turn & 1;
    if (TMA) {
      lost = lost || !wait_here(S, &S.full[stage], turn / 2 & 1);
    } else {
      wait_tiles<0>();
      lost = any_lost(lost);
    }
    if (lost || S.items[stage].slot < 0) {  // (where others have a tile, they come to the barrier behind the reduction)
      any_lost(lost);
      break;
    }
    const Item it = S.items[stage];
    char* const xs = tiles + stage * 2 * kTile;
    char* const fs = xs + kTile;
    const int ch = it.slab * CH, c0 = ch + lane * V, nc = min(V, C.channels - c0), t0 = warp * kTok;
    if (KEEP) {
      if (A.keep_x.codes) keep_tile<T>(xs, A.keep_x, A.keep_access, it, ch, C.channels);
      if (A.keep_f.codes) keep_tile<T>(fs, A.keep_f, A.keep_access, it, ch, C.channels);
    }
    // the map of a warp's first tokens, up to every one of them
    P a[kTok], h[kTok];
    const P bias = biases[stage][lane];
    P at = all<V>(1.f), ht = all<V>(0.f);
    auto reduce = [&](auto whole) {
#pragma unroll
      for (int i = 0; i < kTok; ++i) {
        const P f = L::unpack(*reinterpret_cast<const uint32_t*>(fs + (t0 + i) * kRowBytes + lane * 4));
        const P x = L::unpack(*reinterpret_cast<const uint32_t*>(xs + (t0 + i) * kRowBytes + lane * 4));
        const P c = gate_of(argument_of(f, bias, log2e)), as = decayed(c, at), hs = stepped<COMPLEMENT>(c, x, ht);
        // a token that is not there changes nothing, whatever lies in its place (selected: with a branch
        // around each, their gates follow one another; 11 prompts 47 us, then 45)
        const bool there = decltype(whole)::value || t0 + i < it.n;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          at.v[v] = there ? as.v[v] : at.v[v];
          ht.v[v] = there ? hs.v[v] : ht.v[v];
        }
        a[i] = at, h[i] = ht;
      }
    };
    if (it.n == kSegment) reduce(std::true_type{});
    else reduce(std::false_type{});
    const Map<V> own{at, ht};
    Map<V>(*const maps)[32] = all_maps[stage];
    maps[warp][lane] = own;
    __syncwarp();
    if (any_lost(false)) break;
    if (!TMA) next_tile(turn + 1);
    const Links<T> links{C, lane, it.slab, it.slot - it.idx, 1, it.idx, it.count};
    Map<V> upto{all<V>(1.f), all<V>(0.f)};  // of the warps before this one
#pragma unroll
    for (int w = 0; w < kWarps - 1; ++w)
      if (w < warp) upto = upto.then(maps[w][lane]);
    const bool last = warp == kWarps - 1;
    if (last) links.publish_map(upto.then(own));
    P e = all<V>(__int_as_float(0x7fc00000));
    if (wait_here(S, &S.entered[turn & 3], turn / 4 & 1)) e = enter[turn & 3][lane];
    else lost = true;
    if (lane == 0) arrive(&S.empty[stage]);  // (the tile was read before the barrier)
    if (last && A.state_out && it.idx == it.count - 1) {
      const long long state = state_of(it);
      const P left = upto.then(own)(e);
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (state >= 0 && v < nc) A.state_out[state + v] = left.v[v];
    }
    e = upto(e);
    T* row = seq::row_ptr<T>(A.h, it.row0 + static_cast<long long>(t0), 0) + c0;
    if (A.pairs && nc == V && it.n == kSegment) {
#pragma unroll
      for (int i = 0; i < kTok; ++i, row += A.h.ts) *reinterpret_cast<uint32_t*>(row) = L::pack(fma(a[i], e, h[i]));
    } else {
#pragma unroll
      for (int i = 0; i < kTok; ++i)
        if (t0 + i < it.n) store_word<T>(row + i * A.h.ts, L::pack(fma(a[i], e, h[i])), nc, A.pairs);
    }
  }
}

// ---- backward ----------------------------------------------------------------------

struct BackwardArgs {
  CUtensorMap x_map, f_map, dh_map;  // (TMA)
  Chain C;
  Source x, f;
  Rows dh, dx, df;
  int dh_access, pairs;
  const float* bias;
  const float* saved;
  const float* dstate_out;
  float* dstate_in;
  float* partial;  // [slots][slabs * kChannels] sums of df; null: not wanted
};

// The gradients' own chain runs from a sequence's end: what leaves token t is a_t G_t,
// with G_t = dh_t + what left token t + 1; the map of some tokens is their A and what
// leaves them when nothing enters.  h runs forwards again from the saved state (so
// the map (A, H) of each warp is needed too).  x and dh stay in shared memory until the
// last walk.
// A stage: x and f as they are (or their codes at the same places), dh.
constexpr int kBackwardStage = 3 * kSegment * kRowBytes;

template <typename T, bool COMPLEMENT, bool TMA>
__global__ void __launch_bounds__(kLaunched, 2) backward_kernel(const __grid_constant__ BackwardArgs A) {
  using L = Lane<T>;
  using P = typename L::P;
  constexpr int V = L::kVec, CH = L::kChannels, kGroups = CH / seq::kGroup8;
  constexpr int kTok = kSegment / kWarps, kTile = kSegment * kRowBytes, kStage = kBackwardStage;
  extern __shared__ __align__(128) char tiles[];  // two stages
  // maps: of h, ends: of the gradients' chain (they share A)
  __shared__ Map<V> maps[kWarps][32], ends[kWarps][32];
  __shared__ P enter[4][32], biases[2][32], firsts[2][32];
  __shared__ float sums[kWarps][CH];
  __shared__ float scales[2][2][kSegment][kGroups];
  __shared__ Stages S;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Chain& C = A.C;
  open_stages(S);
  if (warp == kAhead) {
    look_ahead<true>(
        C, S,
        [&](const Item& it) {  // its sums count too
          if (A.partial)
#pragma unroll
            for (int v = 0; v < V; ++v)
              A.partial[(static_cast<long long>(it.slot) * C.slabs + it.slab) * CH + lane * V + v] = 0.f;
        },
        [&](const Item& it, int stage) {
          const int ch = it.slab * CH;
          P b = all<V>(0.f), first = all<V>(0.f);
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const int c = ch + lane * V + v;
            if (c >= C.channels) continue;
            if (A.bias) b.v[v] = __ldg(A.bias + c);
            first.v[v] = __ldg(A.saved + static_cast<long long>(it.slot) * C.channels + c);
          }
          biases[stage][lane] = b;
          firsts[stage][lane] = first;
          // scales: all of them asked for before the first is waited for (rows and groups that are
          // not there: others in their place)
          constexpr int kRows = kSegment / 32;
          uint8_t bytes[2][kRows][kGroups];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const Packed& from = k ? A.f.packed : A.x.packed;
            if (!from.codes || it.n <= 0) continue;
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
              const uint8_t* row = from.scales + (it.row0 + static_cast<long long>(min(32 * r + lane, it.n - 1))) * from.scale_stride;
#pragma unroll
              for (int j = 0; j < kGroups; ++j) bytes[k][r][j] = __ldg(row + min(ch / 32 + j, (C.channels - 1) / 32));
            }
          }
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            if (!(k ? A.f.packed : A.x.packed).codes || it.n <= 0) continue;
#pragma unroll
            for (int r = 0; r < kRows; ++r)
#pragma unroll
              for (int j = 0; j < kGroups; ++j) scales[stage][k][32 * r + lane][j] = seq::scale_of(bytes[k][r][j]);
          }
        },
        [&](const Item& it, int stage) {
          if (!TMA) return;
          char* to = tiles + stage * kStage;
          const int ch = it.slab * CH, x = A.x.packed.codes ? kSegment * CH : kTile, f = A.f.packed.codes ? kSegment * CH : kTile;
          expect_bytes(&S.full[stage], x + f + kTile);
          tma_tile(to, &A.x_map, ch, it.row0, &S.full[stage]);
          tma_tile(to + kTile, &A.f_map, ch, it.row0, &S.full[stage]);
          tma_tile(to + 2 * kTile, &A.dh_map, ch, it.row0, &S.full[stage]);
        });
    return;
  }
  if (warp == kEntering) {
    find_entering<T, true>(
        C, S, enter,
        [&](const Item& it) {
          P e = all<V>(0.f);
          const int c = it.slab * CH + lane * V;
#pragma unroll
          for (int v = 0; v < V; ++v)
            if (A.dstate_out && c + v < C.channels) e.v[v] = __ldg(A.dstate_out + static_cast<long long>(it.seq) * C.channels + c + v);
          return e;
        },
        [](const Item&, const P&) {});
    return;
  }
  auto fetch = [&](int stage) {  // the next tile, by the warps that compute
    const Item& it = S.items[stage];
    char* to = tiles + stage * kStage;
    if (it.slot >= 0 && it.n > 0) {
      const int ch = it.slab * CH;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const Source& from = k ? A.f : A.x;
        if (from.packed.codes)
          load_tile<CH>(from.access, to + k * kTile,
                        reinterpret_cast<const char*>(from.packed.codes) + it.row0 * from.packed.code_stride + ch,
                        from.packed.code_stride, it.n, C.channels - ch);
        else
          load_rows<T>(to + k * kTile, from.rows, from.access, it, ch, C.channels);
      }
      load_rows<T>(to + 2 * kTile, A.dh, A.dh_access, it, ch, C.channels);
    }
    close_tiles();
  };
  const P log2e = kept(all<V>(kLog2e)), offset = kept(all<V>(-8388736.f));
  bool lost = false;
  auto next_tile = [&](uint32_t t) {  // (not TMA) asks for it
    lost = lost || !wait_here(S, &S.full[t & 1], t / 2 & 1);
    if (!lost) fetch(t & 1);
  };
  if (!TMA) next_tile(0);
  for (uint32_t turn = 0;; ++turn) {
    const int stage = turn & 1;
    if (TMA) {
      lost = lost || !wait_here(S, &S.full[stage], turn / 2 & 1);
    } else {
      wait_tiles<0>();
      lost = any_lost(lost);
    }
    const Item& it = S.items[stage];  // (read again where it is used: registers are short)
    if (lost || it.slot < 0) {        // (where others have a tile, they come to the barrier behind the reduction)
      any_lost(lost);
      break;
    }
    const char* const xs = tiles + stage * kStage;
    const char* const fs = xs + kTile;
    const char* const gs = fs + kTile;
    const int c0 = it.slab * CH + lane * V, nc = min(V, C.channels - c0), t0 = warp * kTok;
    const int group = lane * V / seq::kGroup8;
    auto value = [&](const char* tile, int k, int t) {  // of rows in 8 bits
      const float scale = scales[stage][k][t][group];
      P out;
      if constexpr (V == 2) {
        const uint32_t both = *reinterpret_cast<const uint16_t*>(tile + t * CH + lane * V) ^ 0x8080u;  // codes + 128
        out = {{__uint_as_float(0x4b000000u | (both & 0xffu)), __uint_as_float(0x4b000000u | (both >> 8))}};
        out = mul(add(out, offset), all<V>(scale));
      } else {
        out.v[0] = seq::code_to_f32(reinterpret_cast<const int8_t*>(tile)[t * CH + lane], scale);
      }
      return out;
    };
    auto dh_of = [&](int i) { return L::unpack(*reinterpret_cast<const uint32_t*>(gs + (t0 + i) * kRowBytes + lane * 4)); };
    P c[kTok], w[kTok];  // c[i] is t before; w: x, then -df_t / G_t
    const P bias = biases[stage][lane];
    if (A.f.packed.codes) {
#pragma unroll
      for (int i = 0; i < kTok; ++i) c[i] = argument_of(value(fs, 1, t0 + i), bias, log2e);
    } else {
#pragma unroll
      for (int i = 0; i < kTok; ++i)
        c[i] = argument_of(L::unpack(*reinterpret_cast<const uint32_t*>(fs + (t0 + i) * kRowBytes + lane * 4)), bias, log2e);
    }
    P a = all<V>(1.f), h = all<V>(0.f), r = all<V>(0.f);
    if (A.x.packed.codes) {
#pragma unroll
      for (int i = 0; i < kTok; ++i) w[i] = value(xs, 0, t0 + i);
    } else {
#pragma unroll
      for (int i = 0; i < kTok; ++i) w[i] = L::unpack(*reinterpret_cast<const uint32_t*>(xs + (t0 + i) * kRowBytes + lane * 4));
    }
    const bool whole = it.n == kSegment;  // (a token that is not there changes nothing)
    auto reduce = [&](auto all_there) {
#pragma unroll
      for (int i = 0; i < kTok; ++i) {
        if (!decltype(all_there)::value && t0 + i >= it.n) continue;
        c[i] = gate_of(c[i]);
        a = decayed(c[i], a);
        h = stepped<COMPLEMENT>(c[i], w[i], h);
        r = fma(a, dh_of(i), r);  // what leaves the first token is the sum of a_0 .. a_t dh_t
      }
    };
    if (whole) reduce(std::true_type{});
    else reduce(std::false_type{});
    maps[warp][lane] = {a, h};
    const Map<V> own{a, r};
    ends[warp][lane] = own;
    if (any_lost(false)) break;
    const int p = it.count - 1 - it.idx;
    const Links<T> links{C, lane, it.slab, it.slot + p, -1, p, it.count};
    // joined from the last warp on: the first one has the segment's map
    Map<V> upto{all<V>(1.f), all<V>(0.f)};
#pragma unroll
    for (int k = kWarps - 1; k > 0; --k)
      if (k > warp) upto = upto.then(ends[k][lane]);
    if (warp == 0) links.publish_map(upto.then(own));
    // the states before every token, and -df_t / G_t
    h = firsts[stage][lane];
#pragma unroll
    for (int k = 0; k < kWarps - 1; ++k)
      if (k < warp) h = maps[k][lane](h);
    auto walk = [&](auto all_there) {
#pragma unroll
      for (int i = 0; i < kTok; ++i) {
        if (!decltype(all_there)::value && t0 + i >= it.n) continue;
        const P x = w[i], square = mul(c[i], c[i]);
        P slope;  // -a (1 - a)
#pragma unroll
        for (int v = 0; v < V; ++v) slope.v[v] = square.v[v] - fabsf(c[i].v[v]);
        w[i] = mul(slope, COMPLEMENT ? sub(h, x) : h);
        h = stepped<COMPLEMENT>(c[i], x, h);
      }
    };
    if (whole) walk(std::true_type{});
    else walk(std::false_type{});
    compute_sync();  // (maps and ends have been read)
    P e = all<V>(__int_as_float(0x7fc00000));
    if (wait_here(S, &S.entered[turn & 3], turn / 4 & 1)) e = enter[turn & 3][lane];
    else lost = true;
    if (warp == 0 && A.dstate_in && it.idx == 0) {
      const P left = upto.then(own)(e);
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (v < nc) A.dstate_in[static_cast<long long>(it.seq) * C.channels + c0 + v] = left.v[v];
    }
    e = upto(e);
    P sum = all<V>(0.f);
    T* dx = seq::row_ptr<T>(A.dx, it.row0 + static_cast<long long>(t0), 0) + c0;
    T* df = seq::row_ptr<T>(A.df, it.row0 + static_cast<long long>(t0), 0) + c0;
    e = mul(e, all<V>(-1.f));
    auto finish = [&](auto all_there, auto words) {  // with -G and -e
#pragma unroll
      for (int i = kTok - 1; i >= 0; --i) {
        if (!decltype(all_there)::value && t0 + i >= it.n) continue;
        const P G = sub(e, dh_of(i)), of = mul(G, w[i]);
        P ox;
        if (COMPLEMENT) {  // (1 - a) G
          P base;
#pragma unroll
          for (int v = 0; v < V; ++v) base.v[v] = is_rest(c[i].v[v]) ? 0.f : -G.v[v];
          ox = fma(c[i], G, base);
        } else {
          ox = mul(G, all<V>(-1.f));
        }
        e = decayed(c[i], G);
        const uint32_t wx = L::pack(ox), wf = L::pack(of);
        if (decltype(words)::value) {
          *reinterpret_cast<uint32_t*>(dx + i * A.dx.ts) = wx;
          *reinterpret_cast<uint32_t*>(df + i * A.df.ts) = wf;
        } else {
          store_word<T>(dx + i * A.dx.ts, wx, nc, A.pairs);
          store_word<T>(df + i * A.df.ts, wf, nc, A.pairs);
        }
        sum = add(sum, of);
      }
    };
    if (whole && A.pairs && nc == V) finish(std::true_type{}, std::true_type{});
    else finish(std::false_type{}, std::false_type{});
    if (A.partial) {
#pragma unroll
      for (int v = 0; v < V; ++v) sums[warp][lane * V + v] = sum.v[v];
    }
    const long long sums_at = (static_cast<long long>(it.slot) * C.slabs + it.slab) * CH;
    __syncwarp();
    if (lane == 0) arrive(&S.empty[stage]);
    if (!TMA) next_tile(turn + 1);
    if (A.partial) {
      compute_sync();
      if (threadIdx.x < CH) {
        float total = 0.f;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) total += sums[k][threadIdx.x];
        A.partial[sums_at + threadIdx.x] = total;
      }
    }
  }
}

// dbias[c] = sum over the segments of their sums, in a fixed order, in f64; NaN where the call gave up
// (sums may be missing; calls that wait for no maps have no flag of their own).
__global__ void __launch_bounds__(1024) bias_sum_kernel(const float* __restrict__ partial, long long pitch, int slots,
                                                        int channels, const int* gave_up, float* dbias) {
  __shared__ double part[32][33];
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5, x = blockIdx.x * 32 + lane;
  double v = 0;
  if (x < channels) {
#pragma unroll 8
    for (int c = row; c < slots; c += 32) v += partial[c * pitch + x];
  }
  part[row][lane] = v;
  __syncthreads();
  if (row == 0 && x < channels) {
    for (int k = 1; k < 32; ++k) v += part[k][lane];
    const int missing = gave_up ? *gave_up : *const_cast<const volatile int*>(&g_recurrence_status);
    dbias[x] = missing ? __int_as_float(0x7fc00000) : static_cast<float>(v);
  }
}

// ---- one token ---------------------------------------------------------------------

struct StepArgs {
  Rows x, f, h;
  const float* bias;
  const int32_t* slots;
  float* state;
  long long num_slots, units;  // units: tokens * (channels / V)
  int channels, complement;
};

template <typename T, int V>
__global__ void __launch_bounds__(256) step_kernel(const __grid_constant__ StepArgs A) {
  const int per = A.channels / V;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < A.units; i += gridDim.x * 256ll) {
    const long long token = i / per;
    const int c = static_cast<int>(i - token * per) * V;
    const long long slot = A.slots ? __ldg(A.slots + token) : token;
    float h[V], x[V], f[V];
    T* out = seq::row_ptr<T>(A.h, token, 0) + c;
    if (slot < 0 || slot >= A.num_slots) {
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = 0.f;
      seq::store_vec<T, V>(out, h);
      continue;
    }
    float* state = A.state + slot * A.channels + c;
    seq::load_vec<float, V>(state, h);
    seq::load_vec<T, V>(seq::row_ptr<const T>(A.x, token, 0) + c, x);
    seq::load_vec<T, V>(seq::row_ptr<const T>(A.f, token, 0) + c, f);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const Vals<1> b{{A.bias ? __ldg(A.bias + c + v) : 0.f}}, fv{{f[v]}}, xv{{x[v]}}, hv{{h[v]}};
      const Vals<1> g = gate_of(argument_of(fv, b, all<1>(kLog2e)));
      h[v] = (A.complement ? stepped<true>(g, xv, hv) : stepped<false>(g, xv, hv)).v[0];
    }
    seq::store_vec<float, V>(state, h);
    seq::store_vec<T, V>(out, h);
  }
}

// ---- host --------------------------------------------------------------------------

constexpr size_t kAlign = 256;
size_t padded(size_t n) { return (n + kAlign - 1) / kAlign * kAlign; }

int check_desc(const char* who, const to_gated_recurrence_desc* desc) {
  if (!desc) return set_error(TO_ERR_INVALID_ARGUMENT, "%s: null descriptor", who);
  const to_gated_recurrence_desc& d = *desc;
  if (d.dtype != TO_F32 && d.dtype != TO_BF16)
    return set_error(TO_ERR_UNSUPPORTED, "%s: dtype %d (built: f32, bf16)", who, d.dtype);
  if (d.channels < 1 || d.channels > 65536)
    return set_error(TO_ERR_UNSUPPORTED, "%s: %d channels (1 .. 65536)", who, d.channels);
  if (d.complement != 0 && d.complement != 1)
    return set_error(TO_ERR_INVALID_ARGUMENT, "%s: complement %d", who, d.complement);
  if (d.nseq < 0 || d.nseq > 65535)
    return set_error(TO_ERR_INVALID_ARGUMENT, "%s: %d sequences (0 .. 65535)", who, d.nseq);
  if (d.tokens < 0 || d.tokens > INT32_MAX)
    return set_error(TO_ERR_INVALID_ARGUMENT, "%s: %lld tokens", who, (long long)d.tokens);
  if (d.num_slots < 0) return set_error(TO_ERR_INVALID_ARGUMENT, "%s: %lld slots", who, (long long)d.num_slots);
  return ok();
}

int channels_of_tile(const to_gated_recurrence_desc& d) { return kRowBytes / seq::dtype_bytes(d.dtype); }
int slabs_of(const to_gated_recurrence_desc& d) {
  return (d.channels + channels_of_tile(d) - 1) / channels_of_tile(d);
}
// Segments that there may be, whatever the lengths are.
int slots_of(const to_gated_recurrence_desc& d) { return static_cast<int>(d.tokens / kSegment) + d.nseq; }
bool chained(const to_gated_recurrence_desc& d) { return d.tokens > kSegment && d.nseq > 0; }

struct Layout {  // of the workspace: the counter, the maps and the states (cleared), the partial sums
  size_t maps, states, partial, end;
};
Layout layout_of(const to_gated_recurrence_desc& d, bool backward) {
  const size_t values = size_t(slots_of(d)) * slabs_of(d) * channels_of_tile(d);
  Layout l{};
  if (chained(d)) {
    l.maps = kAlign;
    l.states = l.maps + padded(values * sizeof(uint64_t));
    l.partial = l.states + padded(values * sizeof(uint64_t));
  }
  l.end = l.partial + (backward && d.nseq ? padded(values * sizeof(float)) : 0);
  return l;
}

int check_list(const char* who, const char* name, const void* p, bool needed) {
  if (!p) return needed ? set_error(TO_ERR_INVALID_ARGUMENT, "%s: %s is null", who, name) : ok();
  return aligned(p, 4) ? ok() : set_error(TO_ERR_ALIGNMENT, "%s: %s is not 4-byte aligned", who, name);
}

int check_state(const char* who, const char* name, const void* p) {
  return aligned(p, 16) ? ok() : set_error(TO_ERR_ALIGNMENT, "%s: %s is not 16-byte aligned", who, name);
}

int check_workspace(const char* who, const void* p, size_t bytes, size_t need) {
  if (!need) return ok();
  if (!p || bytes < need)
    return set_error(TO_ERR_INVALID_ARGUMENT, "%s: workspace %zu < %zu bytes", who, p ? bytes : 0, need);
  return aligned(p, kAlign) ? ok() : set_error(TO_ERR_ALIGNMENT, "%s: workspace is not 256-byte aligned", who);
}

// The bytes that one access to rows may take.
int access_of(const to_rows& r, int64_t tokens, int32_t dtype) {
  int n = 16;
  while (n > seq::dtype_bytes(dtype) && !seq::rows_aligned(&r, tokens, 1, dtype, n)) n /= 2;
  return n;
}
int access_of(const to_rows8& r, int64_t tokens) {
  int n = 16;
  while (n > 1 && !(aligned(r.codes, n) && (tokens <= 1 || r.code_stride % n == 0))) n /= 2;
  return n;
}

// Whether TMA takes rows (the smallest calls do without the two tensor maps), and their tensor map.
bool tma_takes(const to_rows& r, const to_gated_recurrence_desc& d) {
  return d.tokens >= kSegment && r.token_stride < (1ll << 37) && seq::rows_aligned(&r, d.tokens, 1, d.dtype, 16);
}
int map_of(CUtensorMap* map, CUtensorMapDataType type, int bytes, const void* data, long long pitch, int row,
           const to_gated_recurrence_desc& d) {
  int st = ok();
  const EncodeTiled encode = tensor_map_encoder(&st);
  if (!encode) return st;
  const cuuint64_t dims[2] = {cuuint64_t(d.channels), cuuint64_t(d.tokens)}, strides[1] = {cuuint64_t(pitch * bytes)};
  const cuuint32_t box[2] = {cuuint32_t(row / bytes), cuuint32_t(kSegment)}, steps[2] = {1, 1};
  const CUresult e = encode(map, type, 2, const_cast<void*>(data), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return e == CUDA_SUCCESS ? ok() : set_error(TO_ERR_CUDA, "cuTensorMapEncodeTiled: %d", static_cast<int>(e));
}
bool tma_takes(const to_rows8& r, const to_gated_recurrence_desc& d) {
  return d.tokens >= kSegment && r.code_stride < (1ll << 37) && aligned(r.codes, 16) && r.code_stride % 16 == 0;
}
int map_of(CUtensorMap* map, const to_rows8& r, const to_gated_recurrence_desc& d) {
  return map_of(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, r.codes, r.code_stride, channels_of_tile(d), d);
}
int map_of(CUtensorMap* map, const to_rows& r, const to_gated_recurrence_desc& d) {
  return d.dtype == TO_BF16 ? map_of(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, r.data, r.token_stride, kRowBytes, d)
                            : map_of(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, r.data, r.token_stride, kRowBytes, d);
}

std::atomic<long long> g_maps_wait{kMapsWait}, g_tiles_wait{kTilesWait};  // microseconds

Chain chain_of(const to_gated_recurrence_desc& d, const int32_t* cu, const Layout& l, void* workspace) {
  Chain C{};
  C.maps_wait = 1000 * g_maps_wait.load(std::memory_order_relaxed);
  C.tiles_wait = 1000 * g_tiles_wait.load(std::memory_order_relaxed);
  C.cu = cu;
  C.nseq = d.nseq;
  C.tokens = static_cast<int>(d.tokens);
  C.channels = d.channels;
  C.slabs = slabs_of(d);
  C.slots = slots_of(d);
  if (chained(d)) {
    char* w = static_cast<char*>(workspace);
    C.ticket = reinterpret_cast<unsigned*>(w);
    C.gave_up = reinterpret_cast<int*>(w + sizeof(unsigned));
    C.maps = reinterpret_cast<uint64_t*>(w + l.maps);
    C.states = reinterpret_cast<uint64_t*>(w + l.states);
  }
  return C;
}

// CTAs of a launch: as many as fit the device, or as there are tiles.
unsigned grid_of(const Chain& C, int sms, int per_sm) {
  return static_cast<unsigned>(std::min(static_cast<long long>(C.slots) * C.slabs, static_cast<long long>(sms) * per_sm));
}

}  // namespace

int recurrence_device_status(int reset, int* value) {
  int v = 0;
  TO_CUDA_TRY(cudaMemcpyFromSymbol(&v, g_recurrence_status, sizeof(int)));
  if (reset && v) {
    const int z = 0;
    TO_CUDA_TRY(cudaMemcpyToSymbol(g_recurrence_status, &z, sizeof(int)));
  }
  *value = v;
  return ok();
}

}  // namespace to_b200

using namespace to_b200;

extern "C" {

int64_t to_gated_recurrence_saved_rows(const to_gated_recurrence_desc* desc) {
  return check_desc("to_gated_recurrence_saved_rows", desc) ? 0 : slots_of(*desc);
}

size_t to_gated_recurrence_workspace_bytes(const to_gated_recurrence_desc* desc) {
  return check_desc("to_gated_recurrence_workspace_bytes", desc) ? 0 : layout_of(*desc, false).end;
}

size_t to_gated_recurrence_backward_workspace_bytes(const to_gated_recurrence_desc* desc) {
  return check_desc("to_gated_recurrence_backward_workspace_bytes", desc) ? 0 : layout_of(*desc, true).end;
}

int to_gated_recurrence_wait_limits(int64_t maps_us, int64_t tiles_us) {
  constexpr int64_t kMost = 3600ll * 1000000;
  if (maps_us > kMost || tiles_us > kMost)
    return set_error(TO_ERR_INVALID_ARGUMENT, "to_gated_recurrence_wait_limits: %lld, %lld us", (long long)maps_us,
                     (long long)tiles_us);
  g_maps_wait.store(maps_us < 0 ? kMapsWait : maps_us, std::memory_order_relaxed);
  g_tiles_wait.store(tiles_us < 0 ? kTilesWait : tiles_us, std::memory_order_relaxed);
  return ok();
}

int to_gated_recurrence(const to_gated_recurrence_desc* desc, const to_gated_recurrence_args* args, void* stream) {
  const char* who = "to_gated_recurrence";
  if (int st = check_desc(who, desc)) return st;
  if (!args) return set_error(TO_ERR_INVALID_ARGUMENT, "%s: null arguments", who);
  const to_gated_recurrence_desc& d = *desc;
  const to_gated_recurrence_args& a = *args;
  if (d.nseq == 0) return ok();
  int st = seq::check_rows(who, "x", &a.x, d.tokens, 1, d.channels, d.dtype);
  if (!st) st = seq::check_rows(who, "f", &a.f, d.tokens, 1, d.channels, d.dtype);
  if (!st) st = seq::check_rows(who, "h", &a.h, d.tokens, 1, d.channels, d.dtype);
  if (!st && a.keep_x.codes) st = seq::check_rows8(who, "keep_x", a.keep_x, d.tokens, d.channels);
  if (!st && a.keep_f.codes) st = seq::check_rows8(who, "keep_f", a.keep_f, d.tokens, d.channels);
  if (!st) st = check_list(who, "bias", a.bias, false);
  if (!st) st = check_list(who, "cu_seqlens", a.cu_seqlens, true);
  if (!st) st = check_list(who, "slots", a.slots, false);
  if (!st) st = check_state(who, "state_in", a.state_in);
  if (!st) st = check_state(who, "state_out", a.state_out);
  if (!st) st = check_state(who, "saved", a.saved);
  const Layout l = layout_of(d, false);
  if (!st) st = check_workspace(who, a.workspace, a.workspace_bytes, l.end);
  if (st) return st;
  auto span = [&](const char* name, const to_rows& r) { return seq::span_of(name, &r, d.tokens, 1, d.channels, d.dtype); };
  const seq::Span spans[] = {span("h", a.h),
                             seq::codes_span("keep_x.codes", a.keep_x, d.tokens, d.channels),
                             seq::scales_span("keep_x.scales", a.keep_x, d.tokens, d.channels),
                             seq::codes_span("keep_f.codes", a.keep_f, d.tokens, d.channels),
                             seq::scales_span("keep_f.scales", a.keep_f, d.tokens, d.channels),
                             span("x", a.x), span("f", a.f)};
  if (d.tokens && (st = seq::check_apart(who, spans, 7, 5))) return st;
  const size_t states = size_t(a.slots ? d.num_slots : d.nseq) * d.channels * sizeof(float);
  if (a.state_in != a.state_out && seq::arrays_meet(a.state_in, a.state_out, states))
    return set_error(TO_ERR_INVALID_ARGUMENT, "%s: state_in and state_out share memory in part", who);
  for (const float* p : {a.state_in, static_cast<const float*>(a.state_out)})
    if (p && a.saved && p < a.saved + size_t(slots_of(d)) * d.channels && a.saved < p + states / sizeof(float))
      return seq::refuse_overlap(who, "saved", p == a.state_in ? "state_in" : "state_out");
  ForwardArgs A{};
  A.C = chain_of(d, a.cu_seqlens, l, a.workspace);
  A.x = seq::rows_of(a.x);
  A.f = seq::rows_of(a.f);
  A.h = seq::rows_of(a.h);
  A.x_access = access_of(a.x, d.tokens, d.dtype);
  A.f_access = access_of(a.f, d.tokens, d.dtype);
  A.pairs = access_of(a.h, d.tokens, d.dtype) >= 4;
  A.keep_x = seq::packed_of(a.keep_x);
  A.keep_f = seq::packed_of(a.keep_f);
  A.keep_access = 16;
  for (const to_rows8* k : {&a.keep_x, &a.keep_f})
    if (k->codes) A.keep_access = std::min(A.keep_access, access_of(*k, d.tokens));
  A.bias = a.bias;
  A.slots = a.slots;
  A.num_slots = a.slots ? d.num_slots : d.nseq;
  A.state_in = a.state_in;
  A.state_out = a.state_out;
  A.saved = a.saved;
  int dev = 0;
  const int sms = device_sm_count(&dev);
  if (sms <= 0) return -sms;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (A.C.ticket) TO_CUDA_TRY(cudaMemsetAsync(a.workspace, 0, l.partial, s));
  const unsigned grid = grid_of(A.C, sms, 2);
  constexpr size_t kShared = 4 * size_t(kSegment) * kRowBytes;
  static std::atomic<uint64_t> done[16];
  auto launch = [&](auto t, auto keep, auto complement, auto tma) {
    using K = decltype(keep);
    using M = decltype(complement);
    auto* kernel = forward_kernel<decltype(t), K::value, M::value, decltype(tma)::value>;
    const int which = 8 * (sizeof(t) == 4) + 4 * K::value + 2 * M::value + decltype(tma)::value;
    if (int bad = seq::allow_shared(kernel, kShared, done[which])) return bad;
    kernel<<<grid, kLaunched, kShared, s>>>(A);
    return ok();
  };
  const bool keep = a.keep_x.codes || a.keep_f.codes, tma = tma_takes(a.x, d) && tma_takes(a.f, d);
  if (tma && ((st = map_of(&A.x_map, a.x, d)) || (st = map_of(&A.f_map, a.f, d)))) return st;
  constexpr std::true_type yes{};
  constexpr std::false_type no{};
  auto with = [&](auto t, auto m) {
    if (tma) return keep ? launch(t, yes, m, yes) : launch(t, no, m, yes);
    return keep ? launch(t, yes, m, no) : launch(t, no, m, no);
  };
  if (d.dtype == TO_BF16) st = d.complement ? with(__nv_bfloat16{}, yes) : with(__nv_bfloat16{}, no);
  else st = d.complement ? with(float{}, yes) : with(float{}, no);
  if (st) return st;
  TO_CUDA_TRY(cudaGetLastError());
  return ok();
}

int to_gated_recurrence_backward(const to_gated_recurrence_desc* desc, const to_gated_recurrence_grad_args* args,
                                 void* stream) {
  const char* who = "to_gated_recurrence_backward";
  if (int st = check_desc(who, desc)) return st;
  if (!args) return set_error(TO_ERR_INVALID_ARGUMENT, "%s: null arguments", who);
  const to_gated_recurrence_desc& d = *desc;
  const to_gated_recurrence_grad_args& a = *args;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (int st = check_list(who, "dbias", a.dbias, false)) return st;
  if (d.nseq == 0) {
    if (a.dbias) TO_CUDA_TRY(cudaMemsetAsync(a.dbias, 0, sizeof(float) * d.channels, s));
    return ok();
  }
  int st = a.x8.codes ? seq::check_rows8(who, "x8", a.x8, d.tokens, d.channels)
                      : seq::check_rows(who, "x", &a.x, d.tokens, 1, d.channels, d.dtype);
  if (!st) st = a.f8.codes ? seq::check_rows8(who, "f8", a.f8, d.tokens, d.channels)
                           : seq::check_rows(who, "f", &a.f, d.tokens, 1, d.channels, d.dtype);
  if (!st) st = seq::check_rows(who, "dh", &a.dh, d.tokens, 1, d.channels, d.dtype);
  if (!st) st = seq::check_rows(who, "dx", &a.dx, d.tokens, 1, d.channels, d.dtype);
  if (!st) st = seq::check_rows(who, "df", &a.df, d.tokens, 1, d.channels, d.dtype);
  if (!st) st = check_list(who, "bias", a.bias, false);
  if (!st) st = check_list(who, "cu_seqlens", a.cu_seqlens, true);
  if (!st && !a.saved) st = set_error(TO_ERR_INVALID_ARGUMENT, "%s: saved is null", who);
  if (!st) st = check_state(who, "saved", a.saved);
  if (!st) st = check_state(who, "dstate_out", a.dstate_out);
  if (!st) st = check_state(who, "dstate_in", a.dstate_in);
  const Layout l = layout_of(d, true);
  if (!st) st = check_workspace(who, a.workspace, a.workspace_bytes, l.end);
  if (st) return st;
  auto span = [&](const char* name, const to_rows& r, bool there = true) {
    return there ? seq::span_of(name, &r, d.tokens, 1, d.channels, d.dtype) : seq::Span{};
  };
  const seq::Span spans[] = {span("dx", a.dx), span("df", a.df), span("dh", a.dh), span("x", a.x, !a.x8.codes),
                             span("f", a.f, !a.f8.codes), seq::codes_span("x8.codes", a.x8, d.tokens, d.channels),
                             seq::scales_span("x8.scales", a.x8, d.tokens, d.channels),
                             seq::codes_span("f8.codes", a.f8, d.tokens, d.channels),
                             seq::scales_span("f8.scales", a.f8, d.tokens, d.channels)};
  if (d.tokens && (st = seq::check_apart(who, spans, 9, 2))) return st;
  const size_t states = size_t(d.nseq) * d.channels;
  if (seq::arrays_meet(a.dstate_in, a.dstate_out, states * sizeof(float)))
    return seq::refuse_overlap(who, "dstate_in", "dstate_out");
  if (a.dstate_in && a.dstate_in < a.saved + size_t(slots_of(d)) * d.channels && a.saved < a.dstate_in + states)
    return seq::refuse_overlap(who, "dstate_in", "saved");
  for (const float* p : {static_cast<const float*>(a.dstate_in), a.dstate_out})
    if (a.dbias && p && a.dbias < p + states && p < a.dbias + d.channels)
      return seq::refuse_overlap(who, "dbias", p == a.dstate_in ? "dstate_in" : "dstate_out");
  if (a.dbias && a.dbias < a.saved + size_t(slots_of(d)) * d.channels && a.saved < a.dbias + d.channels)
    return seq::refuse_overlap(who, "dbias", "saved");
  BackwardArgs A{};
  A.C = chain_of(d, a.cu_seqlens, l, a.workspace);
  A.x = {seq::rows_of(a.x), seq::packed_of(a.x8), a.x8.codes ? access_of(a.x8, d.tokens) : access_of(a.x, d.tokens, d.dtype)};
  A.f = {seq::rows_of(a.f), seq::packed_of(a.f8), a.f8.codes ? access_of(a.f8, d.tokens) : access_of(a.f, d.tokens, d.dtype)};
  A.dh = seq::rows_of(a.dh);
  A.dx = seq::rows_of(a.dx);
  A.df = seq::rows_of(a.df);
  A.dh_access = access_of(a.dh, d.tokens, d.dtype);
  A.pairs = access_of(a.dx, d.tokens, d.dtype) >= 4 && access_of(a.df, d.tokens, d.dtype) >= 4;
  A.bias = a.bias;
  A.saved = a.saved;
  A.dstate_out = a.dstate_out;
  A.dstate_in = a.dstate_in;
  A.partial = a.dbias ? reinterpret_cast<float*>(static_cast<char*>(a.workspace) + l.partial) : nullptr;
  int dev = 0;
  const int sms = device_sm_count(&dev);
  if (sms <= 0) return -sms;
  if (A.C.ticket) TO_CUDA_TRY(cudaMemsetAsync(a.workspace, 0, l.partial, s));
  const unsigned grid = grid_of(A.C, sms, 2);
  constexpr size_t kShared = 2 * size_t(kBackwardStage);
  static std::atomic<uint64_t> done[8];
  auto launch = [&](auto t, auto complement, auto tma) {
    auto* kernel = backward_kernel<decltype(t), decltype(complement)::value, decltype(tma)::value>;
    const int which = 4 * (sizeof(t) == 4) + 2 * decltype(complement)::value + decltype(tma)::value;
    if (int bad = seq::allow_shared(kernel, kShared, done[which])) return bad;
    kernel<<<grid, kLaunched, kShared, s>>>(A);
    return ok();
  };
  const bool tma = tma_takes(a.dh, d) && (a.x8.codes ? tma_takes(a.x8, d) : tma_takes(a.x, d)) &&
                   (a.f8.codes ? tma_takes(a.f8, d) : tma_takes(a.f, d));
  if (tma) {
    st = a.x8.codes ? map_of(&A.x_map, a.x8, d) : map_of(&A.x_map, a.x, d);
    if (!st) st = a.f8.codes ? map_of(&A.f_map, a.f8, d) : map_of(&A.f_map, a.f, d);
    if (!st) st = map_of(&A.dh_map, a.dh, d);
    if (st) return st;
  }
  constexpr std::true_type yes{};
  constexpr std::false_type no{};
  auto with = [&](auto t) {
    if (tma) return d.complement ? launch(t, yes, yes) : launch(t, no, yes);
    return d.complement ? launch(t, yes, no) : launch(t, no, no);
  };
  st = d.dtype == TO_BF16 ? with(__nv_bfloat16{}) : with(float{});
  if (st) return st;
  TO_CUDA_TRY(cudaGetLastError());
  if (a.dbias) {
    bias_sum_kernel<<<(d.channels + 31) / 32, 1024, 0, s>>>(
        A.partial, static_cast<long long>(A.C.slabs) * channels_of_tile(d), A.C.slots, d.channels, A.C.gave_up, a.dbias);
    TO_CUDA_TRY(cudaGetLastError());
  }
  return ok();
}

int to_gated_recurrence_step(const to_gated_recurrence_desc* desc, const to_gated_recurrence_args* args, void* stream) {
  const char* who = "to_gated_recurrence_step";
  if (int st = check_desc(who, desc)) return st;
  if (!args) return set_error(TO_ERR_INVALID_ARGUMENT, "%s: null arguments", who);
  const to_gated_recurrence_desc& d = *desc;
  const to_gated_recurrence_args& a = *args;
  if (d.tokens == 0) return ok();
  int st = seq::check_rows(who, "x", &a.x, d.tokens, 1, d.channels, d.dtype);
  if (!st) st = seq::check_rows(who, "f", &a.f, d.tokens, 1, d.channels, d.dtype);
  if (!st) st = seq::check_rows(who, "h", &a.h, d.tokens, 1, d.channels, d.dtype);
  if (!st) st = check_list(who, "bias", a.bias, false);
  if (!st) st = check_list(who, "slots", a.slots, false);
  if (!st && !a.state_out) st = set_error(TO_ERR_INVALID_ARGUMENT, "%s: state_out is null", who);
  if (!st) st = check_state(who, "state_out", a.state_out);
  if (st) return st;
  auto span = [&](const char* name, const to_rows& r) { return seq::span_of(name, &r, d.tokens, 1, d.channels, d.dtype); };
  const seq::Span spans[] = {span("h", a.h), span("x", a.x), span("f", a.f)};
  if ((st = seq::check_apart(who, spans, 3, 1))) return st;
  StepArgs A{};
  A.x = seq::rows_of(a.x);
  A.f = seq::rows_of(a.f);
  A.h = seq::rows_of(a.h);
  A.bias = a.bias;
  A.slots = a.slots;
  A.state = a.state_out;
  A.num_slots = d.num_slots;
  A.channels = d.channels;
  A.complement = d.complement;
  const int e = seq::dtype_bytes(d.dtype);
  const bool vec = d.channels % 4 == 0 && access_of(a.x, d.tokens, d.dtype) >= 4 * e &&
                   access_of(a.f, d.tokens, d.dtype) >= 4 * e && access_of(a.h, d.tokens, d.dtype) >= 4 * e;
  A.units = d.tokens * (d.channels / (vec ? 4 : 1));
  int dev = 0;
  const int sms = device_sm_count(&dev);
  if (sms <= 0) return -sms;
  const unsigned grid = static_cast<unsigned>(std::min<long long>((A.units + 255) / 256, 64ll * sms));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (d.dtype == TO_BF16) {
    if (vec) step_kernel<__nv_bfloat16, 4><<<grid, 256, 0, s>>>(A);
    else step_kernel<__nv_bfloat16, 1><<<grid, 256, 0, s>>>(A);
  } else {
    if (vec) step_kernel<float, 4><<<grid, 256, 0, s>>>(A);
    else step_kernel<float, 1><<<grid, 256, 0, s>>>(A);
  }
  TO_CUDA_TRY(cudaGetLastError());
  return ok();
}

}  // extern "C"

// gated_recurrence.cu -- the gated linear recurrence of every channel
//   a_t = sigmoid(f_t + bias),  h_t = a_t h_{t-1} + (1 - a_t) x_t  (or + x_t),
// over packed sequences in one pass, its gradients in another, and the
// single-token step.
//
// The maps h -> A h + H compose: (A, H) then (A', H') is (A' A, A' H + H'), so a
// sequence is cut into segments of 128 tokens that are reduced at the same time
// and joined afterwards.  A CTA takes a segment and 128 bytes of channels (64 bf16
// or 32 f32, one or two a lane); each of its warps reduces 16 tokens, the maps of
// the warps are joined in shared memory, those of the segments through global
// memory while the CTAs run (below), and every warp then walks its tokens again
// from the state that enters them, out of registers.  So x and f are read once and
// h is written once, and 8 flops and two special functions a value (exp and a
// reciprocal) leave it memory bound.
//
// Gates: with u = exp(-|f|), u / (1 + u) is the smaller of a and 1 - a, accurate to
// f32 relative to itself.  It is kept with f's sign ("s": 1 - a where positive, -a
// where negative), and every step adds s times a difference to the larger term:
//   f >= 0:  h + (1 - a)(x - h)      f < 0:  x + a (h - x)
// so a memory of thousands of tokens does not take over a rounding of a near 1.
//
// Joining the segments: a CTA takes segments in the order of a counter (so a
// segment's predecessors have been taken by CTAs that run), publishes its map as
// soon as it has reduced its tokens, and folds the maps of its predecessors from
// the nearest one whose number is a multiple of 16, whose entering state is
// published too.  What is folded, and in which order, goes by the segment's number
// alone: results do not depend on timing.  Waits are bounded.
#include <algorithm>

#include "rows8.cuh"

namespace to_b200 {
namespace {

using seq::Packed;
using seq::Rows;

constexpr int kSegment = TO_RECURRENCE_SEGMENT;
constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr int kTok = kSegment / kWarps;  // tokens of a warp
constexpr int kRowBytes = 128;           // of a tile's row of values
constexpr int kChain = 16;               // segments between published states
constexpr uint32_t kPolls = 1u << 20;    // of a flag, about half a second

__device__ int g_recurrence_status;

template <typename T>
struct Lane {  // a lane's channels: one 32-bit word of a row
  static constexpr int kVec = 4 / int(sizeof(T));
  static constexpr int kChannels = kRowBytes / int(sizeof(T));  // of a tile
  __device__ __forceinline__ static void unpack(uint32_t w, float (&v)[kVec]) {
    if constexpr (kVec == 1) {
      v[0] = __uint_as_float(w);
    } else {
      v[0] = __uint_as_float(w << 16);
      v[1] = __uint_as_float(w & 0xffff0000u);
    }
  }
  __device__ __forceinline__ static uint32_t pack(const float (&v)[kVec]) {
    if constexpr (kVec == 1) {
      return __float_as_uint(v[0]);
    } else {
      const __nv_bfloat162 p = __floats2bfloat162_rn(v[0], v[1]);
      return *reinterpret_cast<const uint32_t*>(&p);
    }
  }
};

// How a call's segments lie, and what they share (see the head of the file).
struct Chain {
  const int32_t* cu;
  int nseq, tokens, channels, slabs, slots;  // slabs: tiles of channels; slots: segments that there may be
  unsigned long long* ticket;                // null: no sequence is longer than a segment
  int* gave_up;                              // set once a wait of this call has run out
  int* flags;                                // [slots][slabs][2]: the map, the entering state
  float2* maps;                              // [slots][slabs * kChannels]
  float* states;
};

struct Item {
  long long tile;  // number of the segment and slab; -1: no more
  int slot, slab, idx, count, seq, row0, n;
};

__device__ __forceinline__ int bound_of(const Chain& C, int s) {
  const int x = __ldg(C.cu + s);
  return x < 0 ? 0 : x > C.tokens ? C.tokens : x;
}

// The segment of slot w, by the warp together: sequence s owns the slots
// cu[s] / 128 + s and up, enough for its segments (an empty sequence has one).
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

template <bool BACKWARD, typename UNUSED>
__device__ __forceinline__ Item next_item(const Chain& C, unsigned long long ticket, int lane, UNUSED&& unused) {
  Item it;
  for (;;) {
    ticket = __shfl_sync(0xffffffffu, ticket, 0);
    const unsigned long long total = static_cast<unsigned long long>(C.slots) * C.slabs;
    if (ticket >= total) {
      it.tile = -1;
      return it;
    }
    const int at = static_cast<int>(ticket / C.slabs);
    it.slab = static_cast<int>(ticket - static_cast<unsigned long long>(at) * C.slabs);
    find_segment(C, BACKWARD ? C.slots - 1 - at : at, lane, it);
    it.tile = static_cast<long long>(it.slot) * C.slabs + it.slab;
    if (it.idx >= 0) return it;
    unused(it);  // a slot that no segment has
    if (C.ticket) {
      if (lane == 0) ticket = atomicAdd(C.ticket, 1ull);
    } else {
      ticket += gridDim.x;
    }
  }
}

// ---- tiles in shared memory ----------------------------------------------------------

// `rows` rows of ROWB bytes into shared memory, ACCESS bytes at a time; the
// columns from `valid` bytes on become zero.
template <int ACCESS, int ROWB>
__device__ __forceinline__ void load_tile(char* dst, const char* src, long long pitch, int rows, int valid) {
  constexpr int kPer = ROWB / ACCESS;
#pragma unroll 4
  for (int i = threadIdx.x; i < rows * kPer; i += kThreads) {
    const int row = i / kPer, col = (i % kPer) * ACCESS;
    const int bytes = max(0, min(ACCESS, valid - col));
    char* d = dst + row * ROWB + col;
    const char* s = bytes ? src + row * pitch + col : src;
    if constexpr (ACCESS >= 16) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                       static_cast<uint32_t>(__cvta_generic_to_shared(d))),
                   "l"(s), "r"(bytes)
                   : "memory");
    } else if constexpr (ACCESS >= 4) {
      asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(
                       static_cast<uint32_t>(__cvta_generic_to_shared(d))),
                   "l"(s), "n"(ACCESS), "r"(bytes)
                   : "memory");
    } else if constexpr (ACCESS == 2) {
      *reinterpret_cast<uint16_t*>(d) = bytes ? *reinterpret_cast<const uint16_t*>(s) : uint16_t(0);
    } else {
      *reinterpret_cast<uint8_t*>(d) = bytes ? *reinterpret_cast<const uint8_t*>(s) : uint8_t(0);
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

__device__ __forceinline__ void wait_tiles() {
  asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;" ::: "memory");
}

struct Source {  // x or f of a call: rows, or rows in 8 bits
  Rows rows;
  Packed packed;
  int access;  // bytes that one access may take
};

template <typename T>
__device__ __forceinline__ void load_rows(char* dst, const Rows& r, int access, const Item& it, int ch, int channels) {
  load_tile<kRowBytes>(access, dst, reinterpret_cast<const char*>(seq::row_ptr<const T>(r, it.row0, 0) + ch),
                       r.ts * static_cast<long long>(sizeof(T)), it.n, (channels - ch) * static_cast<int>(sizeof(T)));
}

// ---- the recurrence ------------------------------------------------------------------

// The smaller of sigmoid(f) and 1 - sigmoid(f), with f's sign.
__device__ __forceinline__ float gate_of(float f) {
  const float u = __expf(-fabsf(f));
  return copysignf(__fdividef(u, 1.f + u), f);
}
__device__ __forceinline__ bool is_decay(float s) { return __float_as_int(s) < 0; }
// a h
__device__ __forceinline__ float decayed(float s, float h) { return fmaf(-s, h, is_decay(s) ? 0.f : h); }
// one step of the recurrence
__device__ __forceinline__ float stepped(bool complement, float s, float x, float h) {
  return complement ? fmaf(s, x - h, is_decay(s) ? x : h) : fmaf(-s, h, is_decay(s) ? x : h + x);
}

// ---- segments joined while the CTAs run ------------------------------------------------

__device__ __forceinline__ int flag_at(const int* p) {
  int v;
  asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}

__device__ __forceinline__ void raise(int* p) {
  asm volatile("st.release.gpu.global.s32 [%0], 1;" ::"l"(p) : "memory");
}

// What one warp has to do with the other segments of its sequence: position p of
// `count` in the chain's direction, whose slots lie at origin + dir * position.
template <typename T>
struct Links {
  static constexpr int V = Lane<T>::kVec, CH = Lane<T>::kChannels;
  const Chain& C;
  int lane, slab, origin, dir, p, count;

  __device__ __forceinline__ int slot(int at) const { return origin + dir * at; }
  __device__ __forceinline__ int* flag(int at) const {
    return C.flags + (static_cast<long long>(slot(at)) * C.slabs + slab) * 2;
  }
  __device__ __forceinline__ long long place(int at) const {
    return (static_cast<long long>(slot(at)) * C.slabs + slab) * CH + lane * V;
  }
  // The segment's own map, for those behind it.
  __device__ __forceinline__ void publish_map(const float (&a)[V], const float (&h)[V]) const {
    if (p + 1 >= count) return;
#pragma unroll
    for (int v = 0; v < V; ++v) __stcg(C.maps + place(p) + v, make_float2(a[v], h[v]));
    __threadfence();
    __syncwarp();
    if (lane == 0) raise(flag(p));
  }
  __device__ __forceinline__ void publish_state(const float (&h)[V]) const {
    if (p + 1 >= count || p % kChain) return;
#pragma unroll
    for (int v = 0; v < V; ++v) __stcg(C.states + place(p) + v, h[v]);
    __threadfence();
    __syncwarp();
    if (lane == 0) raise(flag(p) + 1);
  }
  // The state that enters position p > 0.
  __device__ __forceinline__ void entering(float (&h)[V]) const {
    const int base = (p - 1) / kChain * kChain, n = p - base;
    const int* f = lane < n ? flag(base + lane) : lane == kChain ? flag(base) + 1 : nullptr;
    bool waiting = f != nullptr;
    for (uint32_t polls = 0; __any_sync(0xffffffffu, waiting); ++polls) {
      if (waiting && flag_at(f)) waiting = false;
      if (polls % 256 == 255) {  // (once a wait has run out, the others of the call need not)
        const bool out = polls > kPolls || flag_at(C.gave_up);
        if (waiting && out) {
          atomicExch(C.gave_up, 1);
          atomicExch(&g_recurrence_status, TO_ERR_TIMEOUT);
          waiting = false;
        }
      }
    }
    __syncwarp();
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = __ldcg(C.states + place(base) + v);
#pragma unroll 8
    for (int k = 0; k < n; ++k) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float2 m = __ldcg(C.maps + place(base + k) + v);
        h[v] = fmaf(m.x, h[v], m.y);
      }
    }
  }
};

// ---- forward -----------------------------------------------------------------------

struct ForwardArgs {
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
  int complement;
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
#pragma unroll
    for (int k = 0; k < 16; ++k) most = max(most, seq::abs_bits(x[k]));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    const int byte = seq::scale_byte(most);
    const float inverse = seq::inverse_scale(byte);
    union { uint4 v; uint32_t w[4]; uint8_t b[16]; } u;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      u.w[k] = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) u.w[k] |= seq::code_of(x[4 * k + j], inverse, byte != 255) << (8 * j);
    }
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

template <typename T, bool KEEP>
__global__ void __launch_bounds__(kThreads, 3) forward_kernel(const __grid_constant__ ForwardArgs A) {
  using L = Lane<T>;
  constexpr int V = L::kVec, CH = L::kChannels;
  __shared__ alignas(16) char xs[kSegment * kRowBytes];
  __shared__ alignas(16) char fs[kSegment * kRowBytes];
  __shared__ float2 maps[kWarps][CH];
  __shared__ float enter[CH];
  __shared__ Item items[2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Chain& C = A.C;
  const bool complement = A.complement;
  unsigned long long ticket = blockIdx.x;
  auto take = [&] {
    if (C.ticket) {
      if (lane == 0) ticket = atomicAdd(C.ticket, 1ull);
    } else {
      ticket += gridDim.x;
    }
  };
  auto fetch = [&](const Item& it) {
    if (it.tile < 0 || it.n <= 0) return;
    load_rows<T>(xs, A.x, A.x_access, it, it.slab * CH, C.channels);
    load_rows<T>(fs, A.f, A.f_access, it, it.slab * CH, C.channels);
  };
  auto no_slot = [](const Item&) {};
  if (warp == kWarps - 1) {
    if (C.ticket && lane == 0) ticket = atomicAdd(C.ticket, 1ull);
    const Item first = next_item<false>(C, ticket, lane, no_slot);
    if (!C.ticket && first.tile >= 0) ticket = first.tile;
    if (lane == 0) items[0] = first;
  }
  __syncthreads();
  fetch(items[0]);
  for (int cur = 0;; cur ^= 1) {
    const Item it = items[cur];
    if (it.tile < 0) break;
    wait_tiles();
    __syncthreads();
    if (warp == kWarps - 1) take();
    const int ch = it.slab * CH, c0 = ch + lane * V, nc = min(V, C.channels - c0);
    if (KEEP) {
      if (A.keep_x.codes) keep_tile<T>(xs, A.keep_x, A.keep_access, it, ch, C.channels);
      if (A.keep_f.codes) keep_tile<T>(fs, A.keep_f, A.keep_access, it, ch, C.channels);
    }
    float bias[V], a[V], h[V], s[kTok][V];
    uint32_t x[kTok];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      bias[v] = A.bias && v < nc ? __ldg(A.bias + c0 + v) : 0.f;
      a[v] = 1.f, h[v] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < kTok; ++i) {
      const int t = warp * kTok + i;
      x[i] = 0;
#pragma unroll
      for (int v = 0; v < V; ++v) s[i][v] = 0.f;  // (a token that is not there changes nothing)
      if (t < it.n) {
        x[i] = *reinterpret_cast<const uint32_t*>(xs + t * kRowBytes + lane * 4);
        float f[V];
        L::unpack(*reinterpret_cast<const uint32_t*>(fs + t * kRowBytes + lane * 4), f);
#pragma unroll
        for (int v = 0; v < V; ++v) s[i][v] = gate_of(f[v] + bias[v]);
      }
      float xv[V];
      L::unpack(x[i], xv);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        a[v] = decayed(s[i][v], a[v]);
        h[v] = stepped(complement, s[i][v], xv[v], h[v]);
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) maps[warp][lane * V + v] = make_float2(a[v], h[v]);
    if (warp == kWarps - 1) {
      const Item next = next_item<false>(C, ticket, lane, no_slot);
      if (!C.ticket && next.tile >= 0) ticket = next.tile;
      if (lane == 0) items[cur ^ 1] = next;
    }
    __syncthreads();
    fetch(items[cur ^ 1]);  // the tiles have been read
    if (warp == 0) {
#pragma unroll
      for (int v = 0; v < V; ++v) a[v] = 1.f, h[v] = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float2 m = maps[w][lane * V + v];
          a[v] *= m.x;
          h[v] = fmaf(m.x, h[v], m.y);
        }
      const Links<T> links{C, lane, it.slab, it.slot - it.idx, 1, it.idx, it.count};
      links.publish_map(a, h);
      const long long state = A.slots ? __ldg(A.slots + it.seq) : it.seq;
      const bool has_state = state >= 0 && state < A.num_slots;
      float e[V];
      if (it.idx > 0) {
        links.entering(e);
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v)
          e[v] = A.state_in && has_state && v < nc ? A.state_in[state * C.channels + c0 + v] : 0.f;
      }
      links.publish_state(e);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        enter[lane * V + v] = e[v];
        if (v < nc) {
          if (A.saved) A.saved[static_cast<long long>(it.slot) * C.channels + c0 + v] = e[v];
          if (A.state_out && has_state && it.idx == it.count - 1)
            A.state_out[state * C.channels + c0 + v] = fmaf(a[v], e[v], h[v]);
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = enter[lane * V + v];
    for (int w = 0; w < warp; ++w)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float2 m = maps[w][lane * V + v];
        h[v] = fmaf(m.x, h[v], m.y);
      }
    T* row = seq::row_ptr<T>(A.h, it.row0 + static_cast<long long>(warp * kTok), 0) + c0;
#pragma unroll
    for (int i = 0; i < kTok; ++i) {
      float xv[V];
      L::unpack(x[i], xv);
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = stepped(complement, s[i][v], xv[v], h[v]);
      if (warp * kTok + i < it.n) store_word<T>(row + i * A.h.ts, L::pack(h), nc, A.pairs);
    }
  }
}

// ---- backward ----------------------------------------------------------------------

struct BackwardArgs {
  Chain C;
  Source x, f;
  Rows dh, dx, df;
  int dh_access, pairs;
  const float* bias;
  const float* saved;
  const float* dstate_out;
  float* dstate_in;
  float* partial;  // [slots][slabs * kChannels] sums of df; null: not wanted
  int complement;
};

// The gradients' own chain runs from a sequence's end: what leaves token t is a_t G_t,
// with G_t = dh_t + what left token t + 1; the map of some tokens is their A and what
// leaves them when nothing enters.  h runs forwards again from the saved state (so
// the map (A, H) of each warp is needed too).
template <typename T>
__global__ void __launch_bounds__(kThreads, 2) backward_kernel(const __grid_constant__ BackwardArgs A) {
  using L = Lane<T>;
  constexpr int V = L::kVec, CH = L::kChannels, kGroups = CH / seq::kGroup8;
  extern __shared__ __align__(16) char tiles[];
  char* const xs = tiles;
  char* const fs = tiles + kSegment * kRowBytes;
  char* const gs = tiles + 2 * kSegment * kRowBytes;
  __shared__ float2 maps[kWarps][CH];
  __shared__ float ends[kWarps][CH], enter[CH], sums[kWarps][CH];
  __shared__ uint8_t scales[2][kSegment][kGroups];
  __shared__ Item items[2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Chain& C = A.C;
  const bool complement = A.complement;
  unsigned long long ticket = blockIdx.x;
  uint8_t byte[kGroups] = {};  // scales of the next tile, this thread's row
  auto fetch = [&](const Item& it) {
    if (it.tile < 0 || it.n <= 0) return;
    const int ch = it.slab * CH;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const Source& S = k ? A.f : A.x;
      char* dst = k ? fs : xs;
      if (!S.packed.codes) {
        load_rows<T>(dst, S.rows, S.access, it, ch, C.channels);
        continue;
      }
      load_tile<CH>(S.access, dst, reinterpret_cast<const char*>(S.packed.codes) + it.row0 * S.packed.code_stride + ch,
                    S.packed.code_stride, it.n, C.channels - ch);
      const int row = threadIdx.x % kSegment;
      if (static_cast<int>(threadIdx.x) / kSegment == k && row < it.n) {
        const uint8_t* from = S.packed.scales + (it.row0 + static_cast<long long>(row)) * S.packed.scale_stride + ch / 32;
#pragma unroll
        for (int j = 0; j < kGroups; ++j) byte[j] = ch + 32 * j < C.channels ? __ldg(from + j) : 0;
      }
    }
    load_rows<T>(gs, A.dh, A.dh_access, it, ch, C.channels);
  };
  auto no_slot = [&](const Item& it) {  // its sums count too
    if (A.partial)
#pragma unroll
      for (int v = 0; v < V; ++v) A.partial[it.tile * CH + lane * V + v] = 0.f;
  };
  if (warp == kWarps - 1) {
    if (C.ticket && lane == 0) ticket = atomicAdd(C.ticket, 1ull);
    const Item first = next_item<true>(C, ticket, lane, no_slot);
    if (!C.ticket && first.tile >= 0)
      ticket = static_cast<unsigned long long>(C.slots - 1 - first.slot) * C.slabs + first.slab;
    if (lane == 0) items[0] = first;
  }
  __syncthreads();
  fetch(items[0]);
  for (int cur = 0;; cur ^= 1) {
    const Item it = items[cur];
    if (it.tile < 0) break;
    wait_tiles();
#pragma unroll
    for (int j = 0; j < kGroups; ++j) scales[threadIdx.x / kSegment][threadIdx.x % kSegment][j] = byte[j];
    __syncthreads();
    if (warp == kWarps - 1) {
      if (C.ticket) {
        if (lane == 0) ticket = atomicAdd(C.ticket, 1ull);
      } else {
        ticket += gridDim.x;
      }
    }
    const int ch = it.slab * CH, c0 = ch + lane * V, nc = min(V, C.channels - c0);
    const int group = lane * V / seq::kGroup8;
    float a[V], h[V], r[V], bias[V], first[V], s[kTok][V], w[kTok][V];
    uint32_t x[kTok], g[kTok];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      bias[v] = A.bias && v < nc ? __ldg(A.bias + c0 + v) : 0.f;
      first[v] = v < nc ? __ldg(A.saved + static_cast<long long>(it.slot) * C.channels + c0 + v) : 0.f;
      a[v] = 1.f, h[v] = r[v] = 0.f;
    }
    auto value = [&](const char* tile, int k, int t, float (&out)[V]) {  // of rows in 8 bits
      const float scale = seq::scale_of(scales[k][t][group]);
      const int8_t* code = reinterpret_cast<const int8_t*>(tile) + t * CH + lane * V;
#pragma unroll
      for (int v = 0; v < V; ++v) out[v] = seq::code_to_f32(code[v], scale);
    };
#pragma unroll
    for (int i = 0; i < kTok; ++i) {
      const int t = warp * kTok + i;
      x[i] = g[i] = 0;
#pragma unroll
      for (int v = 0; v < V; ++v) s[i][v] = 0.f;
      if (t < it.n) {
        float f[V], xv[V];
        if (A.x.packed.codes) {
          value(xs, 0, t, xv);
          x[i] = L::pack(xv);  // (7 bits and a sign: exact)
        } else {
          x[i] = *reinterpret_cast<const uint32_t*>(xs + t * kRowBytes + lane * 4);
        }
        if (A.f.packed.codes) value(fs, 1, t, f);
        else L::unpack(*reinterpret_cast<const uint32_t*>(fs + t * kRowBytes + lane * 4), f);
        g[i] = *reinterpret_cast<const uint32_t*>(gs + t * kRowBytes + lane * 4);
#pragma unroll
        for (int v = 0; v < V; ++v) s[i][v] = gate_of(f[v] + bias[v]);
      }
      float xv[V];
      L::unpack(x[i], xv);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        a[v] = decayed(s[i][v], a[v]);
        h[v] = stepped(complement, s[i][v], xv[v], h[v]);
      }
    }
#pragma unroll
    for (int i = kTok - 1; i >= 0; --i) {
      float gv[V];
      L::unpack(g[i], gv);
#pragma unroll
      for (int v = 0; v < V; ++v) r[v] = decayed(s[i][v], gv[v] + r[v]);
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      maps[warp][lane * V + v] = make_float2(a[v], h[v]);
      ends[warp][lane * V + v] = r[v];
    }
    if (warp == kWarps - 1) {
      const Item next = next_item<true>(C, ticket, lane, no_slot);
      if (!C.ticket && next.tile >= 0)
        ticket = static_cast<unsigned long long>(C.slots - 1 - next.slot) * C.slabs + next.slab;
      if (lane == 0) items[cur ^ 1] = next;
    }
    __syncthreads();
    fetch(items[cur ^ 1]);
    if (warp == 0) {
#pragma unroll
      for (int v = 0; v < V; ++v) a[v] = 1.f, r[v] = 0.f;
#pragma unroll
      for (int k = kWarps - 1; k >= 0; --k)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float m = maps[k][lane * V + v].x;
          a[v] *= m;
          r[v] = fmaf(m, r[v], ends[k][lane * V + v]);
        }
      const int p = it.count - 1 - it.idx;
      const Links<T> links{C, lane, it.slab, it.slot + p, -1, p, it.count};
      links.publish_map(a, r);
      float e[V];
      const long long state = static_cast<long long>(it.seq) * C.channels + c0;
      if (p > 0) {
        links.entering(e);
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v) e[v] = A.dstate_out && v < nc ? __ldg(A.dstate_out + state + v) : 0.f;
      }
      links.publish_state(e);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        enter[lane * V + v] = e[v];
        if (A.dstate_in && it.idx == 0 && v < nc) A.dstate_in[state + v] = fmaf(a[v], e[v], r[v]);
      }
    }
    // the states before every token, and df_t / G_t
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = first[v];
    for (int k = 0; k < warp; ++k)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float2 m = maps[k][lane * V + v];
        h[v] = fmaf(m.x, h[v], m.y);
      }
#pragma unroll
    for (int i = 0; i < kTok; ++i) {
      float xv[V];
      L::unpack(x[i], xv);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float small = fabsf(s[i][v]);
        w[i][v] = fmaf(-small, small, small) * (complement ? h[v] - xv[v] : h[v]);
        h[v] = stepped(complement, s[i][v], xv[v], h[v]);
      }
    }
    __syncthreads();
    float sum[V];
#pragma unroll
    for (int v = 0; v < V; ++v) r[v] = enter[lane * V + v], sum[v] = 0.f;
    for (int k = kWarps - 1; k > warp; --k)
#pragma unroll
      for (int v = 0; v < V; ++v) r[v] = fmaf(maps[k][lane * V + v].x, r[v], ends[k][lane * V + v]);
    T* dx = seq::row_ptr<T>(A.dx, it.row0 + static_cast<long long>(warp * kTok), 0) + c0;
    T* df = seq::row_ptr<T>(A.df, it.row0 + static_cast<long long>(warp * kTok), 0) + c0;
#pragma unroll
    for (int i = kTok - 1; i >= 0; --i) {
      float gv[V], ox[V], of[V];
      L::unpack(g[i], gv);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float G = gv[v] + r[v];
        // (1 - a) G is s G, or G less a G
        r[v] = decayed(s[i][v], G);
        ox[v] = complement ? (is_decay(s[i][v]) ? fmaf(s[i][v], G, G) : s[i][v] * G) : G;
        of[v] = G * w[i][v];
      }
      if (warp * kTok + i < it.n) {
        store_word<T>(dx + i * A.dx.ts, L::pack(ox), nc, A.pairs);
        store_word<T>(df + i * A.df.ts, L::pack(of), nc, A.pairs);
#pragma unroll
        for (int v = 0; v < V; ++v) sum[v] += of[v];
      }
    }
    if (A.partial) {
#pragma unroll
      for (int v = 0; v < V; ++v) sums[warp][lane * V + v] = sum[v];
      __syncthreads();
      if (threadIdx.x < CH) {
        float total = 0.f;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) total += sums[k][threadIdx.x];
        A.partial[it.tile * CH + threadIdx.x] = total;
      }
    }
  }
}

// dbias[c] = sum over the segments of their sums, in a fixed order, in f64.
__global__ void __launch_bounds__(1024) bias_sum_kernel(const float* __restrict__ partial, long long pitch, int slots,
                                                        int channels, float* dbias) {
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
    dbias[x] = static_cast<float>(v);
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
    for (int v = 0; v < V; ++v)
      h[v] = stepped(A.complement, gate_of(f[v] + (A.bias ? __ldg(A.bias + c + v) : 0.f)), x[v], h[v]);
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

struct Layout {  // of the workspace: the counter and the flags, the maps, the states, the partial sums
  size_t flags, maps, states, partial, end;
};
Layout layout_of(const to_gated_recurrence_desc& d, bool backward) {
  const size_t tiles = size_t(slots_of(d)) * slabs_of(d), values = tiles * channels_of_tile(d);
  Layout l{};
  if (chained(d)) {
    l.flags = kAlign;
    l.maps = l.flags + padded(tiles * 2 * sizeof(int));
    l.states = l.maps + padded(values * sizeof(float2));
    l.partial = l.states + padded(values * sizeof(float));
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

Chain chain_of(const to_gated_recurrence_desc& d, const int32_t* cu, const Layout& l, void* workspace) {
  Chain C{};
  C.cu = cu;
  C.nseq = d.nseq;
  C.tokens = static_cast<int>(d.tokens);
  C.channels = d.channels;
  C.slabs = slabs_of(d);
  C.slots = slots_of(d);
  if (chained(d)) {
    char* w = static_cast<char*>(workspace);
    C.ticket = reinterpret_cast<unsigned long long*>(w);
    C.gave_up = reinterpret_cast<int*>(w + sizeof(unsigned long long));
    C.flags = reinterpret_cast<int*>(w + l.flags);
    C.maps = reinterpret_cast<float2*>(w + l.maps);
    C.states = reinterpret_cast<float*>(w + l.states);
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
  A.complement = d.complement;
  int dev = 0;
  const int sms = device_sm_count(&dev);
  if (sms <= 0) return -sms;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (A.C.ticket) TO_CUDA_TRY(cudaMemsetAsync(a.workspace, 0, l.maps, s));
  const unsigned grid = grid_of(A.C, sms, 3);
  const bool keep = a.keep_x.codes || a.keep_f.codes;
  if (d.dtype == TO_BF16) {
    if (keep) forward_kernel<__nv_bfloat16, true><<<grid, kThreads, 0, s>>>(A);
    else forward_kernel<__nv_bfloat16, false><<<grid, kThreads, 0, s>>>(A);
  } else {
    if (keep) forward_kernel<float, true><<<grid, kThreads, 0, s>>>(A);
    else forward_kernel<float, false><<<grid, kThreads, 0, s>>>(A);
  }
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
  A.complement = d.complement;
  int dev = 0;
  const int sms = device_sm_count(&dev);
  if (sms <= 0) return -sms;
  if (A.C.ticket) TO_CUDA_TRY(cudaMemsetAsync(a.workspace, 0, l.maps, s));
  const unsigned grid = grid_of(A.C, sms, 2);
  constexpr size_t kShared = 3 * size_t(kSegment) * kRowBytes;
  static std::atomic<uint64_t> done[2];
  if (d.dtype == TO_BF16) {
    if ((st = seq::allow_shared(backward_kernel<__nv_bfloat16>, kShared, done[0]))) return st;
    backward_kernel<__nv_bfloat16><<<grid, kThreads, kShared, s>>>(A);
  } else {
    if ((st = seq::allow_shared(backward_kernel<float>, kShared, done[1]))) return st;
    backward_kernel<float><<<grid, kThreads, kShared, s>>>(A);
  }
  TO_CUDA_TRY(cudaGetLastError());
  if (a.dbias) {
    bias_sum_kernel<<<(d.channels + 31) / 32, 1024, 0, s>>>(
        A.partial, static_cast<long long>(A.C.slabs) * channels_of_tile(d), A.C.slots, d.channels, a.dbias);
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

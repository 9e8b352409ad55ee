// linear_attention_tc.cu -- the decayed chain (linear_attention.cuh) of bf16
// rows on the 5th-generation tensor cores: tcgen05 + TMEM + TMA.
//
// A CTA takes one segment of one head and walks its chunks of 128 tokens.  With
// Q, K, V the chunk's rows of a, b, c (tiles of 128 x 128, narrower widths
// zero-filled by TMA) and X the state:
//   Sc = Q K^T                    P = Sc masked, decayed and scaled, bf16, in TMEM
//   O  = Q X (bf16 X), its rows scaled in TMEM by inter l^(..), then O += P V
//   U  = (decayed K)^T V          X = l^n X + U (f32, in registers)
// all M = N = 128.  Five or six products of 128^3 a chunk (one more in a sequence's
// first), 2560 or 3072 tensor cycles at the dense bf16 rate, against about 5600 for
// the chunk's 128 KB at this SM's share of the HBM.  A product of two shared operands
// of this size takes all of the shared memory's 128 bytes a cycle, so P and decayed K
// are TMEM operands (K transposed into its lanes by ldmatrix).
//
// Precision: P and X each enter their product with one bf16 rounding, as the
// result's own.  In the chain's first chunk of a sequence a row has few P and, where no
// state enters, nothing else, so that their errors do not average out: there P has a
// second plane, and the result of such a token is rounded once, whatever follows it.
// The state stays f32: decayed K is split into bf16 planes of 8 bits each -- three, which
// reach f32, where the sequence's state is a result, two where only products read it --
// smallest plane first, so few sums pass through the accumulator at full size; a chunk's
// U is added to X in IEEE f32 registers.  (Two planes for chunks that have decayed far by
// the sequence's end are not enough: the tokens after them may weigh nothing.)
//
// Roles (20 warps): one lane issues TMA loads, two chunks ahead, one the
// products; warps 4-11 turn Sc into P, scale O and store the results (a thread:
// one row, 64 columns); warps 12-19 make the planes and hold X (a thread: one row, 64
// columns).  Plane 2 lies in O's columns between one chunk's results and the
// next one's.  Products are issued U, Q X, P V and the next chunk's Sc: the row warps
// store results and make the next P while the state warps make the next planes.  In the states' launch there is
// no Sc and no O: both groups make planes, into two buffers in turn.  Rows past
// a chunk's end are masked: P by selection, K and V by zeroing their rows, since
// 0 * NaN is not 0.  Rows of a reversed chain keep their order in memory; only
// the masks and decays turn round.  For the same reason P V, where P is 0 for the tokens
// that a row does not see, may meet nothing but finite values: warps 2 and 3 look through
// V (a panel each) and, where they find others, note their tokens and take them out once U
// has had them; the row warps then make the results that see them NaN.
//
// Measured on B200, 49152 tokens x 16 heads x 128: outputs 197 to 204 us (4.0 TB/s, 0.61 of
// the copy rate), states 89 to 91 us (4.5 TB/s), each by itself; a call with the scan of 7 us
// 302 us, 350 us back to back on a hot card.  A chunk's outputs take about 7000 cycles:
// Q X, the scaling, P V, Sc and U wait for one another, and products with two shared
// operands take about 110 cycles each instead of 64.
//
// Every wait is bounded; on a timeout the kernel records TO_ERR_TIMEOUT in the
// device status word, waits (bounded) for its copies in flight, frees its TMEM
// and returns.
#include <cuda.h>

#include "linear_attention.cuh"
#include "sm100_primitives.cuh"
#include "tensor_map.hpp"

namespace to_b200 {
__device__ int g_sequence_status = 0;

namespace {

using lin::Chain;
using lin::Segment;

constexpr int kTile = 128;                       // tokens of a chunk, and the padded widths
constexpr uint32_t kPanel = kTile * 128;         // 128 rows of 64 values
constexpr uint32_t kTileBytes = 2 * kPanel;      // 32 KB
constexpr int kRowWarps = 8, kStateWarps = 8;    // P and out; planes and X
constexpr int kFirstRow = 4, kFirstState = kFirstRow + kRowWarps;  // warps 0, 1: loads, products; 2, 3: V
constexpr int kThreads = 32 * (kFirstState + kStateWarps);
constexpr uint32_t kMaxPolls = 1u << 22;
constexpr int kMaxStages = 3;

// Chunks in shared memory, 192 KB of them: tiles Q, K, V each, or K, V.
template <bool STATES>
struct Ring {
  static constexpr int kStages = STATES ? 3 : 2;
  static constexpr uint32_t kK = STATES ? 0 : kTileBytes, kV = kK + kTileBytes, kBytes = kV + kTileBytes;
};

// TMEM columns.  P of each 16 tokens overwrites the first half of their columns of Sc, its
// second plane the other half.
constexpr uint32_t kColS = 0, kColO = 128;
template <bool STATES>
constexpr uint32_t kColU = STATES ? 0 : 256;
// Plane p of a chunk, tokens [64 h, 64 h + 64): 32 columns.
template <bool STATES>
__device__ __forceinline__ uint32_t plane_col(uint32_t chunk, int p, int h) {
  if (STATES) return 128 + 192 * (chunk & 1) + 64 * p + 32 * h;
  return p == 2 ? kColO + 64 * h : 384 + 64 * p + 32 * h;
}

struct Barriers {
  uint64_t full[kMaxStages], empty[kMaxStages];      // (Q and) K of a chunk
  uint64_t full_v[kMaxStages], empty_v[kMaxStages];  // its V
  // once a chunk each
  uint64_t sc_full, p_ready, o1_full, o_free;
  uint64_t planes_ready, u_full, u_free, x_ready;
  // a chunk's stage: V without what is not finite, and then P V; whether a panel had any, and the
  // first token (in the chain's direction) of each column that had
  uint64_t clean[2], o2_full[2];
  int odd[2][2];
  uint32_t tmem;
  int abort;
  alignas(16) int seen[2][kTile];
};

__device__ __forceinline__ bool wait_for(Barriers* b, uint64_t* bar, uint32_t parity) {
  for (uint32_t i = 0; i < kMaxPolls; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 15) == 15 && *reinterpret_cast<volatile int*>(&b->abort)) return false;
  }
  atomicExch(&g_sequence_status, int(TO_ERR_TIMEOUT));
  atomicExch(&b->abort, 1);
  return false;
}

// The same by a whole warp, with one answer.
__device__ __forceinline__ bool warp_wait(Barriers* b, uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, wait_for(b, bar, parity));
}

// The same value, which the compiler takes for a new one: the descriptors made
// from it are not kept from one chunk to the next (they overflowed the uniform
// registers).
__device__ __forceinline__ uint32_t fresh(uint32_t x) {
  asm volatile("" : "+r"(x));
  return x;
}

__device__ __forceinline__ void arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ void tma_tile(uint32_t dst, const CUtensorMap* map, int head, int token, uint64_t* bar) {
#pragma unroll
  for (int p = 0; p < 2; ++p)
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(dst + p * kPanel), "l"(map), "r"(64 * p), "r"(head), "r"(token), "r"(smem_u32(bar))
        : "memory");
}

// Shared-memory descriptor, 128-byte swizzle.  K-major operands (rows of 64
// contiguous K values): 8-row groups 1024 bytes apart.  MN-major ones (rows of
// 64 contiguous M or N values, one row a K value): 8-K groups 1024 bytes apart
// (stride offset), the two 64-value panels kPanel apart (leading offset).
// The upper word is the same for both; steps add to the lower one (no carry:
// shared addresses end below 2^18).
constexpr uint32_t kDescHigh = (1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_k(uint32_t tile, int step) {  // 16 K values a step
  return ((tile >> 4) | (1u << 16)) + (step >> 2) * (kPanel >> 4) + (step & 3) * 2;
}
__device__ __forceinline__ uint32_t desc_mn(uint32_t tile, int step) {
  return ((tile >> 4) | ((kPanel >> 4) << 16)) + step * 128;
}

// D f32, A and B bf16, M = N = 128; bit 16: B is MN-major
constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(kTile >> 3) << 17) |
                            (uint32_t(kTile >> 4) << 24);
constexpr uint32_t kMnB = 1u << 16;

__device__ __forceinline__ void mma(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 da, {%1, %4};\n\tmov.b64 db, {%2, %4};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}"
      ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(kDescHigh), "r"(uint32_t(add)) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 db, {%2, %4};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}"
      ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(kDescHigh), "r"(uint32_t(add)) : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 32 columns of this thread's lane; the wait belongs to the statement, so the
// registers exist only once the load has completed
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float (&x)[32]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(x);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
      "%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const float (&x)[32]) {
  const uint32_t* r = reinterpret_cast<const uint32_t*>(x);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
      ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
        "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
        "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
// 16 lanes x 8 columns: register 2i / 2i+1 holds columns 4i .. 4i+3 of lanes
// 0-7 / 8-15, thread t lane t/4 (or 8 + t/4) and column t%4 of the four --
// what ldmatrix gives of 8 x 8 tiles.
__device__ __forceinline__ void tmem_st_tiles(uint32_t addr, const uint32_t (&r)[4]) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x2.b32 [%0], {%1,%2,%3,%4};"
               ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Four transposed 8 x 8 tiles of bf16; lane l gives the row address l%8 of tile l/8.
__device__ __forceinline__ void ldmatrix_t4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, float (&x)[16]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(x);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ uint32_t tmem_ld1(uint32_t addr) {
  uint32_t x;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=r"(x) : "r"(addr) : "memory");
  return x;
}
__device__ __forceinline__ void tmem_st1(uint32_t addr, uint32_t x) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(addr), "r"(x) : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

__device__ __forceinline__ float lds(uint32_t addr) {
  float x;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(addr));
  return x;
}
__device__ __forceinline__ uint4 lds4(uint32_t addr) {
  uint4 x;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(addr));
  return x;
}
__device__ __forceinline__ void sts1(uint32_t addr, uint32_t a) {
  asm volatile("st.shared.u32 [%0], %1;" ::"r"(addr), "r"(a) : "memory");
}
__device__ __forceinline__ void sts4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// Two bf16, lo: bits 0-15: zero times each added to sum, which stays +0 while all are finite.
__device__ __forceinline__ uint32_t add_zero_times(uint32_t x, uint32_t sum) {
  uint32_t r;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(0u), "r"(sum));
  return r;
}

// (lo, hi) as two bf16 in one register, lo in the low half
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float low_half(uint32_t r) { return __uint_as_float(r << 16); }
__device__ __forceinline__ float high_half(uint32_t r) { return __uint_as_float(r & 0xffff0000u); }

// Tables: l^n, n = 0 .. 128, and from 132 on the 32 factors of a block's columns;
// the first again times `upd`.
constexpr int kTable = 164, kUpdTable = 132;

// The segment of one head that a CTA walks.
struct Walk {
  int seq, head;
  bool begins, last, only;  // the sequence's first segment; its last; its only one
  int edge;             // first row of the segment (forwards), or the row after it (backwards)
  int len;              // its tokens
  int n, updates;       // chunks; those whose state is wanted (not the last's, where no one reads it)
  __device__ __forceinline__ int rows(int i) const { return min(len - i * kTile, kTile); }
  // First row in memory of chunk i.
  __device__ __forceinline__ int first(const Chain& C, int i) const {
    return C.rev ? edge - i * kTile - rows(i) : edge + i * kTile;
  }
};

// False: nothing to do there.
template <bool STATES>
__device__ __forceinline__ bool walk_of(const Chain& C, int item, Walk* w) {
  const int slot = item / C.heads;
  const Segment g = lin::segment_of(C, slot);
  if (g.idx < 0 || (STATES && g.idx == g.count - 1)) return false;
  const int s0 = g.idx * C.seg;  // no overflow: below the sequence's length
  w->seq = g.seq;
  w->head = item - slot * C.heads;
  w->begins = g.idx == 0;
  w->last = g.idx == g.count - 1;
  w->only = g.count == 1;
  w->len = min(C.seg, g.tokens - s0);
  w->edge = C.rev ? g.first + g.tokens - s0 : g.first + s0;
  w->n = (w->len + kTile - 1) / kTile;
  w->updates = STATES || (C.fin && w->last) ? w->n : w->n - 1;
  return true;
}

// Planes FROM .. TO-1 of decayed K: lanes [32 q, 32 q + 32) of K^T, tokens 64 h + 16 g
// .. for g of [g0, g1), from the chunk's tile of K; `lanes`: the quarter's TMEM address.
// All but the last plane (three says whether that is plane 2) are cut off, not rounded,
// so each is the product's own next eight bits.
template <bool STATES, int FROM, int TO>
__device__ __forceinline__ void make_planes(uint32_t tile, uint32_t lanes, uint32_t chunk, uint32_t dec, int cnt,
                                            bool rev, bool three, int q, int h, int g0, int g1, int lane) {
  const uint32_t panel = tile + (q >> 1) * kPanel;
  if (cnt < kTile) {  // rows past the end: zero what this warp reads
    for (int e = lane; e < 64 * (g1 - g0); e += 32) {
      const int row = 64 * h + 16 * g0 + (e >> 2);
      if (row >= cnt) sts4(panel + row * 128 + (((4 * (q & 1) + (e & 3)) ^ (row & 7)) << 4), 0, 0, 0, 0);
    }
    fence_async();  // before the tile is loaded again
    __syncwarp();
  }
  // tile m of an ldmatrix: rows 8 (m & 1) .. of 16 lanes, tokens 8 (m >> 1) .. of 16
  const int m = lane >> 3;
#pragma unroll 1
  for (int g = g0; g < g1; ++g) {
    const int row = 64 * h + 16 * g + 8 * (m >> 1) + (lane & 7);
    float2 d[2];
#pragma unroll
    for (int z = 0; z < 2; ++z) {
      const int j = 64 * h + 16 * g + 8 * z + 2 * (lane & 3), age = rev ? j + 1 : cnt - 1 - j;
      d[z] = make_float2(lds(dec + 4 * max(age, 0)), lds(dec + 4 * max(rev ? age + 1 : age - 1, 0)));
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint32_t k[4], out[TO][4];
      ldmatrix_t4(panel + row * 128 + (((4 * (q & 1) + 2 * half + (m & 1)) ^ (row & 7)) << 4), k);
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        float2 x = __fmul2_rn(make_float2(low_half(k[z]), high_half(k[z])), d[z >> 1]);
#pragma unroll
        for (int p = 0; p < TO; ++p) {
          if (p == 2 || (p == 1 && !three))
            out[p][z] = pack2(x.x, x.y);
          else
            out[p][z] = __byte_perm(__float_as_uint(x.x), __float_as_uint(x.y), 0x7632);
          if (p + 1 < TO)
            x = __ffma2_rn(make_float2(__uint_as_float(__float_as_uint(x.x) & 0xffff0000u),
                                       __uint_as_float(__float_as_uint(x.y) & 0xffff0000u)),
                           make_float2(-1.f, -1.f), x);
        }
      }
#pragma unroll
      for (int p = FROM; p < TO; ++p)
        tmem_st_tiles(lanes + (uint32_t(16 * half) << 16) + 8 * g + plane_col<STATES>(chunk, p, h), out[p]);
    }
  }
  tmem_st_wait();
}

// X of a warp (lane: a row, 64 columns from column `col` on) from or to rows row0 ..
// of a [db][dc] matrix (dc a multiple of 4, as tc_takes asks): through 2.5 KB of shared memory, 16
// columns at a time, so that four lanes take 64 bytes of one row.  (32 lanes in 32
// rows held up the load-store unit, and the other warps' shared loads behind it.)
__device__ __forceinline__ void load_state(float (&X)[64], const float* m, uint32_t stage, int row0, int col, int db,
                                           int dc, int lane) {
  float4 v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int row = row0 + 8 * (i & 3) + (lane >> 2), c = col + 16 * (i >> 2) + 4 * (lane & 3);
    v[i] = row < db && c < dc ? *reinterpret_cast<const float4*>(m + row * dc + c) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
#pragma unroll
  for (int g = 0; g < 4; ++g) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float4 x = v[4 * g + k];
      sts4(stage + (8 * k + (lane >> 2)) * 80 + (lane & 3) * 16, __float_as_uint(x.x), __float_as_uint(x.y),
           __float_as_uint(x.z), __float_as_uint(x.w));
    }
    __syncwarp();
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint4 x = lds4(stage + lane * 80 + 16 * e);
      X[16 * g + 4 * e] = __uint_as_float(x.x);
      X[16 * g + 4 * e + 1] = __uint_as_float(x.y);
      X[16 * g + 4 * e + 2] = __uint_as_float(x.z);
      X[16 * g + 4 * e + 3] = __uint_as_float(x.w);
    }
    __syncwarp();
  }
}

__device__ __forceinline__ void store_state(const float (&X)[64], float* m, uint32_t stage, int row0, int col, int db,
                                            int dc, int lane) {
#pragma unroll
  for (int g = 0; g < 4; ++g) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      sts4(stage + lane * 80 + 16 * e, __float_as_uint(X[16 * g + 4 * e]), __float_as_uint(X[16 * g + 4 * e + 1]),
           __float_as_uint(X[16 * g + 4 * e + 2]), __float_as_uint(X[16 * g + 4 * e + 3]));
    __syncwarp();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int r = 8 * k + (lane >> 2), c = col + 16 * g + 4 * (lane & 3);
      const uint4 x = lds4(stage + r * 80 + (lane & 3) * 16);
      if (row0 + r < db && c < dc) *reinterpret_cast<uint4*>(m + (row0 + r) * dc + c) = x;
    }
    __syncwarp();
  }
}

// Shared memory
constexpr uint32_t kX = 6 * kTileBytes;  // bf16 X, behind the chunks
constexpr uint32_t kTables = kX + kTileBytes;
constexpr uint32_t kBars = kTables + (kTable + kUpdTable) * 4;
constexpr uint32_t kSmem = kBars + sizeof(Barriers);
static_assert(Ring<true>::kStages * Ring<true>::kBytes <= kX && Ring<false>::kStages * Ring<false>::kBytes <= kX, "ring");
static_assert(kBars % 16 == 0 && kSmem <= 232448, "shared memory of a CTA");

// Registers: the launch gives each of the 20 warps 96; those that hold X take some of
// the others' (4 * 64 + 8 * 88 + 8 * 120 = 1920 = 20 * 96).  No kernel may
// spill: with the shared memory taken, a spilled register comes back from L2.  Loops
// stay rolled where registers allow it: the roles run different code at the same time,
// and unrolled they outgrow the instruction caches (stalls for want of instructions were
// three times the issued ones).
template <int N>
__device__ __forceinline__ void registers_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void registers_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }

template <int N>
struct Maps {
  CUtensorMap m[N][3];  // rows of a, b, c
};

template <bool STATES, int N>
__global__ void __launch_bounds__(kThreads, 1)
    chain_tc_kernel(const __grid_constant__ Maps<N> maps, const __grid_constant__ lin::Batch<N> batch) {
  const Chain& C = batch.c[N == 1 ? 0 : blockIdx.y];
  const CUtensorMap* map = maps.m[N == 1 ? 0 : blockIdx.y];
  using R = Ring<STATES>;
  constexpr int kStages = R::kStages;
  extern __shared__ __align__(1024) unsigned char sm[];
  const int item = blockIdx.x;  // segment slot * heads + head
  const float gl = lin::log_decay_of(C, item % C.heads);
  Walk w;
  if (!walk_of<STATES>(C, item, &w)) return;
  const uint32_t base = smem_u32(sm);
  if (base & 1023) {  // the swizzled tiles need it; there is no room left to round up in
    if (threadIdx.x == 0) atomicExch(&g_sequence_status, int(TO_ERR_SCRATCH));
    return;
  }
  Barriers* bar = reinterpret_cast<Barriers*>(sm + kBars);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool rev = C.rev != 0;
  const bool three = C.fin && (STATES || w.last);  // planes: the sequence's state is a result

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&bar->full[i], 1);
      mbar_init(&bar->full_v[i], 1);
      // Q and K are free when their products are done (a commit) and the planes made; V when
      // its products are done and the results, which pass through its tile, stored
      mbar_init(&bar->empty[i], kStateWarps + (STATES ? kRowWarps : 1));
      mbar_init(&bar->empty_v[i], STATES ? 1 : kRowWarps);
    }
    mbar_init(&bar->sc_full, 1);
    mbar_init(&bar->p_ready, kRowWarps);
    mbar_init(&bar->o1_full, 1);
    mbar_init(&bar->o_free, kRowWarps);
    mbar_init(&bar->planes_ready, kStateWarps + (STATES ? kRowWarps : 0));
    mbar_init(&bar->u_full, 1);
    mbar_init(&bar->u_free, kStateWarps);
    mbar_init(&bar->x_ready, kStateWarps);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar->clean[i], 2);
      mbar_init(&bar->o2_full[i], 3);  // the product, and the warps whose notes on V the row warps read
    }
    bar->abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  {
    float* table = reinterpret_cast<float*>(sm + kTables);
    for (int t = threadIdx.x; t < kTable + kUpdTable; t += kThreads) {
      const int n = t < 132 ? t : t < kTable ? (rev ? t - 132 : 163 - t) : t - kTable;
      table[t] = expf(gl * static_cast<float>(n)) * (t < kTable ? 1.f : C.upd);
    }
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&bar->tmem))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = bar->tmem, dec = base + kTables, dec_upd = dec + kTable * 4;
  auto stage_of = [&](uint32_t n) { return base + (STATES ? n % kStages : n & 1) * R::kBytes; };
  auto turn_of = [&](uint32_t n) { return (n / kStages) & 1; };
  bool ok = true;

  if (warp < kFirstRow) {
    registers_down<64>();
    if (warp == 0 && lane == 0) {
      // ---- loads: (Q,) K, V of each chunk ----
      int i = 0, qk = 0;
      for (; i < w.n; ++i) {
        const int token = w.first(C, i);
        uint64_t *full = &bar->full[i % kStages], *full_v = &bar->full_v[i % kStages];
        if (i >= kStages && !(ok = wait_for(bar, &bar->empty[i % kStages], turn_of(i - kStages)))) break;
        mbar_arrive_expect_tx(full, R::kV);
        if (!STATES) tma_tile(stage_of(i), map, w.head / C.a_div, token, full);
        tma_tile(stage_of(i) + R::kK, map + 1, w.head / C.b_div, token, full);
        qk = i + 1;
        if (i >= kStages && !(ok = wait_for(bar, &bar->empty_v[i % kStages], turn_of(i - kStages)))) break;
        mbar_arrive_expect_tx(full_v, kTileBytes);
        tma_tile(stage_of(i) + R::kV, map + 2, w.head / C.c_div, token, full_v);
      }
      // copies still in flight land before the CTA ends
      for (int t = qk > kStages ? qk - kStages : 0; t < qk; ++t) {
        mbar_wait_bounded(&bar->full[t % kStages], turn_of(t), kMaxPolls);
        if (t < i) mbar_wait_bounded(&bar->full_v[t % kStages], turn_of(t), kMaxPolls);
      }
    } else if (warp == 1 && lane == 0) {
      // ---- products ----
      auto scores = [&](int i) {
        const uint32_t sq = fresh(stage_of(i)), tm = fresh(tmem);
        if (!(ok = wait_for(bar, &bar->full[i % kStages], turn_of(i)))) return;
        fence_after();
#pragma unroll
        for (int k = 0; k < kTile / 16; ++k) mma(tm + kColS, desc_k(sq, k), desc_k(sq + R::kK, k), kIdesc, k > 0);
        commit(&bar->sc_full);
      };
      if (!STATES && w.n > 0) scores(0);
      for (int i = 0; i < w.n && ok; ++i) {
        const uint32_t turn = i & 1, sq = fresh(stage_of(i)), sv = sq + R::kV;
        const uint32_t tm = fresh(tmem), sx = fresh(base) + kX;
        if (i < w.updates) {
          const int planes = three ? 3 : 2;
          // (outputs: the state warps have read the last U before they make planes)
          if (!(ok = wait_for(bar, &bar->full_v[i % kStages], turn_of(i)) && wait_for(bar, &bar->planes_ready, turn) &&
                     (!STATES || i == 0 || wait_for(bar, &bar->u_free, turn ^ 1))))
            break;
          fence_after();
#pragma unroll 1
          for (int p = planes - 1; p >= 0; --p)
#pragma unroll
            for (int k = 0; k < kTile / 16; ++k)  // 16 tokens: 8 columns
              mma_ts(tm + kColU<STATES>, tm + plane_col<STATES>(i, p, k >> 2) + (k & 3) * 8, desc_mn(sv, k),
                     kIdesc | kMnB, p < planes - 1 || k > 0);
          commit(&bar->u_full);
        }
        if (!STATES) {
          // x_ready also says that V's rows past the end are zero
          if (!(ok = wait_for(bar, &bar->x_ready, turn) && (i == 0 || wait_for(bar, &bar->o_free, turn ^ 1)))) break;
          fence_after();
#pragma unroll
          for (int k = 0; k < kTile / 16; ++k)
            mma(tm + kColO, desc_k(sq, k), desc_mn(sx, k), kIdesc | kMnB, k > 0);
          commit(&bar->o1_full);
          commit(&bar->empty[i % kStages]);
          // (clean: V has come, too)
          if (!(ok = wait_for(bar, &bar->clean[i & 1], turn_of(i)) && wait_for(bar, &bar->p_ready, turn))) break;
          fence_after();
#pragma unroll
          for (int k = 0; k < kTile / 16; ++k)
            mma_ts(tm + kColO, tm + kColS + k * 16, desc_mn(sv, k), kIdesc | kMnB, true);
          if (w.begins && i == 0) {
#pragma unroll 1
            for (int k = 0; k < kTile / 16; ++k)
              mma_ts(tm + kColO, tm + kColS + k * 16 + 8, desc_mn(sv, k), kIdesc | kMnB, true);
          }
          commit(&bar->o2_full[i & 1]);
        }
        if (STATES) commit(&bar->empty_v[i % kStages]);
        else if (i + 1 < w.n) scores(i + 1);
      }
    } else if (!STATES && warp >= 2) {
      // ---- V without what is not finite: columns [64 p, 64 p + 64) ----
      const int p = warp - 2;
      for (int i = 0; i < w.n; ++i) {
        if (!(ok = warp_wait(bar, &bar->full_v[i % kStages], turn_of(i)))) break;
        const uint32_t panel = stage_of(i) + R::kV + p * kPanel;
        const int pieces = 8 * w.rows(i);  // of 16 bytes
        uint32_t sum[4] = {0, 0, 0, 0};
#pragma unroll 1
        for (int e = lane; e < pieces; e += 32) {
          const uint4 x = lds4(panel + 16 * e);
          sum[0] = add_zero_times(x.x, sum[0]);
          sum[1] = add_zero_times(x.y, sum[1]);
          sum[2] = add_zero_times(x.z, sum[2]);
          sum[3] = add_zero_times(x.w, sum[3]);
        }
        const bool odd = __any_sync(0xffffffffu, (sum[0] | sum[1] | sum[2] | sum[3]) != 0);
        if (odd) {
          // U reads V as it came.  (U of chunk i - 2 is done, since V of chunk i has come; U of chunk
          // i + 1 comes after this chunk's P V: one wait after the other, no turn is missed.)
          if (i < w.updates && !(ok = (i == 0 || warp_wait(bar, &bar->u_full, (i - 1) & 1)) &&
                                      warp_wait(bar, &bar->u_full, i & 1)))
            break;
          int* seen = bar->seen[i & 1] + 64 * p;
          seen[lane] = seen[lane + 32] = rev ? -1 : kTile;
          __syncwarp();
#pragma unroll 1
          for (int e = lane; e < 4 * pieces; e += 32) {  // (rare: two values at a time)
            const int row = e >> 5, col = 8 * ((e >> 2 ^ row) & 7) + 2 * (e & 3);
            const uint32_t x = __float_as_uint(lds(panel + 4 * e));
            uint32_t left = x;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const uint32_t exponent = 0x7f80u << 16 * k;
              if ((x & exponent) != exponent) continue;
              left &= 0xffff0000u >> 16 * k;
              if (rev) atomicMax(seen + col + k, row);
              else atomicMin(seen + col + k, row);
            }
            if (left != x) sts1(panel + 4 * e, left);
          }
          fence_async();
        }
        __syncwarp();
        if (lane == 0) {
          bar->odd[i & 1][p] = odd;
          arrive(&bar->clean[i & 1]);
          arrive(&bar->o2_full[i & 1]);
        }
      }
    }
  } else if (warp < kFirstState) {
    registers_down<88>();
    const int q = warp & 3, h = (warp - kFirstRow) >> 2;
    const uint32_t lanes = tmem + (uint32_t(q * 32) << 16);
    if (STATES) {
      // ---- the planes of every second 32 tokens ----
      for (int i = 0; i < w.n; ++i) {
        if (!(ok = warp_wait(bar, &bar->full[i % kStages], turn_of(i)))) break;
        if (three)
          make_planes<STATES, 0, 3>(stage_of(i) + R::kK, lanes, i, dec_upd, w.rows(i), rev, true, q, h, 2, 4, lane);
        else
          make_planes<STATES, 0, 2>(stage_of(i) + R::kK, lanes, i, dec_upd, w.rows(i), rev, false, q, h, 2, 4, lane);
        // the next planes go where those of chunk i - 1 are read; waited for here, so that no warp
        // arrives for a chunk before all have for the last, and no barrier is two turns ahead
        if (i > 0 && !(ok = warp_wait(bar, &bar->u_full, (i - 1) & 1))) break;
        fence_before();
        __syncwarp();
        if (lane == 0) {
          arrive(&bar->planes_ready);
          arrive(&bar->empty[i % kStages]);
        }
        fence_after();
      }
    } else {
      // ---- P, O and the results: row r of the chunk, columns [64 h, 64 h + 64) ----
      const int r = q * 32 + lane;
      const float intra = C.intra, inter = C.inter;
      const long long pitch = C.out.ts;
      for (int i = 0; i < w.n; ++i) {
        const int cnt = w.rows(i);
        const uint32_t turn = i & 1;
        // P[r][j] = intra Sc[r][j] l^|r - j| where j has been seen by r: blocks of 16
        // columns, of which this warp's rows see all, a triangle, or nothing.
        const bool second = w.begins && i == 0;
        if (!(ok = warp_wait(bar, &bar->sc_full, turn))) break;
        fence_after();
#pragma unroll 1
        for (int part = 0; part < 4; ++part) {
          const int block = 4 * h + part, j0 = 16 * block;
          uint32_t p[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) p[j] = 0;
          const bool diagonal = block >> 1 == q;
          if (diagonal || (block < 2 * q) != rev) {
            float x[16];
            tmem_ld16(lanes + kColS + j0, x);
            if (diagonal) {
#pragma unroll
              for (int j8 = 0; j8 < 16; j8 += 8) {
                float d[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) d[j] = lds(dec + 4 * abs(r - j0 - j8 - j));
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                  const int at = j0 + j8 + j;
                  x[j8 + j] = (rev ? at >= r : at <= r) ? x[j8 + j] * (intra * d[j]) : 0.f;
                }
              }
            } else {
              const float top = intra * lds(dec + 4 * (rev ? j0 - r : r - j0 - 15));
              const float2 b2 = make_float2(top, top);
              const uint32_t col = dec + 4 * (rev ? 132 : 148);
#pragma unroll
              for (int j = 0; j < 16; j += 4) {
                const uint4 d = lds4(col + 4 * j);
                const float2 y0 = __fmul2_rn(make_float2(x[j], x[j + 1]),
                                             __fmul2_rn(b2, make_float2(__uint_as_float(d.x), __uint_as_float(d.y))));
                const float2 y1 = __fmul2_rn(make_float2(x[j + 2], x[j + 3]),
                                             __fmul2_rn(b2, make_float2(__uint_as_float(d.z), __uint_as_float(d.w))));
                x[j] = y0.x;
                x[j + 1] = y0.y;
                x[j + 2] = y1.x;
                x[j + 3] = y1.y;
              }
            }
            if (cnt < kTile) {  // the columns of rows that are not this chunk's
#pragma unroll
              for (int j = 0; j < 16; ++j) x[j] = j0 + j < cnt ? x[j] : 0.f;
            }
#pragma unroll
            for (int j = 0; j < 16; j += 2) p[j >> 1] = pack2(x[j], x[j + 1]);
            if (second) {  // what the rounding left
              uint32_t rest[8];
#pragma unroll
              for (int j = 0; j < 16; j += 2)
                rest[j >> 1] = pack2(x[j] - low_half(p[j >> 1]), x[j + 1] - high_half(p[j >> 1]));
              tmem_st8(lanes + kColS + j0 + 8, rest);
            }
          } else if (second) {
            tmem_st8(lanes + kColS + j0 + 8, p);
          }
          tmem_st8(lanes + kColS + j0, p);
        }
        // Q X, decayed from the chunk's beginning
        const float f = inter * lds(dec + 4 * max(rev ? cnt - 1 - r : r + 1, 0));
        if (!(ok = warp_wait(bar, &bar->o1_full, turn))) break;
        fence_after();
#pragma unroll 1
        for (int part = 0; part < 2; ++part) {
          float x[32];
          tmem_ld32(lanes + kColO + h * 64 + part * 32, x);
#pragma unroll
          for (int j = 0; j < 32; ++j) x[j] *= f;
          tmem_st32(lanes + kColO + h * 64 + part * 32, x);
        }
        tmem_st_wait();
        fence_before();
        __syncwarp();
        if (lane == 0) arrive(&bar->p_ready);
        // results
        if (!(ok = warp_wait(bar, &bar->o2_full[i & 1], turn_of(i)))) break;
        fence_after();
        if (bar->odd[i & 1][h]) {  // NaN for the results that see what has been taken out of V (rare: least code)
#pragma unroll 1
          for (int j = 64 * h; j < 64 * h + 64; ++j) {
            const uint32_t x = tmem_ld1(lanes + kColO + j);
            const int at = bar->seen[i & 1][j];
            tmem_st1(lanes + kColO + j, (rev ? at >= r : at <= r) ? 0x7fffffff : x);
          }
          tmem_st_wait();
        }
        // through this warp's 4 KB of V's tile (its products are done), 128 bytes a row:
        // eight lanes then store a row's piece, instead of 32 rows at a time
        const uint32_t stage = stage_of(i) + R::kV + (warp - kFirstRow) * 4096;
        const int piece = lane & 7, row0 = 32 * q + (lane >> 3);
        const long long first = (w.first(C, i) + row0) * pitch + w.head * C.out.hs + h * 64;
        const bool f32 = C.out_f32;
        float y[2][32];
        tmem_ld32(lanes + kColO + h * 64, y[0]);
        tmem_ld32(lanes + kColO + h * 64 + 32, y[1]);
        fence_before();
        __syncwarp();
        if (lane == 0) arrive(&bar->o_free);
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          const float(&x)[32] = y[part];
          if (f32) {
#pragma unroll
            for (int j = 0; j < 32; j += 4)
              sts4(stage + lane * 128 + (((j / 4) ^ (lane & 7)) << 4), __float_as_uint(x[j]), __float_as_uint(x[j + 1]),
                   __float_as_uint(x[j + 2]), __float_as_uint(x[j + 3]));
          } else {
#pragma unroll
            for (int j = 0; j < 32; j += 8)
              sts4(stage + lane * 128 + (((part * 4 + j / 8) ^ (lane & 7)) << 4), pack2(x[j], x[j + 1]),
                   pack2(x[j + 2], x[j + 3]), pack2(x[j + 4], x[j + 5]), pack2(x[j + 6], x[j + 7]));
          }
          if (part == 1 || f32) {
            __syncwarp();
            const int col = f32 ? part * 32 + piece * 4 : piece * 8, bytes = f32 ? 4 : 2;
            const bool wide = h * 64 + col < C.dc;
            char* at = C.out.p + (first + col) * bytes;
#pragma unroll 1
            for (int k0 = 0; k0 < 8; k0 += 4) {
              uint4 v[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const int row = 4 * (k0 + k) + (lane >> 3);
                v[k] = lds4(stage + row * 128 + ((piece ^ (row & 7)) << 4));
              }
#pragma unroll
              for (int k = 0; k < 4; ++k, at += 4 * pitch * bytes)
                if (wide && row0 + 4 * (k0 + k) < cnt) *reinterpret_cast<uint4*>(at) = v[k];
            }
            __syncwarp();
          }
        }
        fence_async();  // before the tile is loaded again
        __syncwarp();
        if (lane == 0) arrive(&bar->empty_v[i % kStages]);
      }
    }
  } else {
    registers_up<120>();
    // ---- planes of decayed K (their lanes: the same rows of K^T), and the state: row b of
    // X, columns [64 h, 64 h + 64) ----
    const int q = warp & 3, h = (warp - kFirstState) >> 2;
    const int b = q * 32 + lane, t = threadIdx.x - 32 * kFirstState;
    const uint32_t lanes = tmem + (uint32_t(q * 32) << 16);
    const uint32_t own_x = base + kX + h * kPanel + q * 4096;  // the part of bf16 X that this warp writes
    float X[64];
    {
      const float* src = nullptr;
      int src_t = 0;
      if (!STATES) {
        const long long slot = lin::state_slot(C, w.seq);
        if (!w.only) {
          src = C.seg_state + static_cast<long long>(item) * C.db * C.dc;
        } else if (C.init && slot >= 0) {
          src = C.init + (slot * C.heads + w.head) * C.db * C.dc;
          src_t = C.init_t;
        }
      }
      if (src && !src_t) {
        load_state(X, src, own_x, 32 * q, 64 * h, C.db, C.dc, lane);
      } else {
#pragma unroll
        for (int c = 0; c < 64; ++c)
          X[c] = src && b < C.db && h * 64 + c < C.dc ? src[lin::state_index(C, src_t, b, h * 64 + c)] : 0.f;
      }
    }
    // chunk i of X = l^rows X + U
    auto update = [&](int i) {
      if (!(ok = warp_wait(bar, &bar->u_full, i & 1))) return;
      fence_after();
      const float keep = lds(dec + 4 * w.rows(i));
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        float x[32];
        tmem_ld32(lanes + kColU<STATES> + h * 64 + part * 32, x);
#pragma unroll
        for (int c = 0; c < 32; ++c) X[part * 32 + c] = fmaf(keep, X[part * 32 + c], x[c]);
      }
      fence_before();
      __syncwarp();
      if (STATES && lane == 0) arrive(&bar->u_free);
    };
    // one step past the last chunk, where its state is wanted
    for (int i = 0; i <= w.updates || i < w.n; ++i) {
      const bool chunk = i < w.n;
      const int cnt = chunk ? w.rows(i) : 0;
      if (chunk) {
        if (!(ok = warp_wait(bar, &bar->full[i % kStages], turn_of(i)))) break;
        if (cnt < kTile) {
          if (!(ok = warp_wait(bar, &bar->full_v[i % kStages], turn_of(i)))) break;
          const uint32_t v = stage_of(i) + R::kV;
          for (int e = t; e < (kTile - cnt) * 16; e += 256)
            sts4(v + (e & 1) * kPanel + (cnt + (e >> 4)) * 128 + ((e >> 1) & 7) * 16, 0, 0, 0, 0);
          fence_async();
        }
      }
      if (!STATES && i > 0) {
        update(i - 1);
        if (!ok) break;
      }
      if (chunk && i < w.updates) {
        constexpr int kG = STATES ? 2 : 4;
        if (STATES && three)
          make_planes<STATES, 0, STATES ? 3 : 2>(stage_of(i) + R::kK, lanes, i, dec_upd, cnt, rev, true, q, h, 0, kG, lane);
        else
          make_planes<STATES, 0, 2>(stage_of(i) + R::kK, lanes, i, dec_upd, cnt, rev, three, q, h, 0, kG, lane);
        if (!STATES && three) {  // plane 2, once the last results have been read from its columns
          if (i > 0 && !(ok = warp_wait(bar, &bar->o_free, (i - 1) & 1))) break;
          fence_after();
          make_planes<STATES, 2, 3>(stage_of(i) + R::kK, lanes, i, dec_upd, cnt, rev, true, q, h, 0, kG, lane);
        }
        fence_before();
      }
      // (a warp that arrives for chunk i knows that all have arrived for chunk i - 1, whose
      // product it has waited for: no warp can take another's place in the count)
      if (STATES && i > 0) {
        update(i - 1);
        if (!ok) break;
      }
      __syncwarp();
      if (chunk && lane == 0) {
        if (i < w.updates) arrive(&bar->planes_ready);
        arrive(&bar->empty[i % kStages]);
      }
      if (!STATES && chunk) {  // once the product that read the last chunk's X is done
        if (i > 0 && !(ok = warp_wait(bar, &bar->o1_full, (i - 1) & 1))) break;
        const uint32_t row = own_x + lane * 128;
#pragma unroll
        for (int c = 0; c < 8; ++c)
          sts4(row + ((c ^ (b & 7)) << 4), pack2(X[8 * c], X[8 * c + 1]), pack2(X[8 * c + 2], X[8 * c + 3]),
               pack2(X[8 * c + 4], X[8 * c + 5]), pack2(X[8 * c + 6], X[8 * c + 7]));
        fence_async();
        __syncwarp();
        if (lane == 0) arrive(&bar->x_ready);
      }
    }
    float* dst = nullptr;
    if (STATES) {
      dst = C.seg_state + static_cast<long long>(item) * C.db * C.dc;
    } else if (C.fin && w.last) {
      const long long slot = lin::state_slot(C, w.seq);
      if (slot >= 0) dst = C.fin + (slot * C.heads + w.head) * C.db * C.dc;
    }
    if (!STATES && ok && dst && w.n > 0) ok = warp_wait(bar, &bar->o1_full, (w.n - 1) & 1);  // bf16 X has been read
    if (ok && dst) store_state(X, dst, own_x, 32 * q, 64 * h, C.db, C.dc, lane);
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// ---- host ----------------------------------------------------------------------------

int rows_map(EncodeTiled enc, CUtensorMap* m, const seq::Rows& r, int heads, int width, long long tokens) {
  // a stride that no coordinate uses still has to be a valid one
  const long long hs = heads > 1 ? r.hs : 64, ts = tokens > 1 ? r.ts : 64;
  const cuuint64_t dims[3] = {cuuint64_t(width), cuuint64_t(heads), cuuint64_t(tokens)};
  const cuuint64_t strides[2] = {cuuint64_t(hs) * 2, cuuint64_t(ts) * 2};
  const cuuint32_t box[3] = {64, 1, kTile}, step[3] = {1, 1, 1};
  const CUresult e = enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, r.p, dims, strides, box, step,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (e != CUDA_SUCCESS) return set_error(TO_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", int(e));
  return ok();
}

long long items_of(const Chain& C) {
  return (C.seg_state ? lin::segment_slots(C.tokens, C.nseq, C.seg) : C.nseq) * 1ll * C.heads;
}

bool rows_fit(const seq::Rows& r, int heads, long long tokens) {
  const long long most = 1ll << 38;  // bytes of a stride: below the map's 2^40
  return aligned(r.p, 16) && (heads <= 1 || (r.hs % 8 == 0 && r.hs < most)) &&
         (tokens <= 1 || (r.ts % 8 == 0 && r.ts < most));
}

template <bool STATES, int N>
int run(const lin::Batch<N>& B, cudaStream_t s) {
  static std::atomic<uint64_t> done{0};
  int st = seq::allow_shared(chain_tc_kernel<STATES, N>, kSmem, done);
  if (st) return st;
  EncodeTiled enc = tensor_map_encoder(&st);
  if (!enc) return st;
  Maps<N> maps;
  for (int n = 0; n < N; ++n) {
    const Chain& C = B.c[n];
    CUtensorMap* m = maps.m[n];
    if ((st = rows_map(enc, &m[1], C.b, C.heads / C.b_div, C.db, C.tokens))) return st;
    if ((st = rows_map(enc, &m[2], C.c, C.heads / C.c_div, C.dc, C.tokens))) return st;
    m[0] = m[1];  // (not used by the states' launch)
    if (!STATES && (st = rows_map(enc, &m[0], C.a, C.heads / C.a_div, C.db, C.tokens))) return st;
  }
  const dim3 grid(unsigned(items_of(B.c[0])), N);
  chain_tc_kernel<STATES, N><<<grid, kThreads, kSmem, s>>>(maps, B);
  TO_CUDA_TRY(cudaGetLastError());
  return ok();
}

}  // namespace

namespace lin {

// bf16 rows of at most 128 values whose addresses TMA takes (16-byte rows) and
// whose results can be stored 16 bytes at a time.
bool tc_takes(const Chain& C) {
  const int per = C.out_f32 ? 4 : 8;
  return C.tokens > 0 && items_of(C) < INT32_MAX / 2 && C.db <= kTile && C.dc <= kTile &&
         rows_fit(C.a, C.heads / C.a_div, C.tokens) && rows_fit(C.b, C.heads / C.b_div, C.tokens) &&
         rows_fit(C.c, C.heads / C.c_div, C.tokens) && C.dc % per == 0 && aligned(C.out.p, 16) &&
         C.out.ts % per == 0 && C.out.hs % per == 0;
}

template <int N>
int tc_states(const Batch<N>& B, cudaStream_t s) { return run<true, N>(B, s); }
template <int N>
int tc_outputs(const Batch<N>& B, cudaStream_t s) { return run<false, N>(B, s); }
template int tc_states<1>(const Batch<1>&, cudaStream_t);
template int tc_states<3>(const Batch<3>&, cudaStream_t);
template int tc_outputs<1>(const Batch<1>&, cudaStream_t);
template int tc_outputs<3>(const Batch<3>&, cudaStream_t);

}  // namespace lin

int sequence_device_status(int reset, int* value) {
  int v = 0;
  TO_CUDA_TRY(cudaMemcpyFromSymbol(&v, g_sequence_status, sizeof(int)));
  if (reset && v) {
    const int z = 0;
    TO_CUDA_TRY(cudaMemcpyToSymbol(g_sequence_status, &z, sizeof(int)));
  }
  *value = v;
  return ok();
}

}  // namespace to_b200

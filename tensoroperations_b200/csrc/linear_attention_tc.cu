// linear_attention_tc.cu -- the decayed chain (linear_attention.cuh) of bf16
// rows on the 5th-generation tensor cores: tcgen05 + TMEM + TMA.
//
// A work item is one segment of one head; a CTA walks its items and their
// chunks of 128 tokens.  With Q, K, V the chunk's rows of a, b, c (tiles of
// 128 x 128, narrower widths zero-filled by TMA) and X the state:
//   Sc = Q K^T                    P = Sc masked and decayed, bf16, in TMEM
//   O1 = Q X (bf16 X)             O2 = P V
//   U  = (decayed K)^T V          out = intra O2 + inter l^(..) O1
//   X  = l^n X + U                (f32, in registers)
// all M = N = 128.  Six products of 128^3 a chunk (7 with three planes of K):
// 3072 tensor cycles at the dense bf16 rate against about 5600 for the chunk's
// 128 KB at this SM's share of the HBM, so the products hide behind the copies.
//
// Precision: P and X each enter their product with one bf16 rounding, as the
// result's own.  The state stays f32: decayed K is split into PLANES bf16
// values (8 bits each; 3 reach f32, 2 are enough where only out reads the
// state), smallest plane first, so few sums pass through the accumulator at
// full size; a chunk's U is added to X in IEEE f32 registers.
//
// Roles (20 warps): one lane issues TMA loads into a ring of 32 KB tiles, one
// the products; warps 4-11 turn Sc into P and store the results (a thread: one
// row, 64 columns); warps 12-19 make the planes (plane 0 in place of K, which
// Sc has read by then), and hold X (a thread: one row, 64 columns).  Products
// are issued Sc, O1, O2, U: the next chunk's Sc and P run under the state's
// update.  Rows past a chunk's end are masked: P and the planes by selection,
// V by zeroing its rows, since 0 * NaN is not 0.  Rows of a reversed chain keep
// their order in memory; only the masks and decays turn round.
//
// Every wait is bounded; on a timeout the kernel records TO_ERR_TIMEOUT in the
// device status word, waits (bounded) for its copies in flight, frees its TMEM
// and returns.
#include <cuda.h>

#include <mutex>

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
constexpr int kFirstRow = 4, kFirstState = kFirstRow + kRowWarps;  // warps 0, 1: loads, products; 2, 3: none
constexpr int kThreads = 32 * (kFirstState + kStateWarps);
constexpr uint32_t kMaxPolls = 1u << 22;
constexpr int kMaxSlots = 5;

// TMEM columns
constexpr uint32_t kColS = 0, kColO1 = 128, kColO2 = 256, kColU = 384;

struct Barriers {
  uint64_t full[kMaxSlots], empty[kMaxSlots];
  uint64_t sc_full, p_ready, o1_full, o2_full, o_free;
  uint64_t planes_ready, u_full, u_free, x_ready;
  uint64_t row_table, state_table;
  uint32_t tmem;
  int abort;
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

__device__ __forceinline__ void arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ void tma_tile(void* dst, const CUtensorMap* map, int head, int token, uint64_t* bar) {
#pragma unroll
  for (int p = 0; p < 2; ++p)
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(smem_u32(dst) + p * kPanel), "l"(map), "r"(64 * p), "r"(head), "r"(token), "r"(smem_u32(bar))
        : "memory");
}

// Shared-memory descriptor, 128-byte swizzle.  K-major operands (rows of 64
// contiguous K values): 8-row groups 1024 bytes apart.  MN-major ones (rows of
// 64 contiguous M or N values, one row a K value): 8-K groups 1024 bytes apart
// (stride offset), the two 64-value panels kPanel apart (leading offset).
__device__ __forceinline__ uint64_t desc(uint32_t saddr, uint32_t lbo) {
  return (uint64_t((saddr >> 4) & 0x3FFFu)) | (uint64_t((lbo >> 4) & 0x3FFFu) << 16) |
         (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
__device__ __forceinline__ uint64_t desc_k(uint32_t tile, int step) {  // 16 K values a step
  return desc(tile + (step >> 2) * kPanel + (step & 3) * 32, 16);
}
__device__ __forceinline__ uint64_t desc_mn(uint32_t tile, int step) { return desc(tile + step * 2048, kPanel); }

// D f32, A and B bf16, M = N = 128; bits 15 / 16: A / B are MN-major
constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(kTile >> 3) << 17) |
                            (uint32_t(kTile >> 4) << 24);
constexpr uint32_t kMnA = 1u << 15, kMnB = 1u << 16;

__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(uint32_t(add)) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(uint32_t(add)) : "memory");
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
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n\t"
      "tcgen05.wait::st.sync.aligned;"
      ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// (lo, hi) as two bf16 in one register, lo in the low half
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float low_half(uint32_t r) { return __uint_as_float(r << 16); }
__device__ __forceinline__ float high_half(uint32_t r) { return __uint_as_float(r & 0xffff0000u); }

// l^n, n = 0 .. 128, made by the eight warps of a group for their item.  Two
// tables in turn: a warp that has passed an item's barrier knows that all have
// left the table before the last.
constexpr int kTable = kTile + 1;
__device__ __forceinline__ const float* make_table(Barriers* b, uint64_t* bar, float* tables, uint32_t count, int t,
                                                   float gl, bool* ok) {
  float* dec = tables + (count & 1) * kTable;
  if (t < kTable) dec[t] = expf(gl * static_cast<float>(t));
  __syncwarp();
  if ((t & 31) == 0) arrive(bar);
  *ok = warp_wait(b, bar, count & 1);
  return dec;
}

// The chunks of a segment: `n` of them; chunk i's first row in memory and its rows.
struct Walk {
  Segment g;
  int head, n;
  long long s0, s1;
  __device__ __forceinline__ int rows(int i) const {
    const long long left = s1 - s0 - static_cast<long long>(i) * kTile;
    return left < kTile ? static_cast<int>(left) : kTile;
  }
  __device__ __forceinline__ long long first(const Chain& C, int i) const {
    const long long t = s0 + static_cast<long long>(i) * kTile;
    return C.rev ? g.first + g.tokens - t - rows(i) : g.first + t;
  }
};

// Item -> its walk; false: nothing to do there.
template <bool STATES>
__device__ __forceinline__ bool walk_of(const Chain& C, long long item, Walk* w) {
  const long long slot = item / C.heads;
  w->head = static_cast<int>(item - slot * C.heads);
  w->g = lin::segment_of(C, slot);
  if (w->g.idx < 0 || (STATES && w->g.idx == w->g.count - 1)) return false;
  w->s0 = w->g.idx * C.seg;
  w->s1 = min(w->s0 + C.seg, w->g.tokens);
  w->n = static_cast<int>((w->s1 - w->s0 + kTile - 1) / kTile);
  return true;
}

template <bool STATES>
struct Shape {
  static constexpr int kSlots = STATES ? 5 : 4;
  static constexpr uint32_t kPlanes = kSlots * kTileBytes;             // planes 1 and 2
  static constexpr uint32_t kX = kPlanes + 2 * kTileBytes;             // bf16 X
  static constexpr uint32_t kTables = kX + (STATES ? 0 : kTileBytes);  // tables of l^n
  static constexpr uint32_t kBars = kTables + 4 * kTable * 4;
  static constexpr uint32_t kBytes = kBars + sizeof(Barriers);
};
static_assert(Shape<false>::kBars % 8 == 0 && Shape<true>::kBars % 8 == 0, "aligned barriers");
static_assert(Shape<false>::kBytes <= 232448 && Shape<true>::kBytes <= 232448, "shared memory of a CTA");

template <typename TO, bool STATES, int PLANES>
__global__ void __launch_bounds__(kThreads, 1)
    chain_tc_kernel(const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapB,
                    const __grid_constant__ CUtensorMap mapC, const __grid_constant__ Chain C,
                    const long long items) {
  using L = Shape<STATES>;
  constexpr int kSlots = L::kSlots, kPer = STATES ? 2 : 3;  // tiles of a chunk: (Q,) K, V
  extern __shared__ __align__(1024) unsigned char sm[];
  if (smem_u32(sm) & 1023) {  // the swizzled tiles need it; there is no room left to round up in
    if (threadIdx.x == 0) atomicExch(&g_sequence_status, int(TO_ERR_SCRATCH));
    return;
  }
  Barriers* bar = reinterpret_cast<Barriers*>(sm + L::kBars);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kMaxSlots; ++i) {
      mbar_init(&bar->full[i], 1);
      mbar_init(&bar->empty[i], 1);
    }
    mbar_init(&bar->sc_full, 1);
    mbar_init(&bar->p_ready, kRowWarps);
    mbar_init(&bar->o1_full, 1);
    mbar_init(&bar->o2_full, 1);
    mbar_init(&bar->o_free, kRowWarps);
    mbar_init(&bar->planes_ready, kStateWarps);
    mbar_init(&bar->u_full, 1);
    mbar_init(&bar->u_free, kStateWarps);
    mbar_init(&bar->x_ready, kStateWarps);
    mbar_init(&bar->row_table, kRowWarps);
    mbar_init(&bar->state_table, kStateWarps);
    bar->abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&bar->tmem))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = bar->tmem;
  auto slot_of = [&](uint32_t tile) { return sm + (tile % kSlots) * kTileBytes; };
  Walk w;

  if (warp == 0) {
    if (lane == 0) {
      // ---- loads: Q, K, V of each chunk, in ring order (Q's slot is free first) ----
      uint32_t tile = 0;
      bool ok = true;
      for (long long item = blockIdx.x; item < items && ok; item += gridDim.x) {
        if (!walk_of<STATES>(C, item, &w)) continue;
        for (int i = 0; i < w.n && ok; ++i) {
          const int token = static_cast<int>(w.first(C, i));
          for (int x = 0; x < kPer; ++x, ++tile) {
            const uint32_t s = tile % kSlots;
            if (tile >= kSlots && !(ok = wait_for(bar, &bar->empty[s], (tile / kSlots - 1) & 1))) break;
            mbar_arrive_expect_tx(&bar->full[s], kTileBytes);
            if (x == kPer - 1) tma_tile(slot_of(tile), &mapC, w.head / C.c_div, token, &bar->full[s]);
            else if (x == kPer - 2) tma_tile(slot_of(tile), &mapB, w.head / C.b_div, token, &bar->full[s]);
            else tma_tile(slot_of(tile), &mapA, w.head / C.a_div, token, &bar->full[s]);
          }
        }
      }
      // copies still in flight land before the CTA ends
      for (uint32_t t = tile > kSlots ? tile - kSlots : 0; t < tile; ++t)
        mbar_wait_bounded(&bar->full[t % kSlots], (t / kSlots) & 1, kMaxPolls);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      // ---- products ----
      uint32_t n = 0;  // chunks so far
      bool ok = true;
      for (long long item = blockIdx.x; item < items && ok; item += gridDim.x) {
        if (!walk_of<STATES>(C, item, &w)) continue;
        for (int i = 0; i < w.n && ok; ++i, ++n) {
          const uint32_t tq = n * kPer, tk = tq + kPer - 2, tv = tk + 1;
          const uint32_t sk = smem_u32(slot_of(tk)), sv = smem_u32(slot_of(tv));
          auto full = [&](uint32_t t) { return wait_for(bar, &bar->full[t % kSlots], (t / kSlots) & 1); };
          if (!STATES) {
            const uint32_t sq = smem_u32(slot_of(tq)), sx = smem_u32(sm + L::kX);
            if (!(ok = full(tk) && full(tq))) break;
            fence_after();
#pragma unroll
            for (int k = 0; k < kTile / 16; ++k)
              mma(tmem + kColS, desc_k(sq, k), desc_k(sk, k), kIdesc, k > 0);
            commit(&bar->sc_full);
            if (!(ok = wait_for(bar, &bar->x_ready, n & 1) && (n == 0 || wait_for(bar, &bar->o_free, (n - 1) & 1)))) break;
            fence_after();
#pragma unroll
            for (int k = 0; k < kTile / 16; ++k)
              mma(tmem + kColO1, desc_k(sq, k), desc_mn(sx, k), kIdesc | kMnB, k > 0);
            commit(&bar->o1_full);
            commit(&bar->empty[tq % kSlots]);
          }
          if (!(ok = full(tv) && wait_for(bar, &bar->planes_ready, n & 1))) break;
          if (!STATES) {
            if (!(ok = wait_for(bar, &bar->p_ready, n & 1))) break;
            fence_after();
#pragma unroll
            for (int k = 0; k < kTile / 16; ++k)  // 16 tokens: 8 columns; tokens 64 .. start at column 64
              mma_ts(tmem + kColO2, tmem + kColS + (k >> 2) * 64 + (k & 3) * 8, desc_mn(sv, k), kIdesc | kMnB, k > 0);
            commit(&bar->o2_full);
          }
          if (n > 0 && !(ok = wait_for(bar, &bar->u_free, (n - 1) & 1))) break;
          fence_after();
#pragma unroll
          for (int p = PLANES - 1; p >= 0; --p) {
            const uint32_t sp = p == 0 ? sk : smem_u32(sm + L::kPlanes + (p - 1) * kTileBytes);
#pragma unroll
            for (int k = 0; k < kTile / 16; ++k)
              mma(tmem + kColU, desc_mn(sp, k), desc_mn(sv, k), kIdesc | kMnA | kMnB, p < PLANES - 1 || k > 0);
          }
          commit(&bar->u_full);
          commit(&bar->empty[tk % kSlots]);
          commit(&bar->empty[tv % kSlots]);
        }
      }
    }
  } else if (warp < kFirstRow) {
  } else if (warp < kFirstState) {
    if (!STATES) {
      // ---- P and the results: row r of the chunk, columns [64 h, 64 h + 64) ----
      const int q = warp & 3, h = (warp - kFirstRow) >> 2;
      const int r = q * 32 + lane;
      const uint32_t lanes = tmem + (uint32_t(q * 32) << 16);
      uint32_t n = 0, tables = 0;
      bool ok = true;
      for (long long item = blockIdx.x; item < items && ok; item += gridDim.x) {
        if (!walk_of<STATES>(C, item, &w)) continue;
        const float gl = lin::log_decay_of(C, w.head);
        const float* dec = make_table(bar, &bar->row_table, reinterpret_cast<float*>(sm + L::kTables), tables++,
                                      threadIdx.x - 32 * kFirstRow, gl, &ok);
        if (!ok) break;
        for (int i = 0; i < w.n; ++i, ++n) {
          const int cnt = w.rows(i);
          // P[r][j] = Sc[r][j] l^|r - j| where j has been seen by r
          if (!(ok = warp_wait(bar, &bar->sc_full, n & 1))) break;
          fence_after();
#pragma unroll
          for (int part = 0; part < 2; ++part) {
            float x[32];
            tmem_ld32(lanes + kColS + h * 64 + part * 32, x);
            const int j0 = h * 64 + part * 32;
            uint32_t p[16];
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              float y[2];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int far = C.rev ? j0 + j + e - r : r - (j0 + j + e);
                y[e] = far >= 0 && j0 + j + e < cnt ? x[j + e] * dec[far >= 0 ? far : 0] : 0.f;
              }
              p[j >> 1] = pack2(y[0], y[1]);
            }
            tmem_st16(lanes + kColS + h * 64 + part * 16, p);
          }
          fence_before();
          __syncwarp();
          if (lane == 0) arrive(&bar->p_ready);
          // results
          if (!(ok = warp_wait(bar, &bar->o2_full, n & 1) && warp_wait(bar, &bar->o1_full, n & 1))) break;
          fence_after();
          const int age = C.rev ? cnt - 1 - r : r + 1;
          const float f = C.inter * dec[age > 0 ? age : 0];
          const long long token = w.first(C, i) + r;
          TO* dst = seq::row_ptr<TO>(C.out, token, w.head / C.out_div) + h * 64;
#pragma unroll
          for (int part = 0; part < 2; ++part) {
            float x[32], y[32];
            tmem_ld32(lanes + kColO1 + h * 64 + part * 32, x);
            tmem_ld32(lanes + kColO2 + h * 64 + part * 32, y);
            if (part == 1) {  // everything has been read
              fence_before();
              __syncwarp();
              if (lane == 0) arrive(&bar->o_free);
            }
            if (r < cnt) {
#pragma unroll
              for (int j = 0; j < 32; ++j) x[j] = fmaf(f, x[j], C.intra * y[j]);
              constexpr int kV = 16 / int(sizeof(TO));
#pragma unroll
              for (int j = 0; j < 32; j += kV)
                if (h * 64 + part * 32 + j < C.dc) {
                  float t[kV];
#pragma unroll
                  for (int e = 0; e < kV; ++e) t[e] = x[j + e];
                  seq::store_vec<TO, kV>(dst + part * 32 + j, t);
                }
            }
          }
        }
      }
    }
  } else {
    // ---- planes of decayed K, and the state: row b of X, columns [64 h, 64 h + 64) ----
    const int q = warp & 3, h = (warp - kFirstState) >> 2;
    const int b = q * 32 + lane, t = threadIdx.x - 32 * kFirstState;
    const uint32_t lanes = tmem + (uint32_t(q * 32) << 16);
    uint32_t n = 0, tables = 0;
    bool ok = true;
    auto write_x = [&](const float (&X)[64]) {
      unsigned char* row = sm + L::kX + h * kPanel + b * 128;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        uint4 v;
        v.x = pack2(X[8 * c], X[8 * c + 1]);
        v.y = pack2(X[8 * c + 2], X[8 * c + 3]);
        v.z = pack2(X[8 * c + 4], X[8 * c + 5]);
        v.w = pack2(X[8 * c + 6], X[8 * c + 7]);
        *reinterpret_cast<uint4*>(row + ((c ^ (b & 7)) << 4)) = v;
      }
      fence_async();
      __syncwarp();
      if (lane == 0) arrive(&bar->x_ready);
    };
    for (long long item = blockIdx.x; item < items && ok; item += gridDim.x) {
      if (!walk_of<STATES>(C, item, &w)) continue;
      const long long entry = item;  // slot * heads + head
      const long long slot = lin::state_slot(C, w.g.seq);
      const float gl = lin::log_decay_of(C, w.head);
      const float* dec = make_table(bar, &bar->state_table, reinterpret_cast<float*>(sm + L::kTables) + 2 * kTable,
                                    tables++, t, gl, &ok);
      if (!ok) break;
      float X[64];
      const float* src = nullptr;
      int src_t = 0;
      if (!STATES) {
        if (C.seg_state) {
          src = C.seg_state + entry * C.db * C.dc;
        } else if (C.init && slot >= 0) {
          src = C.init + (slot * C.heads + w.head) * C.db * C.dc;
          src_t = C.init_t;
        }
      }
      if (src && b < C.db) {
        if (!src_t && C.dc % 4 == 0) {
          const float4* p = reinterpret_cast<const float4*>(src + static_cast<long long>(b) * C.dc + h * 64);
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            const float4 v = h * 64 + 4 * c < C.dc ? p[c] : make_float4(0.f, 0.f, 0.f, 0.f);
            X[4 * c] = v.x;
            X[4 * c + 1] = v.y;
            X[4 * c + 2] = v.z;
            X[4 * c + 3] = v.w;
          }
        } else {
#pragma unroll
          for (int c = 0; c < 64; ++c)
            X[c] = h * 64 + c < C.dc ? src[lin::state_index(C, src_t, b, h * 64 + c)] : 0.f;
        }
      } else {
#pragma unroll
        for (int c = 0; c < 64; ++c) X[c] = 0.f;
      }
      if (!STATES && w.n > 0) {
        // the product that read the last chunk's X is done
        if (n > 0 && !(ok = warp_wait(bar, &bar->o1_full, (n - 1) & 1))) break;
        write_x(X);
      }
      for (int i = 0; i < w.n; ++i, ++n) {
        const int cnt = w.rows(i);
        const uint32_t tk = n * kPer + kPer - 2, tv = tk + 1;
        if (!(ok = warp_wait(bar, &bar->full[tk % kSlots], (tk / kSlots) & 1))) break;
        if (cnt < kTile) {
          if (!(ok = warp_wait(bar, &bar->full[tv % kSlots], (tv / kSlots) & 1))) break;
          unsigned char* v = slot_of(tv);
          for (int e = t; e < (kTile - cnt) * 16; e += 256)
            *reinterpret_cast<uint4*>(v + (e & 1) * kPanel + (cnt + (e >> 4)) * 128 + ((e >> 1) & 7) * 16) =
                make_uint4(0, 0, 0, 0);
        }
        if (!STATES && !(ok = warp_wait(bar, &bar->sc_full, n & 1))) break;  // Sc has read K
        unsigned char* k = slot_of(tk);
        unsigned char* more = sm + L::kPlanes;
#pragma unroll 2
        for (int e = t; e < 2 * kTile * 8; e += 256) {
          const int j = (e >> 3) & (kTile - 1);  // 16-byte piece e of the tile; its row
          const int age = C.rev ? j + 1 : cnt - 1 - j;
          const float d = C.upd * dec[age >= 0 ? age : 0];
          uint4 raw4 = *reinterpret_cast<const uint4*>(k + e * 16);
          uint32_t in[4] = {raw4.x, raw4.y, raw4.z, raw4.w}, out[3][4];
#pragma unroll
          for (int z = 0; z < 4; ++z) {
            float lo = j < cnt ? low_half(in[z]) * d : 0.f, hi = j < cnt ? high_half(in[z]) * d : 0.f;
#pragma unroll
            for (int p = 0; p < PLANES; ++p) {
              out[p][z] = pack2(lo, hi);
              lo -= low_half(out[p][z]);
              hi -= high_half(out[p][z]);
            }
          }
          *reinterpret_cast<uint4*>(k + e * 16) = make_uint4(out[0][0], out[0][1], out[0][2], out[0][3]);
#pragma unroll
          for (int p = 1; p < PLANES; ++p)
            *reinterpret_cast<uint4*>(more + (p - 1) * kTileBytes + e * 16) =
                make_uint4(out[p][0], out[p][1], out[p][2], out[p][3]);
        }
        fence_async();
        __syncwarp();
        if (lane == 0) arrive(&bar->planes_ready);
        if (!(ok = warp_wait(bar, &bar->u_full, n & 1))) break;
        fence_after();
        const float keep = dec[cnt];
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          float x[32];
          tmem_ld32(lanes + kColU + h * 64 + part * 32, x);
#pragma unroll
          for (int c = 0; c < 32; ++c) X[part * 32 + c] = fmaf(keep, X[part * 32 + c], x[c]);
        }
        fence_before();
        __syncwarp();
        if (lane == 0) arrive(&bar->u_free);
        if (!STATES && i + 1 < w.n) {
          if (!(ok = warp_wait(bar, &bar->o1_full, n & 1))) break;  // O1 has read X
          write_x(X);
        }
      }
      if (!ok) break;
      float* dst = nullptr;
      int dst_t = 0;
      if (STATES) {
        dst = C.seg_state + entry * C.db * C.dc;
      } else if (C.fin && slot >= 0 && w.g.idx == w.g.count - 1) {
        dst = C.fin + (slot * C.heads + w.head) * C.db * C.dc;
        dst_t = C.fin_t;
      }
      if (dst && b < C.db) {
        if (!dst_t && C.dc % 4 == 0) {
          float4* p = reinterpret_cast<float4*>(dst + static_cast<long long>(b) * C.dc + h * 64);
#pragma unroll
          for (int c = 0; c < 16; ++c)
            if (h * 64 + 4 * c < C.dc) p[c] = make_float4(X[4 * c], X[4 * c + 1], X[4 * c + 2], X[4 * c + 3]);
        } else {
#pragma unroll
          for (int c = 0; c < 64; ++c)
            if (h * 64 + c < C.dc) dst[lin::state_index(C, dst_t, b, h * 64 + c)] = X[c];
        }
      }
    }
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

bool rows_fit(const seq::Rows& r, int heads, long long tokens) {
  const long long most = 1ll << 38;  // bytes of a stride: below the map's 2^40
  return aligned(r.p, 16) && (heads <= 1 || (r.hs % 8 == 0 && r.hs < most)) &&
         (tokens <= 1 || (r.ts % 8 == 0 && r.ts < most));
}

template <typename TO, bool STATES, int PLANES>
int launch(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& c, const Chain& C, int sms,
           cudaStream_t s) {
  static std::once_flag once;
  static cudaError_t attr = cudaSuccess;
  std::call_once(once, [] {
    attr = cudaFuncSetAttribute(chain_tc_kernel<TO, STATES, PLANES>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                int(Shape<STATES>::kBytes));
  });
  TO_CUDA_TRY(attr);
  const long long items = (C.seg_state ? lin::segment_slots(C.tokens, C.nseq, C.seg) : C.nseq) * C.heads;
  chain_tc_kernel<TO, STATES, PLANES>
      <<<unsigned(items < sms ? items : sms), kThreads, Shape<STATES>::kBytes, s>>>(a, b, c, C, items);
  TO_CUDA_TRY(cudaGetLastError());
  return ok();
}

template <bool STATES>
int run(const Chain& C, bool f32_out, cudaStream_t s) {
  int st = TO_OK;
  EncodeTiled enc = tensor_map_encoder(&st);
  if (!enc) return st;
  CUtensorMap a, b, c;
  if ((st = rows_map(enc, &a, C.a, C.heads / C.a_div, C.db, C.tokens))) return st;
  if ((st = rows_map(enc, &b, C.b, C.heads / C.b_div, C.db, C.tokens))) return st;
  if ((st = rows_map(enc, &c, C.c, C.heads / C.c_div, C.dc, C.tokens))) return st;
  int dev = 0;
  const int sms = device_sm_count(&dev);
  if (sms <= 0) return -sms;
  // three planes where the state itself is a result
  if (STATES)
    return C.fin ? launch<float, STATES, 3>(a, b, c, C, sms, s) : launch<float, STATES, 2>(a, b, c, C, sms, s);
  if (f32_out) return C.fin ? launch<float, false, 3>(a, b, c, C, sms, s) : launch<float, false, 2>(a, b, c, C, sms, s);
  return C.fin ? launch<__nv_bfloat16, false, 3>(a, b, c, C, sms, s)
               : launch<__nv_bfloat16, false, 2>(a, b, c, C, sms, s);
}

}  // namespace

namespace lin {

// bf16 rows of at most 128 values whose addresses TMA takes (16-byte rows) and
// whose results can be stored 16 bytes at a time.
bool tc_takes(const Chain& C, bool f32_out) {
  const int per = f32_out ? 4 : 8;
  return C.tokens > 0 && C.db <= kTile && C.dc <= kTile && rows_fit(C.a, C.heads / C.a_div, C.tokens) &&
         rows_fit(C.b, C.heads / C.b_div, C.tokens) && rows_fit(C.c, C.heads / C.c_div, C.tokens) &&
         C.dc % per == 0 && aligned(C.out.p, 16) && C.out.ts % per == 0 && C.out.hs % per == 0;
}

int tc_states(const Chain& C, cudaStream_t s) { return run<true>(C, false, s); }
int tc_outputs(const Chain& C, bool f32_out, cudaStream_t s) { return run<false>(C, f32_out, s); }

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

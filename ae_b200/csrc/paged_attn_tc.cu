// Attention of many query rows over a paged cache on the 5th-generation tensor cores: draft trees (a
// few dozen tokens x the query heads of a key head) and prefill chunks.
//
//   S = Q K^T  (128 rows x 128 keys, fp32 in TMEM),  P = 2^(scale log2(e) S - m),  O += P V
//
// with a running maximum m and sum per row.  A row of S lies in one TMEM lane, so a softmax
// thread owns a row: maximum and sum need no exchange between threads.  P goes back into S's TMEM
// columns in the 16-bit type and is the A operand of the second product from there; V is its B
// operand as it lies in memory (keys x dims, "MN-major"), so nothing is transposed.
//
// Two streams of 128 rows keep the tensor pipe and the exponentials busy at once: while the four
// warps of one stream work on their S, the pipe runs the other stream's products.
//  - DUAL (more than 128 rows for a key head): the streams are two row tiles over the same keys, each
//    K and V tile is read once for 256 rows.  Bound by arithmetic: per 128 keys and stream 512 clocks
//    of tensor pipe for each product and 128 exponentials per lane group, 1024 clocks on the
//    special-function units.
//  - otherwise the streams take the even and the odd key tiles of the same 128 rows and are added at
//    the end.  Bound by memory at the sizes of a verify step: a 64 KB tile takes an SM's share of HBM
//    about 2800 clocks, twice what its products and exponentials take.
//
// Measured, both with two row tiles: 16 sequences of up to 16384 keys, trees of 32 tokens, 48 / 8
// heads of 128: 707 MB of cache and 109 GFLOP in 187-225 us (3.1-3.8 TB/s); two chunks of 2048 tokens
// over 8191 keys: 290 GFLOP in 289-370 us (785-1005 TFLOP/s).  Both follow the SM clock (355 and 588 thousand
// clocks a call; the power cap takes it from 1965 to 1590 and 1785 MHz back to back), so what bounds them is the
// chain of a tile: about 3400 clocks for a 128-key tile of a stream (clock stamps), 400 to read S, 280 for the
// maximum, 1400 for the exponentials and P, 1300 until the next S; the two streams' exponentials alone need
// 2048.  With one row tile: 16 sequences of 8192 keys, trees of 32 tokens, 32 / 8 heads of 128: 537 MB in 105 us,
// 0.79 of the measured copy rate.
//
// Keys and values come by TMA, one box per page (its rows of one head) and 64 dims, into a ring of
// five 128-row slots with the 128-byte swizzle.  Keys past the end and pages outside the cache are
// boxes at a page coordinate past the tensor: TMA writes zeros there, and the mask drops them.  Rows
// behind the last key inside a page, and new tokens that a row may not see, may hold anything: where
// a mask cuts a tile, the softmax warps look through V in shared memory before the product, take
// non-finite values out, and the rows that do see them get them added from memory at the end.
//
// Q comes by TMA too, one box of tq tokens x gs heads and 64 dims, as soon as the last segment's
// products with Q are done, so that a segment's first S is there when its predecessor's output has been
// written.
//
// A 4-bit cache (32 / 8 heads, else as above: 73 GFLOP in 205-209 us, bound by the unpacking, 2000 clocks for the
// 128 rows of a slot) has four more warps in the place of TMA's K and V: rows come packed by cp.async into a
// ring of each warp's own, and go as values of the 16-bit type into the slots (scale x code + zero,
// one rounding: the score of a key is then off by at most half a step of each of its values, as if the
// cache were of the 16-bit type; applying the scales to the products instead, as the kernel for few
// rows does, would need the scores of each group of 32 dims by themselves).  V keeps the order in which
// a word's nibbles come out (dims e and e + 4 side by side), and the output's columns are put right
// when they are stored.
//
// Every wait is bounded, and no role waits at a hardware barrier inside its loop: after a failed wait
// each role runs out of segments by itself (the results are void; the caller's status word, if there is
// one, says so).
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "host.h"
#include "kernels.h"
#include "paged_math.cuh"
#include "paged_plan.cuh"

namespace smb {
namespace {

constexpr int kTBK = 128;       // keys of a tile
// warp 0 TMA, warp 1 MMA, warp 2 TMEM, warp 3 segments, warps 4-7 / 8-11 softmax, 12-15 values of a 4-bit cache
constexpr int kTThreads = 384, kTThreads4 = 512;
constexpr int kTRaw = 4;        // slots of packed rows
constexpr int kTOkRing = 8;     // tiles whose page masks are kept: the ring lets K run at most 5 tiles ahead

template <int D, bool DUAL, bool BITS4>
struct TcCfg {
  static constexpr int THREADS = BITS4 ? kTThreads4 : kTThreads;
  static constexpr int NS = BITS4 ? 3 : 5;                  // ring slots
  static constexpr int ROW4 = kv4_row_bytes(D);
  static constexpr int RAW = BITS4 ? 4 * kTRaw * 32 * ROW4 : 0;
  static constexpr int SEG_READERS = 1 + 1 + 256 + (BITS4 ? 128 : 0);  // TMA and MMA warps, softmax threads, ...
  static constexpr int R = DUAL ? 256 : 128;
  static constexpr int TILE = kTBK * D * 2;                 // bytes of a K or V tile, and of 128 rows of Q
  static constexpr int QHALF = R * 128;                     // bytes of 64 dims of Q
  static constexpr int Q = (DUAL ? 2 : 1) * TILE;
  static constexpr int GIVE = DUAL ? 0 : 2 * 128 * 32 * 4;  // 32 columns of each stream's output for the other
  static constexpr int SMEM = Q + NS * TILE + GIVE + RAW + 1024;
};

// TMEM columns: S of the streams at 0 and 128 (P in their first 64), O at 256 and 384.
constexpr uint32_t kTmemS = 0, kTmemO = 256;

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2,
                                            int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::
          "r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::
          "r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

// D[tmem] (+)= A[tmem] * B[smem], kind::f16.
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Descriptor of an MN-major operand (V: rows of 64 dims = 128 bytes, one row per key) in the 128-byte
// swizzle: 8-key groups 1024 bytes apart (stride offset), the next 64 dims `half` bytes on (leading
// offset).
__device__ __forceinline__ uint64_t desc_mnmajor_sw128(uint32_t addr, uint32_t half) {
  uint64_t d = desc_kmajor_sw128(addr) & ~(0x3FFFull << 16);
  return d | static_cast<uint64_t>(half >> 4) << 16;
}
constexpr uint32_t kIdescBMn = 1u << 16;  // B is MN-major

#define SMB_R4(v, i) "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3])
#define SMB_R16(v, i) SMB_R4(v, i), SMB_R4(v, i + 4), SMB_R4(v, i + 8), SMB_R4(v, i + 12)
#define SMB_P4(v, i) "+r"(v[i]), "+r"(v[i + 1]), "+r"(v[i + 2]), "+r"(v[i + 3])
#define SMB_P16(v, i) SMB_P4(v, i), SMB_P4(v, i + 4), SMB_P4(v, i + 8), SMB_P4(v, i + 12)
#define SMB_I4(v, i) "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3])
#define SMB_I16(v, i) SMB_I4(v, i), SMB_I4(v, i + 4), SMB_I4(v, i + 8), SMB_I4(v, i + 12)

// 32 columns of this thread's lane, issued only; tmem_ld_done(v) before v is used.
__device__ __forceinline__ void tmem_ld32_issue(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : SMB_R16(v, 0), SMB_R16(v, 16)
      : "r"(taddr)
      : "memory");
}
// Waits for every issued load; the values pass through so that no use moves before the wait.
__device__ __forceinline__ void tmem_ld_done(uint32_t (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : SMB_P16(v, 0), SMB_P16(v, 16) : : "memory");
}
// The same for 16 columns.
__device__ __forceinline__ void tmem_ld16_wait(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];\n\ttcgen05.wait::ld.sync.aligned;"
      : SMB_R16(v, 0)
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(taddr),
      SMB_I16(v, 0)
      : "memory");
}
__device__ __forceinline__ void tmem_st_done() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// One segment of this CTA's share.  Warp 3 walks the share and hands them to the other roles.
struct Segment {
  int t0, t1;         // its key tiles (t1 = -1: the share is done)
  int keys;           // keys its rows can see
  int prefix, open;   // keys before the new tokens; first key that some row may not see
  int b, kvh;
  int head, heads;    // first query head, heads of a token
  int tok, toks, i0;  // first row of q, tokens, the first one's place among the sequence's new tokens
  int slot;           // of a partial result, -1: the segment lies in this share
};
constexpr int kTSegs = 4;  // segments handed out ahead

// The k-th of the 2 n loads of a segment of n tiles, in the order of their use.
template <bool DUAL>
__device__ __forceinline__ void load_step(int n, int k, int& tile, bool& is_k) {
  if (DUAL || n == 1) {
    tile = k >> 1;
    is_k = (k & 1) == 0;
  } else if (k < 2) {
    tile = k;
    is_k = true;
  } else {
    const int j = k - 2, pairs = n - 2;  // (V i, K i + 2) for i < n - 2, then the last two of V
    is_k = j < 2 * pairs && (j & 1) != 0;
    tile = j < 2 * pairs ? (is_k ? (j >> 1) + 2 : j >> 1) : j - pairs;
  }
}

// Where dim d of a word's eight is among the values that its nibbles give in turn.
__host__ __device__ constexpr int nibble_place(int d) { return 2 * (d & 3) + (d >> 2); }

template <int D, bool DUAL, bool BITS4, typename T>
__global__ void __launch_bounds__(BITS4 ? kTThreads4 : kTThreads, 1)
    paged_attn_tc_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ CUtensorMap tm_q,
                         const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v) {
  using C = TcCfg<D, DUAL, BITS4>;
  using H = Half2<T>;
  constexpr bool kBF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr int R = C::R, TILE = C::TILE, NS = C::NS;
  constexpr uint32_t HALF = kTBK * 128;  // bytes of 64 dims of a tile
  extern __shared__ uint8_t dyn_smem[];
  __shared__ uint64_t full_bar[NS], empty_bar[NS], s_bar[2], p_bar[2][2], o_bar[2], q_full, q_empty, drain_bar, both_bar;
  __shared__ uint64_t seg_full[kTSegs], seg_empty[kTSegs];
  __shared__ Segment s_seg[kTSegs];
  __shared__ uint32_t s_tmem, s_pages[kTOkRing][BITS4 ? 4 : 1];
  __shared__ int s_abort, s_fix;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t raw = smem_u32(dyn_smem);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* sm = dyn_smem + (base - raw);
  const uint32_t q_s = base, ring_s = base + C::Q;
  // the plan lies where the ring will be: every thread but warp 3's is done with it at the barrier behind
  // plan_build, and warp 3 before it hands out the first segment, which the first copy into the ring follows
  PlanShared* plan = reinterpret_cast<PlanShared*>(sm + C::Q);

  if (tid == 0) {
    s_abort = 0;
    s_fix = 0;
    for (int i = 0; i < NS; ++i) {
      mbar_init(&full_bar[i], BITS4 ? 128 : 1);
      mbar_init(&empty_bar[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_bar[i], 1);
      mbar_init(&p_bar[i][0], 128);
      mbar_init(&p_bar[i][1], 128);
      mbar_init(&o_bar[i], 1);
    }
    for (int i = 0; i < kTSegs; ++i) {
      mbar_init(&seg_full[i], 1);
      mbar_init(&seg_empty[i], C::SEG_READERS);
    }
    mbar_init(&q_full, 1);
    mbar_init(&q_empty, 1);
    mbar_init(&drain_bar, 1);
    mbar_init(&both_bar, 256);
    fence_mbarrier_init();
    prefetch_tmap(&tm_q);
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
  }
  if (warp == 2) {
    tmem_alloc(&s_tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;

  pdl_wait_prior_grids();
  pdl_launch_dependents();
  const int cta = blockIdx.x;
  const long long W = plan_build<kTBK>(a, plan, gridDim.x);
  fence_async_proxy();  // (TMA writes there next)
  __syncthreads();
  int* status = a.status;
  volatile int* abort_flag = &s_abort;

  {
    // The i-th segment of the share; false when it is done, or after a failed wait.
    auto next_segment = [&](int i, Segment& g) {
      if (!mbar_wait(&seg_full[i % kTSegs], (i / kTSegs) & 1, status, abort_flag)) return false;
      g = s_seg[i % kTSegs];
      return g.t1 >= 0;
    };
    Segment g{};
    int seg = 0;
    if (warp < 4) {
      // (the shares' sum is what the block is launched with: 384 x 168, 512 x 128)
      if constexpr (BITS4) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
      else asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
      if (warp == 0) {
        // ---------------------------------------------------------------- TMA
        const int psb = min(1 << a.c.page_shift, kTBK);  // rows of a box
        const int pages = kTBK / psb, boxes = pages * (D / 64);
        const int page_mask = (1 << a.c.page_shift) - 1;
        int it = 0, tc = 0;
        // a tile's boxes, one per page and 64 dims (at most 32: a lane issues one)
        auto load = [&](const CUtensorMap* map, int t, bool is_k) {
          const int slot = it % NS;
          const int p = lane % pages, j = t * kTBK + p * psb;
          const bool in = j < g.keys;
          const int page = in ? a.table[g.b * a.table_stride + (j >> a.c.page_shift)] : -1;
          const bool good = page >= 0 && page < a.c.num_pages;
          const uint32_t bad = __ballot_sync(0xffffffffu, in && lane < pages && !good);
          if (is_k) {
            if (lane == 0) {
              s_pages[tc % kTOkRing][0] = ~bad;
              if (bad != 0) record_status(status, kDevBadPage);
            }
            ++tc;
          }
          mbar_wait(&empty_bar[slot], ((it / NS) & 1) ^ 1, status, abort_flag);
          if (lane == 0) mbar_arrive_expect_tx(&full_bar[slot], TILE);
          __syncwarp();
          if (lane < boxes) {
            const int h = lane / pages;
            tma_load_4d(ring_s + slot * TILE + h * HALF + p * psb * 128, map, &full_bar[slot], h * 64, j & page_mask,
                        g.kvh, good ? page : static_cast<int>(a.c.num_pages));
          }
          ++it;
        };
        while (__all_sync(0xffffffffu, next_segment(seg, g))) {
          if (lane == 0) mbar_arrive(&seg_empty[seg % kTSegs]);
          const int n = g.t1 - g.t0;
          if constexpr (!BITS4) load(&tm_k, g.t0, true);
          mbar_wait(&q_empty, (seg & 1) ^ 1, status, abort_flag);
          if (lane == 0) {
            mbar_arrive_expect_tx(&q_full, a.tq * a.gs * (D / 64) * 128);
#pragma unroll
            for (int h = 0; h < D / 64; ++h) tma_load_3d(q_s + h * C::QHALF, &tm_q, &q_full, h * 64, g.head, g.tok);
          }
          __syncwarp();
          ++seg;
          if constexpr (BITS4) continue;
          if constexpr (DUAL) {
            for (int t = g.t0; t < g.t1; ++t) {
              if (t > g.t0) load(&tm_k, t, true);
              load(&tm_v, t, false);
            }
          } else {
            if (n > 1) load(&tm_k, g.t0 + 1, true);
            for (int i = 0; i < n; ++i) {
              load(&tm_v, g.t0 + i, false);
              if (i + 2 < n) load(&tm_k, g.t0 + i + 2, true);
            }
          }
        }
        // the copies into every slot have landed before the CTA may end
        for (int i = max(0, it - NS); i < it; ++i)
          mbar_wait(&full_bar[i % NS], (i / NS) & 1, status, nullptr);
        if (seg > 0) mbar_wait(&q_full, (seg - 1) & 1, status, nullptr);
      } else if (warp == 3) {
        // ---------------------------------------------------------------- segments
        Work k;
        bool more = work_begin<kTBK>(a, plan, W, cta, gridDim.x, k);
        fence_async_proxy();
        __syncwarp();  // (the first segment gives the plan's place to the ring: every lane has read it)
        if (!more && lane == 0) leave_record(a, cta, k);
        while (more) {
          const Cursor& cur = k.cur;
          Segment n;
          n.t0 = k.t0;
          n.t1 = k.t1;
          n.slot = k.slot;
          n.keys = cur.keys;
          const int sub = cur.vh % a.nsub;
          n.kvh = cur.vh / a.nsub;
          n.b = cur.b;
          n.head = n.kvh * a.g + sub * a.gs;
          n.heads = min(a.gs, a.g - sub * a.gs);
          n.i0 = cur.qt * a.tq;
          n.tok = cur.s.s0 + n.i0;
          n.toks = min(a.tq, cur.s.n - n.i0);
          n.prefix = cur.s.L - cur.s.n;
          n.open = a.tree != nullptr ? n.prefix : n.prefix + n.i0 + 1;
          mbar_wait(&seg_empty[seg % kTSegs], ((seg / kTSegs) & 1) ^ 1, status, abort_flag);
          if (lane == 0) {
            s_seg[seg % kTSegs] = n;
            mbar_arrive(&seg_full[seg % kTSegs]);
          }
          __syncwarp();
          ++seg;
          more = !k.final && work_next<kTBK>(a, W, cta, gridDim.x, k);
          if (!more && lane == 0) leave_record(a, cta, k);
        }
        mbar_wait(&seg_empty[seg % kTSegs], ((seg / kTSegs) & 1) ^ 1, status, abort_flag);
        if (lane == 0) {
          s_seg[seg % kTSegs].t1 = -1;
          mbar_arrive(&seg_full[seg % kTSegs]);
        }
      } else if (warp == 1 && lane == 0) {
        // ---------------------------------------------------------------- MMA
        constexpr uint32_t idesc_s = idesc_f16(kBF16, 128, kTBK);
        constexpr uint32_t idesc_o = idesc_f16(kBF16, 128, D) | kIdescBMn;
        int it = 0, np[2] = {0, 0};
        auto wait_full = [&](int i) {
          mbar_wait(&full_bar[i % NS], (i / NS) & 1, status, abort_flag);
          tc_fence_after();
        };
        auto qk = [&](int i, int s) {  // S_s = Q_s K^T, K in the slot of step i
          const uint32_t ks = ring_s + (i % NS) * TILE, qs = q_s + (DUAL ? s * (128 * 128) : 0);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t qo = (kk / 4) * C::QHALF + (kk % 4) * 32, ko = (kk / 4) * HALF + (kk % 4) * 32;
            umma_f16(tmem + kTmemS + s * 128, desc_kmajor_sw128(qs + qo), desc_kmajor_sw128(ks + ko), idesc_s, kk > 0);
          }
        };
        // O_s (+)= P_s V, each half as soon as its 64 keys of P are there
        auto pv = [&](int i, int s, bool first) {
          const uint32_t vs = ring_s + (i % NS) * TILE;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            mbar_wait(&p_bar[s][h], np[s] & 1, status, abort_flag);
            tc_fence_after();
#pragma unroll
            for (int kk = 4 * h; kk < 4 * h + 4; ++kk)
              umma_f16_ts(tmem + kTmemO + s * 128, tmem + kTmemS + s * 128 + kk * 8,
                          desc_mnmajor_sw128(vs + kk * 2048, HALF), idesc_o, !(first && kk == 0));
          }
          ++np[s];
        };
        while (next_segment(seg, g)) {
          mbar_arrive(&seg_empty[seg % kTSegs]);
          const int n = g.t1 - g.t0;
          mbar_wait(&q_full, seg & 1, status, abort_flag);
          tc_fence_after();
          ++seg;
          if constexpr (DUAL) {
            int kslot = it++;
            wait_full(kslot);
            qk(kslot, 0);
            umma_commit(&s_bar[0]);
            qk(kslot, 1);
            umma_commit(&s_bar[1]);
            umma_commit(&empty_bar[kslot % NS]);
            if (n == 1) umma_commit(&q_empty);
            for (int t = 0; t < n; ++t) {
              const bool more = t + 1 < n;
              const int vslot = it++;
              if (more) kslot = it++;
              wait_full(vslot);
              pv(vslot, 0, t == 0);
              if (more) {
                wait_full(kslot);
                qk(kslot, 0);
                umma_commit(&s_bar[0]);
              } else {
                umma_commit(&o_bar[0]);
              }
              pv(vslot, 1, t == 0);
              umma_commit(&empty_bar[vslot % NS]);
              if (more) {
                qk(kslot, 1);
                umma_commit(&s_bar[1]);
                umma_commit(&empty_bar[kslot % NS]);
                if (t + 2 == n) umma_commit(&q_empty);  // the segment's last product with Q
              } else {
                umma_commit(&o_bar[1]);
              }
            }
          } else {
            for (int s = 0; s < min(n, 2); ++s) {
              wait_full(it);
              qk(it, s);
              umma_commit(&empty_bar[it % NS]);
              umma_commit(&s_bar[s]);
              ++it;
            }
            if (n <= 2) umma_commit(&q_empty);
            for (int t = 0; t < n; ++t) {
              const int s = t & 1;
              wait_full(it);
              pv(it, s, t < 2);
              umma_commit(&empty_bar[it % NS]);
              ++it;
              if (t + 2 < n) {
                wait_full(it);
                qk(it, s);
                umma_commit(&empty_bar[it % NS]);
                umma_commit(&s_bar[s]);
                if (t + 3 == n) umma_commit(&q_empty);  // the segment's last product with Q
                ++it;
              } else {
                umma_commit(&o_bar[s]);
              }
            }
          }
        }
        umma_commit(&drain_bar);
        mbar_wait(&drain_bar, 0, status, nullptr);
      }
    } else if (BITS4 && warp >= 12) {
      // ------------------------------------------------------------------ values of a 4-bit cache
      asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
      if constexpr (BITS4) {
        constexpr int ROW = C::ROW4, CH = ROW / 16, G = D / 32;
        const int w4 = warp - 12;  // this warp's 32 keys of a tile
        uint8_t* raw = sm + C::Q + NS * TILE + C::GIVE + w4 * (kTRaw * 32 * ROW);
        const uint32_t raw_s = smem_u32(raw);
        const int page_mask = (1 << a.c.page_shift) - 1;
        int it = 0, tc = 0;
        while (__all_sync(0xffffffffu, next_segment(seg, g))) {
          mbar_arrive(&seg_empty[seg % kTSegs]);
          ++seg;
          const int n = g.t1 - g.t0;
          const int* table = a.table + g.b * a.table_stride;
          // the page of this lane's key for step k (one step ahead of its loads)
          auto look_up = [&](int k) {
            if (k >= 2 * n) return -1;
            int tile;
            bool is_k;
            load_step<DUAL>(n, k, tile, is_k);
            const int j = (g.t0 + tile) * kTBK + w4 * 32 + lane;
            return j < g.keys ? table[j >> a.c.page_shift] : -1;
          };
          int page = look_up(0);
          auto issue = [&](int k) {
            if (k < 2 * n) {
              int tile;
              bool is_k;
              load_step<DUAL>(n, k, tile, is_k);
              const int j = (g.t0 + tile) * kTBK + w4 * 32 + lane;
              const bool in = j < g.keys, ok = in && page >= 0 && page < a.c.num_pages;
              const long long off = ok ? page * a.c.page_stride + (j & page_mask) * a.c.token_stride : 0;
              const uint32_t okm = __ballot_sync(0xffffffffu, ok);
              if (is_k) {
                if (in && !ok) record_status(status, kDevBadPage);
                // (what lies behind the keys is masked by the keys' number)
                const uint32_t lost = __ballot_sync(0xffffffffu, in && !ok);
                if (lane == 0) s_pages[(tc + tile) % kTOkRing][w4] = ~lost;
              }
              page = look_up(k + 1);
              const uint8_t* src = (is_k ? a.c.k : a.c.v) + g.kvh * a.c.head_stride;
              const uint32_t dst = raw_s + (k % kTRaw) * (32 * ROW);
#pragma unroll
              for (int i = 0; i < CH; ++i) {
                const int idx = i * 32 + lane, key = idx / CH, ch = idx % CH;
                const long long o = __shfl_sync(0xffffffffu, off, key) + ch * 16;
                cp_async16(dst + key * ROW + ch * 16, src + o, (okm >> key) & 1u);
              }
            }
            cp_commit();
          };
#pragma unroll
          for (int k = 0; k < kTRaw - 1; ++k) issue(k);
#pragma unroll 1
          for (int k = 0; k < 2 * n; ++k) {
            cp_wait<kTRaw - 2>();
            __syncwarp();
            issue(k + kTRaw - 1);  // (into the slot that the last step left)
            int tile;
            bool is_k;
            load_step<DUAL>(n, k, tile, is_k);
            const int slot = it % NS;
            mbar_wait(&empty_bar[slot], ((it / NS) & 1) ^ 1, status, abort_flag);
            ++it;
            const uint8_t* rows = raw + (k % kTRaw) * (32 * ROW);
            uint8_t* out = sm + C::Q + slot * TILE;
#pragma unroll 2
            for (int i = 0; i < G; ++i) {
              // eight lanes store to eight different 16-byte columns: two groups x four rows
              int key, gr;
              if (G == 4) {
                key = i * 8 + ((lane >> 1) & 3) + ((lane >> 4) & 1) * 4;
                gr = (lane & 1) + ((lane >> 3) & 1) * 2;
              } else {
                key = i * 16 + (lane >> 1);
                gr = lane & 1;
              }
              const uint4 codes = *reinterpret_cast<const uint4*>(rows + key * ROW + gr * 16);
              const uint32_t sz = *reinterpret_cast<const uint32_t*>(rows + key * ROW + D / 2 + gr * 4);
              const uint32_t s2 = __byte_perm(sz, sz, 0x1010), z2 = __byte_perm(sz, sz, 0x3232);
              const int r = w4 * 32 + key;
              uint8_t* dst = out + (gr >> 1) * HALF + r * 128;
              const uint32_t* cw = &codes.x;
#pragma unroll
              for (int wd = 0; wd < 4; ++wd) {
                const uint32_t c = cw[wd];
                const uint32_t p0 = H::dequant(nib<T, 0>(c), s2, z2), p1 = H::dequant(nib<T, 1>(c), s2, z2);
                const uint32_t p2 = H::dequant(nib<T, 2>(c), s2, z2), p3 = H::dequant(nib<T, 3>(c), s2, z2);
                uint4 v = make_uint4(p0, p1, p2, p3);
                if (is_k)
                  v = make_uint4(__byte_perm(p0, p1, 0x5410), __byte_perm(p2, p3, 0x5410), __byte_perm(p0, p1, 0x7632),
                                 __byte_perm(p2, p3, 0x7632));
                *reinterpret_cast<uint4*>(dst + ((((gr & 1) * 4 + wd) ^ (r & 7)) << 4)) = v;
              }
            }
            fence_async_proxy();
            mbar_arrive(&full_bar[slot]);
          }
          cp_wait<0>();
          __syncwarp();
          tc += n;
        }
      }
    } else {
      // ------------------------------------------------------------------ softmax and output
      if constexpr (BITS4) asm volatile("setmaxnreg.inc.sync.aligned.u32 176;");
      else asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
      const int s = (warp - 4) >> 2;                  // stream
      const int row = (warp & 3) * 32 + lane;         // TMEM lane
      const int r = DUAL ? s * 128 + row : row;       // row of the row tile
      const uint32_t t_lane = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
      const uint32_t t_s = t_lane + kTmemS + s * 128, t_o = t_lane + kTmemO + s * 128;
      int it = 0, tc = 0, ns = 0, no = 0;
      const int tok_r = r / a.gs, sub_r = r % a.gs;
      int nb = 0;
      auto both = [&]() {  // the streams meet (bounded, unlike a named barrier)
        __syncwarp();
        mbar_arrive(&both_bar);
        mbar_wait(&both_bar, nb & 1, status, abort_flag);
        __syncwarp();
        ++nb;
      };
      while (__all_sync(0xffffffffu, next_segment(seg, g))) {
        mbar_arrive(&seg_empty[seg % kTSegs]);
        ++seg;
        const int n = g.t1 - g.t0;
        const bool row_ok = tok_r < g.toks && sub_r < g.heads;
        const long long tok = g.tok + tok_r;
        const int head = g.head + sub_r;
        const bool some = __any_sync(0xffffffffu, row_ok);  // a row of this warp is in use
        float m = kNegInf, l = 0.f;
        auto visible = [&](int j) {  // this row, key j
          if (!row_ok || j >= g.keys) return false;
          const int lj = j - g.prefix;
          if (a.tree == nullptr) return lj <= g.i0 + tok_r;
          if (lj < 0) return true;
          return (lj >> 5) < a.tree_words &&
                 ((static_cast<uint32_t>(a.tree[tok * a.tree_stride + (lj >> 5)]) >> (lj & 31)) & 1u) != 0;
        };
        for (int i = DUAL ? 0 : s; i < n; i += DUAL ? 1 : 2) {
          const int j0 = (g.t0 + i) * kTBK;
          const bool cut = j0 + kTBK > g.open || j0 + kTBK > g.keys;
          mbar_wait(&s_bar[s], ns & 1, status, abort_flag);
          tc_fence_after();
          // (with two row tiles over the same V the first stream looks after it for both: a thread fences its own
          // stores, and the second stream's product is issued behind the first one's)
          if (cut && (!DUAL || s == 0)) {
            // V: what no mask stops from entering the product has to be finite.  (S being there says that
            // what its slot held before has been used, so that the wait can only be for this V.)
            const int vstep = it + (DUAL ? 2 * i + 1 : i + min(i + 2, n));
            mbar_wait(&full_bar[vstep % NS], (vstep / NS) & 1, status, abort_flag);
            uint4* vp = reinterpret_cast<uint4*>(sm + C::Q + (vstep % NS) * TILE);
            bool bad = false;
#pragma unroll 4
            for (int c = 0; c < D / 8; ++c) {
              const int at = c * 128 + (tid & 127);  // 16 bytes of key (at / 8) % 128
              uint4 v = vp[at];
              uint32_t* u = reinterpret_cast<uint32_t*>(&v);
              bool hit = false;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if (H::nonfinite(u[e] & 0xffffu)) u[e] &= 0xffff0000u, hit = true;
                if (H::nonfinite(u[e] >> 16)) u[e] &= 0xffffu, hit = true;
              }
              if (hit) {
                bad = true;
                // (not for rows behind the keys; before the value goes)
                if (j0 + ((at >> 3) & 127) < g.keys) *reinterpret_cast<volatile int*>(&s_fix) = 1;
                __threadfence_block();
                vp[at] = v;
              }
            }
            if (bad) fence_async_proxy();
          }
          if (!some) {  // nothing to weigh: the product may have what is there
            mbar_arrive(&p_bar[s][0]);
            mbar_arrive(&p_bar[s][1]);
            ++ns;
            continue;
          }
          const uint32_t* ok = s_pages[(tc + i) % kTOkRing];  // a bit per page, or per key of a 4-bit cache
          const bool masked = cut || (BITS4 ? (ok[0] & ok[BITS4 ? 1 : 0] & ok[BITS4 ? 2 : 0] & ok[BITS4 ? 3 : 0]) : ok[0]) != 0xffffffffu;
          uint32_t x[4][32];
#pragma unroll
          for (int q = 0; q < 4; ++q) tmem_ld32_issue(t_s + q * 32, x[q]);
#pragma unroll
          for (int q = 0; q < 4; ++q) tmem_ld_done(x[q]);
          if (masked) {
            const int psb = min(1 << a.c.page_shift, kTBK);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const int jq = j0 + q * 32;
              uint32_t see = 0;  // bit e: this row sees key jq + e
              const int left = min(32, g.keys - jq);
              if (row_ok && left > 0) {
                see = left == 32 ? 0xffffffffu : (1u << left) - 1u;
                const int lj = jq - g.prefix;
                if (a.tree == nullptr) {
                  const int c = g.i0 + tok_r - lj + 1;
                  see &= c >= 32 ? 0xffffffffu : c <= 0 ? 0u : (1u << c) - 1u;
                } else if (lj > -32) {
                  const int w0 = lj >> 5, sh = lj & 31;  // (floor: lj may be negative)
                  const int* words = a.tree + tok * a.tree_stride;
                  const uint32_t lo = w0 < 0 ? 0xffffffffu : w0 < a.tree_words ? static_cast<uint32_t>(words[w0]) : 0u;
                  const uint32_t hi = w0 + 1 < a.tree_words ? static_cast<uint32_t>(words[w0 + 1]) : 0u;
                  see &= __funnelshift_r(lo, hi, sh);
                }
                if constexpr (BITS4) {
                  see &= ok[q];
                } else if (ok[0] != 0xffffffffu) {
                  for (int e = 0; e < 32; ++e)
                    if (!((ok[0] >> ((q * 32 + e) / psb)) & 1u)) see &= ~(1u << e);
                }
              }
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!((see >> e) & 1u)) x[q][e] = __float_as_uint(kNegInf);
            }
          }

          float top[4] = {kNegInf, kNegInf, kNegInf, kNegInf};
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int e = 0; e < 32; e += 2)
              top[(e >> 1) & 3] = max3(top[(e >> 1) & 3], __uint_as_float(x[q][e]), __uint_as_float(x[q][e + 1]));
          const float tmax = max3(max3(top[0], top[1], top[2]), top[3], top[3]) * a.scale_log2;
          const bool grew = tmax > m + (kGrow + H::kLift);  // (paged_math.cuh)
          if (__any_sync(0xffffffffu, grew)) {
            const float now = grew ? tmax - H::kLift : m;
            const float f = m == kNegInf ? 0.f : exp2_fast(m - now);
            m = now;
            l *= f;
            if (i >= (DUAL ? 1 : 2)) {
              // (this stream's last product is complete: it was issued before the S just waited for)
#pragma unroll 2
              for (int q = 0; q < D / 16; ++q) {
                uint32_t o[16];
                tmem_ld16_wait(t_o + q * 16, o);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                tmem_st16(t_o + q * 16, o);
              }
              tmem_st_done();
            }
          }
          const float mm = m == kNegInf ? 0.f : m;
          const uint64_t scale2 = pair(a.scale_log2, a.scale_log2), mm2 = pair(-mm, -mm);
          uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t p[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              float v0, v1;
              unpair(fma2(pair(__uint_as_float(x[q][2 * e]), __uint_as_float(x[q][2 * e + 1])), scale2, mm2), v0, v1);
              v0 = exp2_fast(v0);
              v1 = exp2_fast(v1);
              sum[e & 1] = add2(sum[e & 1], pair(v0, v1));
              p[e] = H::pack(v0, v1);
            }
            tmem_st16(t_s + q * 16, p);
            if (q & 1) {  // the product starts on the first 64 keys while the others are worked on
              tmem_st_done();
              tc_fence_before();
              mbar_arrive(&p_bar[s][q >> 1]);
            }
          }
          float s0, s1;
          unpair(add2(sum[0], sum[1]), s0, s1);
          l += s0 + s1;
          ++ns;
        }

        // ---- output
        const bool mine = DUAL || n > s;  // this stream had a tile
        if (mine) {
          mbar_wait(&o_bar[s], no & 1, status, abort_flag);
          ++no;
          tc_fence_after();
        }
        const bool whole = g.slot < 0;
        const long long slot = g.slot;
        float f_own = 1.f, f_other = 0.f;
        if constexpr (!DUAL) {
          float2* ml = reinterpret_cast<float2*>(sm + C::Q + NS * TILE);
          ml[s * 128 + row] = make_float2(m, l);
          both();
          const float2 o = ml[(s ^ 1) * 128 + row];
          both();  // (the outputs go to the same place)
          const float mx = fmaxf(m, o.x);
          // a stream with no visible key has a maximum of -inf and an output of 0
          f_own = m == kNegInf ? 1.f : exp2_fast(m - mx);
          f_other = o.x == kNegInf ? 1.f : exp2_fast(o.x - mx);
          l = s == 0 ? l * f_own + o.y * f_other : o.y * f_other + l * f_own;
          m = mx;
        }
        const bool fix = *reinterpret_cast<volatile int*>(&s_fix) != 0;
        float inv = 1.f;
        if (whole) inv = l == 0.f ? 0.f : 1.f / l;
        auto load_o = [&](int q, uint32_t (&o)[32]) {  // 32 columns of this stream's output
          __syncwarp();
          if (mine) {
            tmem_ld32_issue(t_o + q * 32, o);
            tmem_ld_done(o);
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0u;
          }
          if (fix && row_ok) {
            // non-finite values that were taken out of this stream's masked tiles, and that this row sees
            for (int i = DUAL ? 0 : s; i < n; i += DUAL ? 1 : 2) {
              const int j0 = (g.t0 + i) * kTBK;
              if (j0 + kTBK <= g.open && j0 + kTBK <= g.keys) continue;
              for (int j = j0; j < min(j0 + kTBK, g.keys); ++j) {
                if (!visible(j)) continue;
                const int page = a.table[g.b * a.table_stride + (j >> a.c.page_shift)];
                if (page < 0 || page >= a.c.num_pages) continue;
                const uint8_t* v = a.c.v + page * a.c.page_stride + g.kvh * a.c.head_stride +
                                   (j & ((1 << a.c.page_shift) - 1)) * a.c.token_stride;
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                  float f;
                  int at = e;
                  if constexpr (BITS4) {
                    const uint32_t sz = *reinterpret_cast<const uint32_t*>(v + D / 2 + q * 4);
                    f = H::lo(value_of<T>((v[q * 16 + e / 2] >> (4 * (e & 1))) & 15u, sz));  // (as it was unpacked)
                    at = (e & ~7) + nibble_place(e & 7);
                  } else {
                    f = to_f32<T>(reinterpret_cast<const T*>(v)[q * 32 + e]);
                  }
                  if (!isfinite(f)) o[at] = __float_as_uint(__uint_as_float(o[at]) + f);
                }
              }
            }
          }
          __syncwarp();
        };
        auto store_o = [&](int q, const uint32_t (&o)[32]) {
          if (!row_ok) return;
          auto col = [&](int d) { return __uint_as_float(o[BITS4 ? (d & ~7) + nibble_place(d & 7) : d]); };
          if (whole) {
            uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + tok * a.o_ts + head * a.o_hs + q * 32);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint4 v;
              v.x = H::pack(col(8 * c) * inv, col(8 * c + 1) * inv);
              v.y = H::pack(col(8 * c + 2) * inv, col(8 * c + 3) * inv);
              v.z = H::pack(col(8 * c + 4) * inv, col(8 * c + 5) * inv);
              v.w = H::pack(col(8 * c + 6) * inv, col(8 * c + 7) * inv);
              dst[c] = v;
            }
          } else {
            float* dst = a.part_o + (slot * D + q * 32) * R + r;  // rows innermost: a warp's store is one line
#pragma unroll
            for (int e = 0; e < 32; ++e) dst[e * R] = col(e);
          }
        };
        if constexpr (DUAL) {
#pragma unroll 1
          for (int q = 0; q < D / 32; ++q) {
            uint32_t o[32];
            load_o(q, o);
            store_o(q, o);
          }
        } else {
          // each stream finishes half of the columns: it leaves the other's, 32 at a time, as [column][row]
          constexpr int HQ = D / 64;
          float* give = reinterpret_cast<float*>(sm + C::Q + NS * TILE) + s * (32 * 128);
          const float* take = reinterpret_cast<const float*>(sm + C::Q + NS * TILE) + (s ^ 1) * (32 * 128);
#pragma unroll 1
          for (int q = 0; q < HQ; ++q) {
            uint32_t o[32];
            load_o((s ^ 1) * HQ + q, o);
#pragma unroll
            for (int e = 0; e < 32; ++e) give[e * 128 + row] = __uint_as_float(o[e]) * f_own;
            both();
            load_o(s * HQ + q, o);
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              // (the sum in the streams' order on both sides)
              const float own = __uint_as_float(o[e]) * f_own, other = take[e * 128 + row];
              o[e] = __float_as_uint(s == 0 ? own + other : other + own);
            }
            store_o(s * HQ + q, o);
            if (q + 1 < HQ) both();
          }
        }
        if ((DUAL || s == 0) && row_ok) {
          if (!whole) {
            *reinterpret_cast<float2*>(a.part_ml + (slot * R + r) * 2) = make_float2(m, l);
          } else if (a.lse != nullptr) {
            a.lse[tok * (static_cast<long long>(a.c.Hkv) * a.g) + head] = l == 0.f ? kNegInf : (m + log2f(l)) * kLn2;
          }
        }
        tc_fence_before();
        it += 2 * n;
        tc += n;
        if constexpr (!DUAL) both();  // both streams are done with the exchange
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 2) tmem_dealloc(tmem, 512);
}

struct Variant {
  const void* fn;
  int smem, threads;
};
template <int D, bool DUAL, bool BITS4>
Variant variant(bool bf16) {
  using C = TcCfg<D, DUAL, BITS4>;
  return {bf16 ? reinterpret_cast<const void*>(paged_attn_tc_kernel<D, DUAL, BITS4, __nv_bfloat16>)
               : reinterpret_cast<const void*>(paged_attn_tc_kernel<D, DUAL, BITS4, __half>),
          C::SMEM, C::THREADS};
}
template <int D>
Variant variant(bool dual, bool bits4, bool bf16) {
  if (dual) return bits4 ? variant<D, true, true>(bf16) : variant<D, true, false>(bf16);
  return bits4 ? variant<D, false, true>(bf16) : variant<D, false, false>(bf16);
}

std::atomic<int> g_smem_seen[16][64];

bool encode(CUtensorMap* map, const void* base, bool bf16, int rank, const cuuint64_t* dims, cuuint64_t* strides,
            const cuuint32_t* box) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return false;
  const cuuint32_t ones[4] = {1, 1, 1, 1};
  // (the stride of a dimension of size 1 means nothing; the encoder wants a usable one)
  for (int i = 1; i < rank; ++i)
    if (dims[i] == 1) strides[i - 1] = 16;
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank, const_cast<void*>(base),
            dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Rows [page_size][kv_heads][num_pages] of D values; boxes of 64 dims x one page's rows (at most a tile).
bool encode_cache(CUtensorMap* map, const PagedCacheArgs& c, const void* base, int D, bool bf16) {
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(D), 1ull << c.page_shift, static_cast<cuuint64_t>(c.Hkv),
                              static_cast<cuuint64_t>(c.num_pages)};
  cuuint64_t strides[3] = {static_cast<cuuint64_t>(c.token_stride), static_cast<cuuint64_t>(c.head_stride),
                           static_cast<cuuint64_t>(c.page_stride)};
  const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(std::min(1 << c.page_shift, kTBK)), 1, 1};
  return encode(map, base, bf16, 4, dims, strides, box);
}

// Rows [heads][tokens] of q; boxes of 64 dims x gs heads x tq tokens: the rows of a row tile.
bool encode_queries(CUtensorMap* map, const AttnArgs& a, int D, bool bf16) {
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(a.c.Hkv) * a.g,
                              static_cast<cuuint64_t>(a.N)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(a.q_hs) * 2, static_cast<cuuint64_t>(a.q_ts) * 2};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(a.gs), static_cast<cuuint32_t>(a.tq)};
  return encode(map, a.q, bf16, 3, dims, strides, box);
}

}  // namespace

bool tc_takes(const PagedCacheArgs& c, bool bits4) {
  return bits4 || (c.page_shift >= 3 && c.num_pages >= 1 && c.num_pages < 0x7fffffffll);
}

// Two row tiles at a time where a key head has more than 128 rows: at 136 to 192 rows (16 sequences of
// 8192 keys) 148-150 us against 197-205 with the keys read once per row tile (16 bits), 180-187 against
// 290-302 (4 bits); at 128 rows 146 against 109-117.
bool plan_attn_tc(int N, int B, int g, int D, bool bits4, int sms, AttnPlan* p) {
  if (D > 128 || g > 128) return false;
  const long long rows = (static_cast<long long>(N) * g + B - 1) / B;
  if (rows <= (bits4 ? kTcAboveRows4 : kTcAboveRows16)) return false;
  p->rows = rows > 128 ? 256 : 128;
  p->grid = sms;
  p->min_tiles = 2;
  p->seg_cost = 3;
  return true;
}

cudaError_t launch_attn_tc(AttnArgs a, const AttnPlan& p, int D, bool bf16, bool bits4, cudaStream_t stream, bool pdl,
                           bool* fits) {
  CUtensorMap tq, tk, tv;
  *fits = encode_queries(&tq, a, D, bf16);
  if (bits4) {
    tk = tv = tq;  // (not used)
  } else {
    *fits = *fits && encode_cache(&tk, a.c, a.c.k, D, bf16) && encode_cache(&tv, a.c, a.c.v, D, bf16);
  }
  if (!*fits) return cudaSuccess;
  const bool dual = p.rows == 256;
  const Variant v = D == 64 ? variant<64>(dual, bits4, bf16) : variant<128>(dual, bits4, bf16);
  cudaError_t err = ensure_dyn_smem(v.fn, v.smem, g_smem_seen[(D == 128) * 8 + dual * 4 + bits4 * 2 + bf16], 64);
  if (err != cudaSuccess) return err;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.grid);
  cfg.blockDim = dim3(v.threads);
  cfg.dynamicSmemBytes = v.smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  void* params[] = {&a, &tq, &tk, &tv};
  err = cudaLaunchKernelExC(&cfg, v.fn, params);
  if (err != cudaSuccess) return err;
  return launch_attn_join(a, p, D, bf16, stream, pdl);
}

}  // namespace smb

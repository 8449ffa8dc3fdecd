// Attention of the new tokens of each sequence over its paged cache, for few query rows per key
// head (decode, small draft trees) and for every cache the tcgen05 kernel does not take: 16-bit
// caches with any page size or head size, and 4-bit caches.
//
//   out_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = 2^(scale log2(e) q_i.k_j - m_i)
//
// One pass over the keys with a running maximum m (base-2 units) and sum per row.  Bound by
// memory at these sizes: a key head's rows are read once for all of its g query heads and all
// new tokens (up to 16 or 32 rows), so the kernel is built to stream.
//
// Measured: 32 sequences of up to 32768 keys, one token, 32 / 8 heads of 128, fp16: 2.77 GB in 427-448 us,
// 6.2-6.5 TB/s, 0.94-0.99 of the measured copy rate.
//
// A warp owns a ring of NST stages in shared memory, KS keys each (K and V rows), filled by its
// own cp.async and read only by itself: no CTA barrier while keys stream, the four warps of a CTA
// drift apart freely, and 2 CTAs of an SM keep 48 to 130 KB of loads in flight (one SM's share of
// bandwidth x latency is about 44 KB).  The warps' partial results meet once per segment.
// Matrix products are m16n8k16 with the query rows as the 16: at 16 rows the legacy pipe needs
// 16 flop per byte of cache, far below its balance.
//
// 16-bit rows sit in shared memory with their 16-byte chunks XOR-ed by the row, so ldmatrix meets
// no bank conflict.  4-bit rows stay packed until they are in registers:
//  - keys: a thread's fragment of a group of 32 dims is one 32-bit word (its 8 dims; the query
//    fragments are laid out in the same order), each nibble becomes 16 + code by one shift and one
//    and-or (the nibble set into the mantissa of 16.0); scale and zero are applied to the product of
//    a group, s (q.(16 + code)) + (z - 16 s) sum(q), in 32 bits: the scores see no rounding of keys.
//  - values: pairs along the keys are made by one byte permute of two keys' words, then
//    (16 + code) - 16 (exact) times scale plus zero, one rounding to the 16-bit type as a 16-bit
//    cache would have it.
//
// What is masked contributes nothing whatever it holds: rows past the keys and rows of bad pages
// are zero-filled, and where a mask cuts a tile, non-finite values are taken out of the product
// and added to the rows that do see them.  For a 4-bit group that means its unpacked values: they may
// overflow the 16-bit type though scale and zero are finite.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "paged_math.cuh"
#include "paged_plan.cuh"

namespace smb {
namespace {

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

template <int D, int MT, bool BITS4>
struct MmaCfg {
  static constexpr int R = 16 * MT;
  static constexpr int KS = BITS4 ? 32 : 16;       // keys of a warp's stage
  static constexpr int BK = 4 * KS;                // keys of a CTA's tile
  static constexpr int ROW = BITS4 ? kv4_row_bytes(D) : 2 * D;
  static constexpr int NST = BITS4 ? 4 : 3;
  static constexpr int STAGE = 2 * KS * ROW;
  static constexpr int QF = MT * (D / 16) * 512;   // query fragments in fragment order
  static constexpr int RING = 4 * NST * STAGE;
  static constexpr int OP = D + 4;                 // floats of a row of the merge buffer
  static constexpr int MERGE = 4 * R * OP * 4;
  static constexpr int BODY = RING > MERGE ? RING : MERGE;
  static constexpr int ML = 4 * R * 8;             // (m, l) of each warp's rows
  static constexpr int SMEM = QF + BODY + ML + 128;
  static constexpr int CTAS = SMEM <= 56 * 1024 ? 4 : SMEM <= 75 * 1024 ? 3 : SMEM <= 113 * 1024 ? 2 : 1;
};

template <int D, int MT, bool BITS4, typename T>
__global__ void __launch_bounds__(128, (MmaCfg<D, MT, BITS4>::CTAS > 2 && MT == 2) ? 2 : MmaCfg<D, MT, BITS4>::CTAS)
    paged_attn_mma_kernel(const __grid_constant__ AttnArgs a) {
  using C = MmaCfg<D, MT, BITS4>;
  using H = Half2<T>;
  constexpr int R = C::R, KS = C::KS, BK = C::BK, ROW = C::ROW, NST = C::NST;
  constexpr int CH = ROW / 16;   // 16-byte chunks of a row
  constexpr int KT = D / 16;     // k steps of q.k, pairs of n tiles of p.v
  constexpr int G = D / 32;      // groups of a 4-bit row
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ PlanShared s_plan;
  __shared__ uint32_t s_ok[4][NST];
  uint4* qf = reinterpret_cast<uint4*>(smem);
  uint8_t* body = smem + C::QF;
  float2* s_ml = reinterpret_cast<float2*>(smem + C::QF + C::BODY);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int r4 = lane >> 2, c4 = lane & 3;
  uint8_t* ring = body + warp * NST * C::STAGE;
  const uint32_t ring_s = smem_u32(ring);

  pdl_wait_prior_grids();
  pdl_launch_dependents();
  const int cta = blockIdx.x;
  const long long W = plan_build<BK>(a, &s_plan, gridDim.x);
  Work k;
  if (!work_begin<BK>(a, &s_plan, W, cta, gridDim.x, k)) {
    if (tid == 0) leave_record(a, cta, k);
    return;
  }

  while (true) {
    const Cursor& cur = k.cur;
    const int t0 = k.t0, t1 = k.t1;
    const int kvh = cur.vh / a.nsub, sub = cur.vh % a.nsub;
    const int heads = min(a.gs, a.g - sub * a.gs);
    const int tok0 = cur.qt * a.tq, toks = min(a.tq, cur.s.n - tok0);
    const int prefix = cur.s.L - cur.s.n;  // keys before the new tokens (negative: fewer keys than tokens)
    auto row_ok = [&](int r) { return r < toks * a.gs && r % a.gs < heads; };
    auto sees = [&](int r, int j) {  // row r of the tile, key j < L
      const int i = tok0 + r / a.gs, lj = j - prefix;
      if (a.tree == nullptr) return lj <= i;
      if (lj < 0) return true;
      if ((lj >> 5) >= a.tree_words) return false;
      return ((static_cast<uint32_t>(a.tree[(cur.s.s0 + i) * a.tree_stride + (lj >> 5)]) >> (lj & 31)) & 1u) != 0;
    };

    // ---- query fragments, in the order the products read them
    float qsum[BITS4 ? MT : 1][2][BITS4 ? G : 1];
    if constexpr (!BITS4) {
      for (int i = tid; i < MT * KT * 32; i += 128) {
        const int ln = i & 31, kk = (i >> 5) % KT, mt = (i >> 5) / KT;
        uint32_t v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = mt * 16 + (ln >> 2) + (e & 1) * 8;
          const int d = kk * 16 + (ln & 3) * 2 + (e >> 1) * 8;
          v[e] = 0;
          if (row_ok(r)) {
            const T* p = static_cast<const T*>(a.q) + (cur.s.s0 + tok0 + r / a.gs) * a.q_ts +
                         (kvh * a.g + sub * a.gs + r % a.gs) * a.q_hs + d;
            v[e] = *reinterpret_cast<const uint32_t*>(p);
          }
        }
        qf[i] = make_uint4(v[0], v[1], v[2], v[3]);
      }
    } else {
      // group gq, thread c4: dims 32 gq + 8 c4 + (0..7); nibble e pairs dims e and e + 4
      for (int i = tid; i < MT * G * 32; i += 128) {
        const int ln = i & 31, gq = (i >> 5) % G, mt = (i >> 5) / G;
        uint4 rowv[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = mt * 16 + (ln >> 2) + e * 8;
          rowv[e] = make_uint4(0u, 0u, 0u, 0u);
          if (row_ok(r)) {
            const T* p = static_cast<const T*>(a.q) + (cur.s.s0 + tok0 + r / a.gs) * a.q_ts +
                         (kvh * a.g + sub * a.gs + r % a.gs) * a.q_hs + gq * 32 + (ln & 3) * 8;
            rowv[e] = *reinterpret_cast<const uint4*>(p);
          }
        }
        auto pair = [&](const uint4& v, int e) {  // dims (e, e + 4)
          const uint32_t lo = e < 2 ? v.x : v.y, hi = e < 2 ? v.z : v.w;
          return __byte_perm(lo, hi, (e & 1) ? 0x7632 : 0x5410);
        };
#pragma unroll
        for (int s = 0; s < 2; ++s)
          qf[(mt * KT + 2 * gq + s) * 32 + ln] =
              make_uint4(pair(rowv[0], 2 * s), pair(rowv[1], 2 * s), pair(rowv[0], 2 * s + 1), pair(rowv[1], 2 * s + 1));
      }
    }
    __syncthreads();
    if constexpr (BITS4) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int gq = 0; gq < G; ++gq) {
          float s0 = 0.f, s1 = 0.f;
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const uint4 v = qf[(mt * KT + 2 * gq + s) * 32 + lane];
            s0 += (H::lo(v.x) + H::hi(v.x)) + (H::lo(v.z) + H::hi(v.z));
            s1 += (H::lo(v.y) + H::hi(v.y)) + (H::lo(v.w) + H::hi(v.w));
          }
#pragma unroll
          for (int o = 1; o < 4; o <<= 1) {
            s0 += __shfl_xor_sync(0xffffffffu, s0, o);
            s1 += __shfl_xor_sync(0xffffffffu, s1, o);
          }
          qsum[mt][0][gq] = s0;
          qsum[mt][1][gq] = s1;
        }
    }

    float O[MT][2 * KT][4];
    float m[MT][2], l[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int t = 0; t < 2 * KT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) O[mt][t][e] = 0.f;
      m[mt][0] = m[mt][1] = kNegInf;
      l[mt][0] = l[mt][1] = 0.f;
    }

    const uint8_t* kbase = a.c.k + kvh * a.c.head_stride;
    const uint8_t* vbase = a.c.v + kvh * a.c.head_stride;
    const int* table = a.table + cur.b * a.table_stride;
    const int page_mask = (1 << a.c.page_shift) - 1;
    // page of the key that this lane looks up for tile t (one tile ahead of its loads)
    auto look_up = [&](int t) {
      const int j = t * BK + warp * KS + (KS == 32 ? lane : (lane & 15));
      return (t < t1 && j < cur.keys) ? table[j >> a.c.page_shift] : -1;
    };
    int page = look_up(t0);
    auto issue = [&](int t) {
      if (t < t1) {
        const int st = (t - t0) % NST;
        const int j = t * BK + warp * KS + (KS == 32 ? lane : (lane & 15));
        const bool in = j < cur.keys;
        const bool ok = in && page >= 0 && page < a.c.num_pages;
        if (in && !ok) record_status(a.status, kDevBadPage);
        const long long off = ok ? page * a.c.page_stride + (j & page_mask) * a.c.token_stride : 0;
        const uint32_t okm = __ballot_sync(0xffffffffu, ok);
        if (lane == 0) s_ok[warp][st] = okm;
        page = look_up(t + 1);
        const uint32_t dst = ring_s + st * C::STAGE;
#pragma unroll
        for (int i = 0; i < KS * CH; i += 32) {
          const int idx = i + lane;
          const int key = min(idx / CH, KS - 1), ch = idx % CH;
          const long long o = __shfl_sync(0xffffffffu, off, key) + ch * 16;
          const bool fill = (okm >> key) & 1u;
          if ((KS * CH) % 32 == 0 || idx < KS * CH) {
            const uint32_t d = BITS4 ? dst + key * ROW + ch * 16 : dst + key * ROW + ((ch ^ (key & 7)) << 4);
            cp_async16(d, kbase + o, fill);
            cp_async16(d + KS * ROW, vbase + o, fill);
          }
        }
      }
      cp_commit();
    };
#pragma unroll
    for (int s = 0; s < NST - 1; ++s) issue(t0 + s);

    for (int t = t0; t < t1; ++t) {
      cp_wait<NST - 2>();
      __syncwarp();
      issue(t + NST - 1);
      const int st = (t - t0) % NST;
      uint8_t* ks = ring + st * C::STAGE;
      uint8_t* vs = ks + KS * ROW;
      const uint32_t ks_s = ring_s + st * C::STAGE, vs_s = ks_s + KS * ROW;
      const int j0 = t * BK + warp * KS;
      const uint32_t okm = s_ok[warp][st];
      // the first key that some row may not see
      const int open = a.tree != nullptr ? prefix : prefix + tok0 + 1;
      const bool masked = okm != 0xffffffffu || j0 + KS > open;

      float S[MT][KS / 8][4];
      if constexpr (!BITS4) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) S[mt][n][e] = 0.f;
        const int key = (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
        for (int kk = 0; kk < KT; ++kk) {
          uint32_t b[4];
          ldsm4(ks_s + key * ROW + (((2 * kk + ((lane >> 3) & 1)) ^ (key & 7)) << 4), b);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            const uint4 q4 = qf[(mt * KT + kk) * 32 + lane];
            const uint32_t q[4] = {q4.x, q4.y, q4.z, q4.w};
            H::mma(S[mt][0], q, b[0], b[1]);
            H::mma(S[mt][1], q, b[2], b[3]);
          }
        }
      } else {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int n = 0; n < KS / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) S[mt][n][e] = 0.f;
#pragma unroll
        for (int gq = 0; gq < G; ++gq) {
          uint32_t q[MT][2][4];
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
              const uint4 q4 = qf[(mt * KT + 2 * gq + s) * 32 + lane];
              q[mt][s][0] = q4.x;
              q[mt][s][1] = q4.y;
              q[mt][s][2] = q4.z;
              q[mt][s][3] = q4.w;
            }
#pragma unroll
          for (int n = 0; n < KS / 8; ++n) {
            const uint32_t wd = *reinterpret_cast<const uint32_t*>(ks + (n * 8 + r4) * ROW + gq * 16 + c4 * 4);
            const uint32_t b0 = nib<T, 0>(wd), b1 = nib<T, 1>(wd), b2 = nib<T, 2>(wd), b3 = nib<T, 3>(wd);
            const uint32_t sz0 = *reinterpret_cast<const uint32_t*>(ks + (n * 8 + 2 * c4) * ROW + D / 2 + gq * 4);
            const uint32_t sz1 = *reinterpret_cast<const uint32_t*>(ks + (n * 8 + 2 * c4 + 1) * ROW + D / 2 + gq * 4);
            const float sa = H::lo(sz0), sb = H::lo(sz1);
            const float za = fmaf(-16.f, sa, H::hi(sz0)), zb = fmaf(-16.f, sb, H::hi(sz1));
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              float acc[4] = {0.f, 0.f, 0.f, 0.f};
              H::mma(acc, q[mt][0], b0, b1);
              H::mma(acc, q[mt][1], b2, b3);
              S[mt][n][0] = fmaf(sa, acc[0], fmaf(za, qsum[mt][0][gq], S[mt][n][0]));
              S[mt][n][1] = fmaf(sb, acc[1], fmaf(zb, qsum[mt][0][gq], S[mt][n][1]));
              S[mt][n][2] = fmaf(sa, acc[2], fmaf(za, qsum[mt][1][gq], S[mt][n][2]));
              S[mt][n][3] = fmaf(sb, acc[3], fmaf(zb, qsum[mt][1][gq], S[mt][n][3]));
            }
          }
        }
      }

      if (masked) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int n = 0; n < KS / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int kl = n * 8 + 2 * c4 + (e & 1), r = mt * 16 + r4 + (e >> 1) * 8;
              if (!((okm >> kl) & 1u) || !sees(r, j0 + kl) || !row_ok(r)) S[mt][n][e] = kNegInf;
              else S[mt][n][e] *= a.scale_log2;
            }
        // non-finite values behind the mask: to the rows that see them directly, out of the product
        bool bad = false;
        if constexpr (!BITS4) {
          for (int i = lane; i < KS * D / 2; i += 32) {
            const uint32_t v = reinterpret_cast<const uint32_t*>(vs)[i];
            bad = bad || H::nonfinite(v & 0xffffu) || H::nonfinite(v >> 16);
          }
        } else {
          for (int i = lane; i < KS * G; i += 32) {
            bad = bad || group_overflows<T>(*reinterpret_cast<const uint32_t*>(vs + (i / G) * ROW + D / 2 + (i % G) * 4));
          }
        }
        if (__any_sync(0xffffffffu, bad)) {
          for (int kl = 0; kl < KS; ++kl) {
            if (!((okm >> kl) & 1u)) continue;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
              for (int hh = 0; hh < 2; ++hh) {
                const int r = mt * 16 + r4 + hh * 8;
                if (!row_ok(r) || !sees(r, j0 + kl)) continue;
#pragma unroll
                for (int t2 = 0; t2 < 2 * KT; ++t2)
#pragma unroll
                  for (int e = 0; e < 2; ++e) {
                    float v;
                    if constexpr (!BITS4) {
                      const int d = t2 * 8 + 2 * c4 + e;
                      v = to_f32<T>(*reinterpret_cast<const T*>(vs + kl * ROW + (((d >> 3) ^ (kl & 7)) << 4) + (d & 7) * 2));
                    } else {
                      const int d = (2 * c4 + e) * (D / 8) + t2;
                      const uint32_t sz = *reinterpret_cast<const uint32_t*>(vs + kl * ROW + D / 2 + (d >> 5) * 4);
                      v = H::lo(value_of<T>((vs[kl * ROW + (d >> 1)] >> (4 * (d & 1))) & 15u, sz));
                    }
                    if (!isfinite(v)) O[mt][t2][hh * 2 + e] += v;
                  }
              }
          }
          __syncwarp();
          if constexpr (!BITS4) {
            for (int i = lane; i < KS * D; i += 32) {
              uint16_t* p = reinterpret_cast<uint16_t*>(vs) + i;
              if (H::nonfinite(*p)) *p = 0;
            }
          } else {
            for (int i = lane; i < KS * G; i += 32) {
              uint8_t* row = vs + (i / G) * ROW;
              uint32_t* sz = reinterpret_cast<uint32_t*>(row + D / 2 + (i % G) * 4);
              if (group_overflows<T>(*sz)) take_out_nonfinite<T>(reinterpret_cast<uint32_t*>(row + (i % G) * 16), sz);
            }
          }
          __syncwarp();
        }
      } else {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int n = 0; n < KS / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) S[mt][n][e] *= a.scale_log2;
      }

      // running maximum (paged_math.cuh)
      uint32_t P[MT][KS / 16][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        float top[2] = {kNegInf, kNegInf};
#pragma unroll
        for (int n = 0; n < KS / 8; ++n) {
          top[0] = fmaxf(top[0], fmaxf(S[mt][n][0], S[mt][n][1]));
          top[1] = fmaxf(top[1], fmaxf(S[mt][n][2], S[mt][n][3]));
        }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
          top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], o));
          top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], o));
        }
        // (m = -inf: any finite maximum is above it)
        const bool grew = top[0] > m[mt][0] + (kGrow + H::kLift) || top[1] > m[mt][1] + (kGrow + H::kLift);
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float now = fmaxf(m[mt][h], top[h] - H::kLift);
            const float f = m[mt][h] == kNegInf ? 0.f : exp2_fast(m[mt][h] - now);
            m[mt][h] = now;
            l[mt][h] *= f;
#pragma unroll
            for (int t2 = 0; t2 < 2 * KT; ++t2) {
              // (nothing was added to a row whose maximum was -inf but what the mask let in unscaled)
              if (f != 0.f || isfinite(O[mt][t2][2 * h])) O[mt][t2][2 * h] *= f;
              if (f != 0.f || isfinite(O[mt][t2][2 * h + 1])) O[mt][t2][2 * h + 1] *= f;
            }
          }
        }
        const float m0 = m[mt][0] == kNegInf ? 0.f : m[mt][0], m1 = m[mt][1] == kNegInf ? 0.f : m[mt][1];
#pragma unroll
        for (int n = 0; n < KS / 8; ++n) {
          const float p0 = exp2_fast(S[mt][n][0] - m0), p1 = exp2_fast(S[mt][n][1] - m0);
          const float p2 = exp2_fast(S[mt][n][2] - m1), p3 = exp2_fast(S[mt][n][3] - m1);
          l[mt][0] += p0 + p1;
          l[mt][1] += p2 + p3;
          P[mt][n >> 1][(n & 1) * 2] = H::pack(p0, p1);
          P[mt][n >> 1][(n & 1) * 2 + 1] = H::pack(p2, p3);
        }
      }

      if constexpr (!BITS4) {
        const int key = (lane & 7) + (((lane >> 3) & 1) << 3);
#pragma unroll
        for (int dd = 0; dd < KT; ++dd) {
          uint32_t b[4];
          ldsm4_t(vs_s + key * ROW + (((2 * dd + (lane >> 4)) ^ (key & 7)) << 4), b);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            H::mma(O[mt][2 * dd], P[mt][0], b[0], b[1]);
            H::mma(O[mt][2 * dd + 1], P[mt][0], b[2], b[3]);
          }
        }
      } else {
        constexpr int WD = D / 64;  // 32-bit words of a thread's D / 8 dims (r4 * D / 8 on)
#pragma unroll
        for (int k2 = 0; k2 < KS / 16; ++k2) {
          const uint8_t* row[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) row[e] = vs + (k2 * 16 + 2 * c4 + (e & 1) + (e >> 1) * 8) * ROW;
#pragma unroll
          for (int wv = 0; wv < WD; ++wv) {
            const int word = r4 * WD + wv;
            uint32_t sz[4], wd[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              wd[e] = *reinterpret_cast<const uint32_t*>(row[e] + word * 4);
              sz[e] = *reinterpret_cast<const uint32_t*>(row[e] + D / 2 + (word >> 2) * 4);
            }
            uint32_t b[2][8];
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
              const uint32_t s2 = __byte_perm(sz[2 * hh], sz[2 * hh + 1], 0x5410);
              const uint32_t z2 = __byte_perm(sz[2 * hh], sz[2 * hh + 1], 0x7632);
              const uint32_t x = __byte_perm(wd[2 * hh], wd[2 * hh + 1], 0x5410);
              const uint32_t y = __byte_perm(wd[2 * hh], wd[2 * hh + 1], 0x7632);
              b[hh][0] = H::dequant(nib<T, 0>(x), s2, z2);
              b[hh][1] = H::dequant(nib<T, 1>(x), s2, z2);
              b[hh][2] = H::dequant(nib<T, 2>(x), s2, z2);
              b[hh][3] = H::dequant(nib<T, 3>(x), s2, z2);
              b[hh][4] = H::dequant(nib<T, 0>(y), s2, z2);
              b[hh][5] = H::dequant(nib<T, 1>(y), s2, z2);
              b[hh][6] = H::dequant(nib<T, 2>(y), s2, z2);
              b[hh][7] = H::dequant(nib<T, 3>(y), s2, z2);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) H::mma(O[mt][wv * 8 + e], P[mt][k2], b[0][e], b[1][e]);
          }
        }
      }
      __syncwarp();
    }
    cp_wait<0>();

    // ---- join the four warps
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) l[mt][h] += __shfl_xor_sync(0xffffffffu, l[mt][h], o);
        if (c4 == 0) s_ml[warp * R + mt * 16 + r4 + h * 8] = make_float2(m[mt][h], l[mt][h]);
      }
    __syncthreads();  // the (m, l) pairs; and every warp is done with its ring
    float* merge = reinterpret_cast<float*>(body);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = mt * 16 + r4 + h * 8;
        float top = kNegInf;
#pragma unroll
        for (int w2 = 0; w2 < 4; ++w2) top = fmaxf(top, s_ml[w2 * R + r].x);
        // a warp whose keys this row does not see has a maximum of -inf and an output of 0
        const float f = m[mt][h] == kNegInf ? 1.f : exp2_fast(m[mt][h] - top);
        float* dst = merge + (warp * R + r) * C::OP;
#pragma unroll
        for (int t2 = 0; t2 < 2 * KT; ++t2) {
          if constexpr (!BITS4) {
            *reinterpret_cast<float2*>(dst + t2 * 8 + 2 * c4) = make_float2(O[mt][t2][2 * h] * f, O[mt][t2][2 * h + 1] * f);
          } else {
            dst[2 * c4 * (D / 8) + t2] = O[mt][t2][2 * h] * f;
            dst[(2 * c4 + 1) * (D / 8) + t2] = O[mt][t2][2 * h + 1] * f;
          }
        }
      }
    __syncthreads();
    const bool whole = k.slot < 0;
    const long long slot = k.slot;
    for (int i = tid; i < R * (D / 8); i += 128) {
      const int r = i % R, d = (i / R) * 8;  // (rows innermost: so are the partial results')
      if (!row_ok(r)) continue;
      float top = kNegInf, sum = 0.f;
#pragma unroll
      for (int w2 = 0; w2 < 4; ++w2) top = fmaxf(top, s_ml[w2 * R + r].x);
#pragma unroll
      for (int w2 = 0; w2 < 4; ++w2) {
        const float2 ml = s_ml[w2 * R + r];
        // (a sum of NaN scores keeps its NaN also under a maximum of -inf)
        sum += ml.x == kNegInf ? ml.y : ml.y * exp2_fast(ml.x - top);
      }
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = 0.f;
#pragma unroll
      for (int w2 = 0; w2 < 4; ++w2) {
        const float4* p = reinterpret_cast<const float4*>(merge + (w2 * R + r) * C::OP + d);
        const float4 x = p[0], y = p[1];
        o[0] += x.x; o[1] += x.y; o[2] += x.z; o[3] += x.w;
        o[4] += y.x; o[5] += y.y; o[6] += y.z; o[7] += y.w;
      }
      if (whole) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const long long tok = cur.s.s0 + tok0 + r / a.gs;
        const int head = kvh * a.g + sub * a.gs + r % a.gs;
        uint4 v;
        v.x = H::pack(o[0] * inv, o[1] * inv);
        v.y = H::pack(o[2] * inv, o[3] * inv);
        v.z = H::pack(o[4] * inv, o[5] * inv);
        v.w = H::pack(o[6] * inv, o[7] * inv);
        *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + tok * a.o_ts + head * a.o_hs + d) = v;
        if (d == 0 && a.lse != nullptr)
          a.lse[tok * (static_cast<long long>(a.c.Hkv) * a.g) + head] = sum == 0.f ? kNegInf : (top + log2f(sum)) * kLn2;
      } else {
        float* p = a.part_o + (slot * D + d) * R + r;
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e * R] = o[e];
        if (d == 0) *reinterpret_cast<float2*>(a.part_ml + (slot * R + r) * 2) = make_float2(top, sum);
      }
    }
    if (k.final || !work_next<BK>(a, W, cta, gridDim.x, k)) {
      if (tid == 0) leave_record(a, cta, k);
      break;
    }
    __syncthreads();  // the merge buffer is the next segment's ring
  }
}

// Joins the parts of the segments that were cut: CTA c takes the segment that its record names, a
// thread one row and 16 dims of it (rows along the lanes, as the parts lie), the parts in the order
// of their CTAs.
template <int D, typename T>
__global__ void __launch_bounds__(128) paged_join_kernel(const __grid_constant__ AttnArgs a, int R) {
  using H = Half2<T>;
  constexpr int CW = 16;  // dims of a thread
  pdl_wait_prior_grids();
  pdl_launch_dependents();
  const int c = blockIdx.x;
  const JoinRecord rec = a.records[c];
  if (rec.last < 0) return;
  const int last = rec.last, i = blockIdx.y * 128 + threadIdx.x;
  const int r = i % R, d = (i / R) * CW;
  if (r >= rec.rows || r % a.gs >= rec.heads || d >= D) return;
  const long long first = rec.slot;
  float top = kNegInf, sum = 0.f;
#pragma unroll 8
  for (int p = c; p <= last; ++p) top = fmaxf(top, a.part_ml[((p == c ? first : 2ll * p) * R + r) * 2]);
  float acc[CW];
#pragma unroll
  for (int e = 0; e < CW; ++e) acc[e] = 0.f;
#pragma unroll 2
  for (int p = c; p <= last; ++p) {
    const long long at = p == c ? first : 2ll * p;
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + (at * R + r) * 2);
    const float* o = a.part_o + (at * D + d) * R + r;
    float v[CW];
#pragma unroll
    for (int e = 0; e < CW; ++e) v[e] = o[e * R];
    const float f = ml.x == kNegInf ? 1.f : exp2_fast(ml.x - top);
    sum = fmaf(ml.y, f, sum);
#pragma unroll
    for (int e = 0; e < CW; ++e) acc[e] = fmaf(v[e], f, acc[e]);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const long long tok = rec.tok + r / a.gs;
  const int head = rec.head + r % a.gs;
  uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + tok * a.o_ts + head * a.o_hs + d);
#pragma unroll
  for (int e = 0; e < CW / 8; ++e) {
    uint4 v;
    v.x = H::pack(acc[8 * e] * inv, acc[8 * e + 1] * inv);
    v.y = H::pack(acc[8 * e + 2] * inv, acc[8 * e + 3] * inv);
    v.z = H::pack(acc[8 * e + 4] * inv, acc[8 * e + 5] * inv);
    v.w = H::pack(acc[8 * e + 6] * inv, acc[8 * e + 7] * inv);
    dst[e] = v;
  }
  if (d == 0 && a.lse != nullptr)
    a.lse[tok * (static_cast<long long>(a.c.Hkv) * a.g) + head] = sum == 0.f ? kNegInf : (top + log2f(sum)) * kLn2;
}

struct Variant {
  const void* fn;
  int smem, ctas;
};

template <int D, int MT, bool BITS4, typename T>
Variant variant() {
  using C = MmaCfg<D, MT, BITS4>;
  return {reinterpret_cast<const void*>(paged_attn_mma_kernel<D, MT, BITS4, T>), C::SMEM,
          (C::CTAS > 2 && MT == 2) ? 2 : C::CTAS};
}
template <int D, bool BITS4, typename T>
Variant by_rows(int rows) {
  if constexpr (D <= 128) {
    if (rows > 16) return variant<D, 2, BITS4, T>();
  }
  return variant<D, 1, BITS4, T>();
}
template <typename T>
Variant by_size(int D, int rows, bool bits4) {
  if (D == 64) return bits4 ? by_rows<64, true, T>(rows) : by_rows<64, false, T>(rows);
  if (D == 128) return bits4 ? by_rows<128, true, T>(rows) : by_rows<128, false, T>(rows);
  return bits4 ? by_rows<256, true, T>(rows) : by_rows<256, false, T>(rows);
}

std::atomic<int> g_smem_seen[24][64];

}  // namespace

// 32 rows where a sequence brings more than 16 on average (each key fragment then serves twice the
// rows); heads of 256 keep to 16, whose outputs already fill the registers.
AttnPlan plan_attn_mma(int N, int B, int g, int D, bool bits4, int sms) {
  AttnPlan p;
  const long long rows = (static_cast<long long>(N) * g + B - 1) / B;
  p.rows = rows > 16 && D <= 128 ? 32 : 16;
  p.grid = sms * by_size<__half>(D, p.rows, bits4).ctas;
  p.min_tiles = 2;
  p.seg_cost = 4;
  return p;
}

cudaError_t launch_attn_mma(AttnArgs a, const AttnPlan& p, int D, bool bf16, bool bits4, cudaStream_t stream, bool pdl) {
  const Variant v = bf16 ? by_size<__nv_bfloat16>(D, p.rows, bits4) : by_size<__half>(D, p.rows, bits4);
  const int idx = (((D == 64 ? 0 : D == 128 ? 1 : 2) * 2 + (p.rows == 32)) * 2 + bits4) * 2 + bf16;
  cudaError_t err = ensure_dyn_smem(v.fn, v.smem, g_smem_seen[idx], 64);
  if (err != cudaSuccess) return err;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.grid);
  cfg.blockDim = dim3(128);
  cfg.dynamicSmemBytes = v.smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  void* params[] = {&a};
  err = cudaLaunchKernelExC(&cfg, v.fn, params);
  if (err != cudaSuccess) return err;
  return launch_attn_join(a, p, D, bf16, stream, pdl);
}

cudaError_t launch_attn_join(const AttnArgs& a, const AttnPlan& p, int D, bool bf16, cudaStream_t stream, bool pdl) {
  const void* fn;
  if (D == 64)
    fn = bf16 ? reinterpret_cast<const void*>(paged_join_kernel<64, __nv_bfloat16>)
              : reinterpret_cast<const void*>(paged_join_kernel<64, __half>);
  else if (D == 128)
    fn = bf16 ? reinterpret_cast<const void*>(paged_join_kernel<128, __nv_bfloat16>)
              : reinterpret_cast<const void*>(paged_join_kernel<128, __half>);
  else
    fn = bf16 ? reinterpret_cast<const void*>(paged_join_kernel<256, __nv_bfloat16>)
              : reinterpret_cast<const void*>(paged_join_kernel<256, __half>);
  int R = p.rows;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.grid, (R * (D / 16) + 127) / 128);
  cfg.blockDim = dim3(128);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  void* params[] = {const_cast<AttnArgs*>(&a), &R};
  return cudaLaunchKernelExC(&cfg, fn, params);
}

}  // namespace smb

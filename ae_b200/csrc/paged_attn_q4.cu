// Attention of up to 8 query rows of a key head (decode: one token of up to 8 query heads) over a
// paged 4-bit cache.
//
// Bound by instructions: a byte of cache holds two values, each of which has to be unpacked, and at
// 8 rows there is nothing to share that over.  So the products are turned round, S^T = K Q^T and
// O^T = V^T P^T: the keys and the dims are the 16 rows of an m16n8k16 product and the query rows its 8
// columns, so no half of a product is padding, the output takes half the registers (three CTAs to
// an SM) and the scales and exponentials are worked on for the rows that exist.  P^T comes from S^T by
// transposing 8 x 8 blocks in registers (movmatrix).  Measured: 32 sequences of up to 32768 keys, one
// token, 32 / 8 heads of 128: 865 MB in 269 us, 3.2 TB/s (330 us with the query rows as the 16; rings of
// 2 / 3 / 4 stages 276 / 268 / 267 us); the integer pipe, which unpacks the codes, is 56 % busy, the issue
// slots 57 %.  The rest is as in the kernel for more rows: a warp streams keys of its own through its own
// ring, scores see no rounding of the keys (scales and zeros are applied to each group's product in 32
// bits), values are rounded once to the 16-bit type.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "paged_math.cuh"
#include "paged_plan.cuh"

namespace smb {
namespace {

template <int D>
struct Q4Cfg {
  static constexpr int R = 8;
  static constexpr int KS = 32;          // keys of a warp's stage
  static constexpr int BK = 4 * KS;      // keys of a CTA's tile
  static constexpr int ROW = kv4_row_bytes(D);
  static constexpr int NST = 3;
  static constexpr int STAGE = 2 * KS * ROW;
  static constexpr int RING = 4 * NST * STAGE;
  static constexpr int OP = D + 4;       // floats of a row of the merge buffer
  static constexpr int MERGE = 4 * R * OP * 4;
  static constexpr int BODY = RING > MERGE ? RING : MERGE;
  static constexpr int SMEM = BODY + 4 * R * 8 + 128;
  static constexpr int FIT = SMEM <= 54 * 1024 ? 4 : SMEM <= 73 * 1024 ? 3 : SMEM <= 111 * 1024 ? 2 : 1;
  static constexpr int CTAS = D == 256 ? std::min(FIT, 2) : FIT;
};

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

template <int D, typename T>
__global__ void __launch_bounds__(128, Q4Cfg<D>::CTAS) paged_attn_q4_kernel(const __grid_constant__ AttnArgs a) {
  using C = Q4Cfg<D>;
  using H = Half2<T>;
  constexpr int R = C::R, KS = C::KS, BK = C::BK, ROW = C::ROW, NST = C::NST;
  constexpr int CH = ROW / 16, G = D / 32, MTD = D / 16, WD = D / 64;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ PlanShared s_plan;
  __shared__ uint32_t s_ok[4][NST];
  uint8_t* body = smem;
  float2* s_ml = reinterpret_cast<float2*>(smem + C::BODY);
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
    const int prefix = cur.s.L - cur.s.n;
    auto row_ok = [&](int r) { return r < toks * a.gs && r % a.gs < heads; };
    auto sees = [&](int r, int j) {  // row r of the tile, key j < L
      const int i = tok0 + r / a.gs, lj = j - prefix;
      if (a.tree == nullptr) return lj <= i;
      if (lj < 0) return true;
      if ((lj >> 5) >= a.tree_words) return false;
      return ((static_cast<uint32_t>(a.tree[(cur.s.s0 + i) * a.tree_stride + (lj >> 5)]) >> (lj & 31)) & 1u) != 0;
    };

    // ---- loads of the first stages, then the queries
    const uint8_t* kbase = a.c.k + kvh * a.c.head_stride;
    const uint8_t* vbase = a.c.v + kvh * a.c.head_stride;
    const int* table = a.table + cur.b * a.table_stride;
    const int page_mask = (1 << a.c.page_shift) - 1;
    auto look_up = [&](int t) {  // page of this lane's key of tile t (one tile ahead of its loads)
      const int j = t * BK + warp * KS + lane;
      return (t < t1 && j < cur.keys) ? table[j >> a.c.page_shift] : -1;
    };
    int page = look_up(t0);
    auto issue = [&](int t) {
      if (t < t1) {
        const int st = (t - t0) % NST;
        const int j = t * BK + warp * KS + lane;
        const bool in = j < cur.keys;
        const bool ok = in && page >= 0 && page < a.c.num_pages;
        if (in && !ok) record_status(a.status, kDevBadPage);
        const long long off = ok ? page * a.c.page_stride + (j & page_mask) * a.c.token_stride : 0;
        const uint32_t okm = __ballot_sync(0xffffffffu, ok);
        if (lane == 0) s_ok[warp][st] = okm;
        page = look_up(t + 1);
        const uint32_t dst = ring_s + st * C::STAGE;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          const int idx = i * 32 + lane, key = idx / CH, ch = idx % CH;
          const long long o = __shfl_sync(0xffffffffu, off, key) + ch * 16;
          const bool fill = (okm >> key) & 1u;
          cp_async16(dst + key * ROW + ch * 16, kbase + o, fill);
          cp_async16(dst + KS * ROW + key * ROW + ch * 16, vbase + o, fill);
        }
      }
      cp_commit();
    };
#pragma unroll
    for (int s = 0; s < NST - 1; ++s) issue(t0 + s);

    // thread (r4, c4): row r4, dims 8 c4 + (0..7) of each group, in pairs (e, e + 4) as the nibbles come
    uint32_t q[G][4];
    float qs[G][2];  // the groups' sums of rows 2 c4 and 2 c4 + 1
#pragma unroll
    for (int g = 0; g < G; ++g) {
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (row_ok(r4)) {
        const T* p = static_cast<const T*>(a.q) + (cur.s.s0 + tok0 + r4 / a.gs) * a.q_ts +
                     (kvh * a.g + sub * a.gs + r4 % a.gs) * a.q_hs + g * 32 + c4 * 8;
        v = *reinterpret_cast<const uint4*>(p);
      }
      q[g][0] = __byte_perm(v.x, v.z, 0x5410);
      q[g][1] = __byte_perm(v.x, v.z, 0x7632);
      q[g][2] = __byte_perm(v.y, v.w, 0x5410);
      q[g][3] = __byte_perm(v.y, v.w, 0x7632);
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) s += H::lo(q[g][e]) + H::hi(q[g][e]);
      s += __shfl_xor_sync(0xffffffffu, s, 1);
      s += __shfl_xor_sync(0xffffffffu, s, 2);
      qs[g][0] = __shfl_sync(0xffffffffu, s, 8 * c4);
      qs[g][1] = __shfl_sync(0xffffffffu, s, 8 * c4 + 4);
    }

    float O[MTD][4];
    float m[2] = {kNegInf, kNegInf}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int t = 0; t < MTD; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) O[t][e] = 0.f;
    // dim of O[t][e] (e / 2: which of the two rows of the product)
    auto dim_of = [&](int t, int e) { return r4 * (D / 8) + (t >> 2) * 8 + (t & 3) + (e >> 1) * 4; };

#pragma unroll 1
    for (int t = t0; t < t1; ++t) {
      cp_wait<NST - 2>();
      __syncwarp();
      issue(t + NST - 1);
      const int st = (t - t0) % NST;
      uint8_t* ks = ring + st * C::STAGE;
      uint8_t* vs = ks + KS * ROW;
      const int j0 = t * BK + warp * KS;
      const uint32_t okm = s_ok[warp][st];
      const int open = a.tree != nullptr ? prefix : prefix + tok0 + 1;  // first key some row may not see
      const bool masked = okm != 0xffffffffu || j0 + KS > open;

      float S[2][4];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const uint8_t* row0 = ks + (kb * 16 + r4) * ROW;
        const uint8_t* row1 = row0 + 8 * ROW;
        uint32_t z0[G], z1[G];
        if constexpr (G == 2) {
          const uint2 x = *reinterpret_cast<const uint2*>(row0 + D / 2), y = *reinterpret_cast<const uint2*>(row1 + D / 2);
          z0[0] = x.x, z0[1] = x.y, z1[0] = y.x, z1[1] = y.y;
        } else {
#pragma unroll
          for (int i = 0; i < G / 4; ++i) {
            const uint4 x = *reinterpret_cast<const uint4*>(row0 + D / 2 + i * 16);
            const uint4 y = *reinterpret_cast<const uint4*>(row1 + D / 2 + i * 16);
            z0[4 * i] = x.x, z0[4 * i + 1] = x.y, z0[4 * i + 2] = x.z, z0[4 * i + 3] = x.w;
            z1[4 * i] = y.x, z1[4 * i + 1] = y.y, z1[4 * i + 2] = y.z, z1[4 * i + 3] = y.w;
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) S[kb][e] = 0.f;
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const uint32_t w0 = *reinterpret_cast<const uint32_t*>(row0 + g * 16 + c4 * 4);
          const uint32_t w1 = *reinterpret_cast<const uint32_t*>(row1 + g * 16 + c4 * 4);
          float acc[4] = {0.f, 0.f, 0.f, 0.f};
          const uint32_t f0[4] = {nib<T, 0>(w0), nib<T, 0>(w1), nib<T, 1>(w0), nib<T, 1>(w1)};
          H::mma(acc, f0, q[g][0], q[g][1]);
          const uint32_t f1[4] = {nib<T, 2>(w0), nib<T, 2>(w1), nib<T, 3>(w0), nib<T, 3>(w1)};
          H::mma(acc, f1, q[g][2], q[g][3]);
          const float s0 = H::lo(z0[g]), s1 = H::lo(z1[g]);
          const float o0 = fmaf(-16.f, s0, H::hi(z0[g])), o1 = fmaf(-16.f, s1, H::hi(z1[g]));
          S[kb][0] = fmaf(s0, acc[0], fmaf(o0, qs[g][0], S[kb][0]));
          S[kb][1] = fmaf(s0, acc[1], fmaf(o0, qs[g][1], S[kb][1]));
          S[kb][2] = fmaf(s1, acc[2], fmaf(o1, qs[g][0], S[kb][2]));
          S[kb][3] = fmaf(s1, acc[3], fmaf(o1, qs[g][1], S[kb][3]));
        }
      }

      if (masked) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int kl = kb * 16 + r4 + (e >> 1) * 8, r = 2 * c4 + (e & 1);
            if (!((okm >> kl) & 1u) || !row_ok(r) || !sees(r, j0 + kl)) S[kb][e] = kNegInf;
            else S[kb][e] *= a.scale_log2;
          }
        // non-finite values behind the mask: to the rows that see them directly, out of the product
        bool bad = false;
        for (int i = lane; i < KS * G; i += 32) {
          bad = bad || group_overflows<T>(*reinterpret_cast<const uint32_t*>(vs + (i / G) * ROW + D / 2 + (i % G) * 4));
        }
        if (__any_sync(0xffffffffu, bad)) {
          for (int kl = 0; kl < KS; ++kl) {
            if (!((okm >> kl) & 1u)) continue;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int r = 2 * c4 + h;
              if (!row_ok(r) || !sees(r, j0 + kl)) continue;
#pragma unroll
              for (int t2 = 0; t2 < MTD; ++t2)
#pragma unroll
                for (int e = h; e < 4; e += 2) {
                  const int d = dim_of(t2, e);
                  const uint32_t sz = *reinterpret_cast<const uint32_t*>(vs + kl * ROW + D / 2 + (d >> 5) * 4);
                  const float v = H::lo(value_of<T>((vs[kl * ROW + (d >> 1)] >> (4 * (d & 1))) & 15u, sz));
                  if (!isfinite(v)) O[t2][e] += v;
                }
            }
          }
          __syncwarp();
          for (int i = lane; i < KS * G; i += 32) {
            uint8_t* row = vs + (i / G) * ROW;
            uint32_t* sz = reinterpret_cast<uint32_t*>(row + D / 2 + (i % G) * 4);
            if (group_overflows<T>(*sz)) take_out_nonfinite<T>(reinterpret_cast<uint32_t*>(row + (i % G) * 16), sz);
          }
          __syncwarp();
        }
      } else {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int e = 0; e < 4; ++e) S[kb][e] *= a.scale_log2;
      }

      // running maximum (paged_math.cuh)
      float top[2];
      bool grew = false;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        top[h] = fmaxf(fmaxf(S[0][h], S[0][2 + h]), fmaxf(S[1][h], S[1][2 + h]));
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], o));
        grew = grew || top[h] > m[h] + (kGrow + H::kLift);
      }
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float now = fmaxf(m[h], top[h] - H::kLift);
          const float f = m[h] == kNegInf ? 0.f : exp2_fast(m[h] - now);
          m[h] = now;
          l[h] *= f;
#pragma unroll
          for (int t2 = 0; t2 < MTD; ++t2)
#pragma unroll
            for (int e = h; e < 4; e += 2)
              if (f != 0.f || isfinite(O[t2][e])) O[t2][e] *= f;
        }
      }
      uint32_t P[2][2];  // P^T of 16 keys: rows r4, keys 2 c4 and 2 c4 + 1, then those 8 on
      {
        const float m0 = m[0] == kNegInf ? 0.f : m[0], m1 = m[1] == kNegInf ? 0.f : m[1];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float p0 = exp2_fast(S[kb][2 * i] - m0), p1 = exp2_fast(S[kb][2 * i + 1] - m1);
            l[0] += p0;
            l[1] += p1;
            P[kb][i] = transpose8x8(H::pack(p0, p1));
          }
      }

#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const uint8_t* row[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) row[e] = vs + (kb * 16 + 2 * c4 + (e & 1) + (e >> 1) * 8) * ROW;
#pragma unroll
        for (int wv = 0; wv < WD; ++wv) {
          const int word = r4 * WD + wv;
          uint32_t x[2], y[2], s2[2], z2[2];
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            const uint32_t wa = *reinterpret_cast<const uint32_t*>(row[2 * hh] + word * 4);
            const uint32_t wb = *reinterpret_cast<const uint32_t*>(row[2 * hh + 1] + word * 4);
            const uint32_t za = *reinterpret_cast<const uint32_t*>(row[2 * hh] + D / 2 + (word >> 2) * 4);
            const uint32_t zb = *reinterpret_cast<const uint32_t*>(row[2 * hh + 1] + D / 2 + (word >> 2) * 4);
            x[hh] = __byte_perm(wa, wb, 0x5410);
            y[hh] = __byte_perm(wa, wb, 0x7632);
            s2[hh] = __byte_perm(za, zb, 0x5410);
            z2[hh] = __byte_perm(za, zb, 0x7632);
          }
          auto product = [&](auto nibble) {
            constexpr int E = decltype(nibble)::value;
            const uint32_t f[4] = {H::dequant(nib<T, E>(x[0]), s2[0], z2[0]), H::dequant(nib<T, E>(y[0]), s2[0], z2[0]),
                                   H::dequant(nib<T, E>(x[1]), s2[1], z2[1]), H::dequant(nib<T, E>(y[1]), s2[1], z2[1])};
            H::mma(O[wv * 4 + E], f, P[kb][0], P[kb][1]);
          };
          product(std::integral_constant<int, 0>{});
          product(std::integral_constant<int, 1>{});
          product(std::integral_constant<int, 2>{});
          product(std::integral_constant<int, 3>{});
        }
      }
      __syncwarp();
    }
    cp_wait<0>();

    // ---- join the four warps
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], o);
      if (r4 == 0) s_ml[warp * R + 2 * c4 + h] = make_float2(m[h], l[h]);
    }
    __syncthreads();  // the (m, l) pairs; and every warp is done with its ring
    float* merge = reinterpret_cast<float*>(body);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = 2 * c4 + h;
      float top = kNegInf;
#pragma unroll
      for (int w2 = 0; w2 < 4; ++w2) top = fmaxf(top, s_ml[w2 * R + r].x);
      const float f = m[h] == kNegInf ? 1.f : exp2_fast(m[h] - top);  // (no visible key: an output of 0)
      float* dst = merge + (warp * R + r) * C::OP;
#pragma unroll
      for (int t2 = 0; t2 < MTD; ++t2)
#pragma unroll
        for (int e = h; e < 4; e += 2) dst[dim_of(t2, e)] = O[t2][e] * f;
    }
    __syncthreads();
    const bool whole = k.slot < 0;
    const long long slot = k.slot;
    for (int i = tid; i < R * (D / 8); i += 128) {
      const int r = i % R, d = (i / R) * 8;
      if (!row_ok(r)) continue;
      float top = kNegInf, sum = 0.f;
#pragma unroll
      for (int w2 = 0; w2 < 4; ++w2) top = fmaxf(top, s_ml[w2 * R + r].x);
#pragma unroll
      for (int w2 = 0; w2 < 4; ++w2) {
        const float2 ml = s_ml[w2 * R + r];
        sum += ml.x == kNegInf ? ml.y : ml.y * exp2_fast(ml.x - top);
      }
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = 0.f;
#pragma unroll
      for (int w2 = 0; w2 < 4; ++w2)
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] += merge[(w2 * R + r) * C::OP + d + e];
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

struct Variant {
  const void* fn;
  int smem, ctas;
};
template <typename T>
Variant variant(int D) {
  if (D == 64) return {reinterpret_cast<const void*>(paged_attn_q4_kernel<64, T>), Q4Cfg<64>::SMEM, Q4Cfg<64>::CTAS};
  if (D == 128) return {reinterpret_cast<const void*>(paged_attn_q4_kernel<128, T>), Q4Cfg<128>::SMEM, Q4Cfg<128>::CTAS};
  return {reinterpret_cast<const void*>(paged_attn_q4_kernel<256, T>), Q4Cfg<256>::SMEM, Q4Cfg<256>::CTAS};
}

std::atomic<int> g_smem_seen[6][64];

}  // namespace

bool plan_attn_q4(int N, int B, int g, int D, int sms, AttnPlan* p) {
  const long long rows = (static_cast<long long>(N) * g + B - 1) / B;
  if (rows > 8) return false;
  p->rows = 8;
  p->grid = sms * variant<__half>(D).ctas;
  p->min_tiles = 2;
  p->seg_cost = 4;
  return true;
}

cudaError_t launch_attn_q4(AttnArgs a, const AttnPlan& p, int D, bool bf16, cudaStream_t stream, bool pdl) {
  const Variant v = bf16 ? variant<__nv_bfloat16>(D) : variant<__half>(D);
  cudaError_t err = ensure_dyn_smem(v.fn, v.smem, g_smem_seen[(D == 64 ? 0 : D == 128 ? 1 : 2) * 2 + bf16], 64);
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

}  // namespace smb

// Append to a paged cache: RMS norm of each query and key head (optional), rotary positions and
// the write of keys and values into their cache rows, in one pass over the projection's output.
//
//   x <- x * rsqrt(mean(x^2) + eps) * w,   angle_i = position * inv_freq_i,
//   (a, b) -> (a cos - b sin, b cos + a sin)   for the pairs (i, i + rot/2) or (2i, 2i + 1).
//
// Positions reach far beyond what a 32-bit product resolves (at position 10^6 its error is 0.06 rad),
// so the angle is formed in 64 bits, as a fraction of a turn, and only that fraction goes to
// sincospi in 32 bits (error below 2^-23 of a turn).  Everything between the load and the store is in
// 32 bits; one rounding at the store.
//
// Bound by memory when there are many tokens, and close to it by instructions, so the arithmetic of a
// row is kept to out = (A x + B x') rstd with x' the other half of each pair: A and B (rotation times
// norm weight, with the sign of the half) are the same for all heads of a token and stay in
// registers.  A warp takes a token, or a part of its rows when there are few tokens; rows pass through
// a ring of its own in shared memory, filled ahead by cp.async, from which a lane reads its 16 bytes
// and the 16 bytes with the other halves.  Warps share nothing, so nothing waits at a barrier.
//
// Measured: 8199 tokens, 32 / 8 heads of 128 with norms: 202 MB in 41 us, 4.9 TB/s (0.75 of the measured
// copy rate; issue slots 75 % busy).
//
// A 4-bit row keeps, for each 32 values, zero = rn(min), scale = rn((max - min) / 15) in the
// 16-bit type (rounded down if 15 scale + zero would overflow it: 0 to 65504 in fp16) and codes
// rint((x - zero) / scale) in [0, 15]; the codes are formed with the rounded scale and zero, so their
// rounding is not added to the codes' own.  A group with a NaN has both NaN, one with an infinity an
// infinite scale and codes of 0: either way it reads as NaN.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "paged.h"
#include "paged_math.cuh"

namespace smb {
namespace {

template <typename T>
struct Pack8 {
  union {
    uint4 u;
    T t[8];
  };
};

// Two 16-bit values of a word as a pair of 32-bit ones.
template <typename T>
__device__ __forceinline__ uint64_t wide(uint32_t v) {
  return pair(Half2<T>::lo(v), Half2<T>::hi(v));
}
__device__ __forceinline__ uint4 swap_pairs(uint4 v) {
  return make_uint4(__byte_perm(v.x, 0, 0x1032), __byte_perm(v.y, 0, 0x1032), __byte_perm(v.z, 0, 0x1032),
                    __byte_perm(v.w, 0, 0x1032));
}

// Minimum and maximum that are NaN if one of the two is.
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The (scale, zero) of a 4-bit group whose smallest and largest values are mn and mx, with the scale taken down
// where needed for code 15 to stay finite; as it is where mx or the zero does not fit the type.
template <typename T>
__device__ __forceinline__ uint32_t fit_scale(uint32_t sz, float mn, float mx) {
  using H = Half2<T>;
  if (H::nonfinite(H::pack(mx, 0.f) & 0xffffu) || H::nonfinite(sz >> 16)) return sz;
  const uint32_t zero = sz & 0xffff0000u;
  if (H::nonfinite(sz & 0xffffu)) sz = zero | (H::pack(mx / 15.f - mn / 15.f, 0.f) & 0xffffu);  // (the span itself did)
  if (group_overflows<T>(sz)) sz = zero | H::towards_zero(H::kMost / 15.f - H::hi(zero) / 15.f);
  return sz;
}

constexpr int kAppendWarps = 4;   // of a CTA
constexpr int kAppendStages = 8;  // steps of the ring: 7 x 512 bytes in flight per warp

// `parts` warps share a token.
template <int D, typename T, bool BITS4, bool NORM>
__global__ void __launch_bounds__(32 * kAppendWarps, 8) kv_append_kernel(const __grid_constant__ AppendArgs a, int parts) {
  constexpr int LPR = D / 8;        // lanes per row
  constexpr int RPS = 32 / LPR;     // rows per step
  constexpr unsigned kAll = 0xffffffffu;
  __shared__ __align__(16) uint4 s_ring[kAppendWarps][kAppendStages][32];
  __shared__ float2 s_angles[kAppendWarps][D / 2];
  pdl_wait_prior_grids();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int lane8 = lane % LPR, rsub = lane / LPR;
  const int Hkv = a.c.Hkv;
  const unsigned unit = blockIdx.x * kAppendWarps + warp;  // (below 2^31)
  const unsigned token = unit / parts;
  if (token >= a.N) return;
  const long long tok = token;
  const int part = static_cast<int>(unit - token * parts);
  // this warp's steps of the token's queries, keys and values
  const int sq = (a.Hq + RPS - 1) / RPS, sk = (Hkv + RPS - 1) / RPS, all = sq + 2 * sk;
  const int step_lo = all * part / parts, step_hi = all * (part + 1) / parts;

  const int nq = max(0, min(step_hi, sq) - step_lo);
  const int k_lo = max(step_lo - sq, 0), nk = max(0, min(step_hi - sq, sk) - k_lo);
  const int v_lo = max(step_lo - sq - sk, 0), nv = max(0, step_hi - sq - sk - v_lo);

  // loads run ahead of the rows' arithmetic, through the same three kinds
  uint4(*ring)[32] = s_ring[warp];
  const T* src;
  long long src_step;
  int src_rows, src_left, src_kind = 0, src_stage = 0;
  auto open_source = [&]() {
    const int first = (src_kind == 0 ? step_lo : src_kind == 1 ? k_lo : v_lo) * RPS + rsub;
    const long long hs = src_kind == 0 ? a.q_hs : src_kind == 1 ? a.k_hs : a.v_hs;
    src = static_cast<const T*>(src_kind == 0 ? a.q : src_kind == 1 ? a.k : a.v) +
          tok * (src_kind == 0 ? a.q_ts : src_kind == 1 ? a.k_ts : a.v_ts) + first * hs + lane8 * 8;
    src_step = hs * RPS;
    src_rows = (src_kind == 0 ? a.Hq : Hkv) - first;  // rows from this lane's on
    src_left = src_kind == 0 ? nq : src_kind == 1 ? nk : nv;
  };
  open_source();
  auto issue = [&]() {
    while (src_left == 0 && src_kind < 2) {
      ++src_kind;
      open_source();
    }
    if (src_left > 0) {
      if (src_rows > 0)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(&ring[src_stage][lane])), "l"(src) : "memory");
      src += src_step;
      src_rows -= RPS;
      --src_left;
      src_stage = (src_stage + 1) % kAppendStages;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kAppendStages - 1; ++i) issue();

  const long long slot = a.slots[tok];
  const int half = a.rot / 2;
  float2* s_cs = s_angles[warp];
  if (step_lo < sq + sk) {
    for (int i = lane; i < half; i += 32) {
      const double turns = static_cast<double>(a.positions[tok]) * a.inv_freq[i] * 0.15915494309189533577;
      float s, c;
      sincospif(2.0f * static_cast<float>(turns - rint(turns)), &s, &c);
      s_cs[i] = make_float2(c * a.rope_scale, s * a.rope_scale);
    }
  }
  const long long page = slot >> a.c.page_shift;
  const bool keep = slot >= 0 && page < a.c.num_pages;
  if (slot >= 0 && !keep && lane == 0) record_status(a.status, kDevBadPage);
  const long long cache_off =
      keep ? page * a.c.page_stride + (slot & ((1ll << a.c.page_shift) - 1)) * a.c.token_stride : 0;

  // the lane with the other half of this lane's pairs (half is a multiple of 8)
  const bool turn = lane8 * 8 < a.rot;
  const bool low = lane8 * 8 < half;
  const int from = turn && !a.interleaved ? (low ? lane8 + half / 8 : lane8 - half / 8) : lane8;

  uint64_t A[4], B[4];  // pairs of dims
  bool normed = false;
  auto coefficients = [&](const T* w) {
    normed = NORM && w != nullptr;
    uint4 wo = make_uint4(0u, 0u, 0u, 0u), wp = wo;
    if (normed) {
      wo = __ldg(reinterpret_cast<const uint4*>(w + lane8 * 8));
      wp = __ldg(reinterpret_cast<const uint4*>(w + from * 8));
      if (a.interleaved) wp = swap_pairs(wo);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float2 c0 = make_float2(1.f, 0.f), c1 = c0;
      if (turn) {
        const int at = a.interleaved ? lane8 * 4 + e : (low ? lane8 * 8 : lane8 * 8 - half) + 2 * e;
        c0 = s_cs[at];
        c1 = s_cs[a.interleaved ? at : at + 1];
        if (a.interleaved || low) c0.y = -c0.y;
        if (!a.interleaved && low) c1.y = -c1.y;
      }
      A[e] = pair(c0.x, c1.x);
      B[e] = pair(c0.y, c1.y);
      if (normed) {
        A[e] = mul2(A[e], wide<T>((&wo.x)[e]));
        B[e] = mul2(B[e], wide<T>((&wp.x)[e]));
      }
    }
  };

  int stage = 0;
  // `n` steps of one kind; rows [first, rows) go to dst, `dst_step` bytes a step apart
  auto run = [&](auto kind, int n, int first, int rows, uint8_t* dst, long long dst_step, bool store) {
    constexpr int K = decltype(kind)::value;
    int left = rows - first;  // rows from this lane's on
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kAppendStages - 2) : "memory");
      __syncwarp();
      issue();  // (into the stage that the last step left)
      const uint4* at = ring[stage];
      stage = (stage + 1) % kAppendStages;
      const bool there = store && left > 0;
      left -= RPS;
      uint4 o = at[lane];
      uint64_t f[4];
      if (K != 2 || BITS4) {
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = wide<T>((&o.x)[e]);
      }
      if (K != 2 && (half > 0 || normed)) {
        uint4 y = make_uint4(0u, 0u, 0u, 0u);  // (outside the rotated dims nothing of x' may come through)
        if (turn) {
          y = at[rsub * LPR + from];
          if (a.interleaved) y = swap_pairs(y);
        }
        uint64_t g[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) g[e] = fma2(A[e], f[e], mul2(B[e], wide<T>((&y.x)[e])));
        if (NORM && normed) {
          float s0, s1;
          unpair(fma2(f[3], f[3], fma2(f[2], f[2], fma2(f[1], f[1], mul2(f[0], f[0])))), s0, s1);
          float ss = s0 + s1;
#pragma unroll
          for (int s = LPR / 2; s > 0; s >>= 1) ss += __shfl_xor_sync(kAll, ss, s);
          const float rstd = rsqrtf(ss * (1.0f / D) + a.eps);
#pragma unroll
          for (int e = 0; e < 4; ++e) g[e] = mul2(g[e], pair(rstd, rstd));
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float lo, hi;
          f[e] = g[e];
          unpair(g[e], lo, hi);
          (&o.x)[e] = Half2<T>::pack(lo, hi);
        }
      }
      if (K == 0 || !BITS4) {
        if (there) *reinterpret_cast<uint4*>(dst + lane8 * 16) = o;
      } else {
        float v[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) unpair(f[e], v[2 * e], v[2 * e + 1]);
        float mn = v[0], mx = v[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) {
          mn = min_nan(mn, v[e]);
          mx = max_nan(mx, v[e]);
        }
#pragma unroll
        for (int s = 1; s < 4; s <<= 1) {
          mn = min_nan(mn, __shfl_xor_sync(kAll, mn, s));
          mx = max_nan(mx, __shfl_xor_sync(kAll, mx, s));
        }
        const float span = mx - mn;
        uint32_t sz = Half2<T>::pack(__fdiv_rn(span, 15.0f), mn);
        float scale = Half2<T>::lo(sz), zero = Half2<T>::hi(sz);
        // (below 0.98 of the largest number no rounding of scale and zero takes code 15 past it)
        if (fmaxf(mx, span) > 0.98f * Half2<T>::kMost) {
          sz = fit_scale<T>(sz, mn, mx);
          const float down = span > 3.3e38f ? 0.25f : 1.f;  // (v - zero may pass 32 bits: a quarter of everything)
          scale = Half2<T>::lo(sz) * down, zero = Half2<T>::hi(sz) * down;
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] *= down;
        }
        // (a group of one value, or with a scale below the type, has codes of 0)
        const float inv = scale > 0.f ? __frcp_rn(scale) : 0.f;
        uint32_t codes = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          // the quotient corrected by its remainder: values of 16 bits meet the middle between two codes
          // often, and a quotient off by a last place would round the wrong way there
          const float x = v[e] - zero, q = x * inv;
          // the code's integer in the low bits of 2^23 + code (round to nearest even); NaN gives 0
          const float c = fminf(fmaxf(fmaf(fmaf(-q, scale, x), inv, q), 0.f), 15.f) + 8388608.f;
          codes |= (__float_as_uint(c) & 15u) << (4 * e);
        }
        if (there) {
          *reinterpret_cast<uint32_t*>(dst + lane8 * 4) = codes;
          if ((lane8 & 3) == 0) *reinterpret_cast<uint32_t*>(dst + D / 2 + lane8) = sz;
        }
      }
      dst += dst_step;
      __syncwarp();
    }
  };
  __syncwarp();
  if (nq > 0) {
    coefficients(static_cast<const T*>(a.q_norm));
    const int first = step_lo * RPS + rsub;
    run(std::integral_constant<int, 0>{}, nq, first, a.Hq,
        reinterpret_cast<uint8_t*>(static_cast<T*>(a.q_out) + (tok * a.Hq + first) * D), RPS * D * 2, true);
  }
  if (nk > 0) {
    coefficients(static_cast<const T*>(a.k_norm));
    const int first = k_lo * RPS + rsub;
    run(std::integral_constant<int, 1>{}, nk, first, Hkv, a.c.k + cache_off + first * a.c.head_stride,
        RPS * a.c.head_stride, keep);
  }
  if (nv > 0) {
    const int first = v_lo * RPS + rsub;
    run(std::integral_constant<int, 2>{}, nv, first, Hkv, a.c.v + cache_off + first * a.c.head_stride,
        RPS * a.c.head_stride, keep);
  }
}

// Rows of a 4-bit cache as 16-bit values: a thread takes 8 codes of one row.  A negative slot,
// or one past the cache, reads as zeros.
template <int D, typename T>
__global__ void __launch_bounds__(256) kv4_read_kernel(const __grid_constant__ Kv4ReadArgs a) {
  constexpr int LPR = D / 8;
  pdl_wait_prior_grids();
  pdl_launch_dependents();
  const long long i = blockIdx.x * 256ll + threadIdx.x;
  const int lane8 = static_cast<int>(i % LPR);
  const long long row = i / LPR;
  if (row >= static_cast<long long>(a.M) * a.Hkv) return;
  const long long m = row / a.Hkv;
  const int h = static_cast<int>(row % a.Hkv);
  const long long slot = a.slots[m], page = slot >> a.page_shift;
  Pack8<T> o;
  o.u = make_uint4(0u, 0u, 0u, 0u);
  if (slot >= 0 && page < a.num_pages) {
    const uint8_t* p = a.cache + page * a.page_stride + (slot & ((1ll << a.page_shift) - 1)) * a.token_stride +
                       h * a.head_stride;
    const uint32_t codes = *reinterpret_cast<const uint32_t*>(p + lane8 * 4);
    const T* sz = reinterpret_cast<const T*>(p + D / 2 + (lane8 >> 2) * 4);
    const float s = to_f32<T>(sz[0]), z = to_f32<T>(sz[1]);
#pragma unroll
    for (int e = 0; e < 8; ++e) o.t[e] = from_f32<T>(fmaf(static_cast<float>((codes >> (4 * e)) & 15u), s, z));
  }
  *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + row * D + lane8 * 8) = o.u;
}

cudaError_t launch(const void* fn, dim3 grid, dim3 block, void** params, cudaStream_t stream, bool pdl) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  return cudaLaunchKernelExC(&cfg, fn, params);
}

template <int D, typename T>
const void* append_fn_t(bool bits4, bool norm) {
  if (bits4)
    return norm ? reinterpret_cast<const void*>(kv_append_kernel<D, T, true, true>)
                : reinterpret_cast<const void*>(kv_append_kernel<D, T, true, false>);
  return norm ? reinterpret_cast<const void*>(kv_append_kernel<D, T, false, true>)
              : reinterpret_cast<const void*>(kv_append_kernel<D, T, false, false>);
}
template <int D>
const void* append_fn(bool bf16, bool bits4, bool norm) {
  return bf16 ? append_fn_t<D, __nv_bfloat16>(bits4, norm) : append_fn_t<D, __half>(bits4, norm);
}

template <int D>
const void* read_fn(bool bf16) {
  return bf16 ? reinterpret_cast<const void*>(kv4_read_kernel<D, __nv_bfloat16>)
              : reinterpret_cast<const void*>(kv4_read_kernel<D, __half>);
}

}  // namespace

cudaError_t launch_kv_append(const AppendArgs& a, int D, bool bf16, bool bits4, int sms, cudaStream_t stream, bool pdl) {
  const bool norm = a.q_norm != nullptr || a.k_norm != nullptr;
  const void* fn = D == 64    ? append_fn<64>(bf16, bits4, norm)
                   : D == 128 ? append_fn<128>(bf16, bits4, norm)
                              : append_fn<256>(bf16, bits4, norm);
  // few tokens: several warps to a token, until the SMs' 32 warps are there or a warp has four steps
  const int rps = 256 / D, steps = (a.Hq + rps - 1) / rps + 2 * ((a.c.Hkv + rps - 1) / rps);
  int parts = static_cast<int>(std::min<long long>((32ll * sms + a.N - 1) / a.N, (steps + 3) / 4));
  void* params[] = {const_cast<AppendArgs*>(&a), &parts};
  const long long units = static_cast<long long>(a.N) * parts;
  return launch(fn, dim3(static_cast<unsigned>((units + kAppendWarps - 1) / kAppendWarps)), dim3(32 * kAppendWarps), params,
                stream, pdl);
}

cudaError_t launch_kv4_read(const Kv4ReadArgs& a, int D, bool bf16, cudaStream_t stream, bool pdl) {
  const void* fn = D == 64 ? read_fn<64>(bf16) : D == 128 ? read_fn<128>(bf16) : read_fn<256>(bf16);
  const long long threads = static_cast<long long>(a.M) * a.Hkv * (D / 8);
  void* params[] = {const_cast<Kv4ReadArgs*>(&a)};
  return launch(fn, dim3(static_cast<unsigned>((threads + 255) / 256)), dim3(256), params, stream, pdl);
}

}  // namespace smb

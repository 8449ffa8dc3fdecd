// Append to a paged cache: RMS norm of each query and key head (optional), rotary positions and
// the write of keys and values into their cache rows, in one pass over the projection's output.
//
//   x <- x * rsqrt(mean(x^2) + eps) * w,   angle_i = position * inv_freq_i,
//   (a, b) -> (a cos - b sin, b cos + a sin)   for the pairs (i, i + rot/2) or (2i, 2i + 1).
//
// A token's rotation is shared by its heads, so a CTA takes one token (or a slice of its heads
// when there are few tokens): the angles once into shared memory, then every row by D/8 lanes
// with 16-byte accesses.  Positions reach far beyond what a 32-bit product resolves (at
// position 10^6 its error is 0.06 rad), so the angle is formed in 64 bits, as a fraction of a
// turn, and only that fraction goes to sincospi in 32 bits (error below 2^-23 of a turn).
// Everything between the load and the store is in 32 bits; one rounding at the store.
//
// A 4-bit row keeps, for each 32 values, zero = rn(min), scale = rn((max - min) / 15) in the
// 16-bit type and codes rint((x - zero) / scale) in [0, 15]; the codes are formed with the
// rounded scale and zero, so their rounding is not added to the codes' own.
#include "common.cuh"
#include "kernels.h"
#include "paged.h"

namespace smb {
namespace {

template <typename T>
struct Pack8 {
  union {
    uint4 u;
    T t[8];
  };
};

template <int D, typename T, bool BITS4>
__global__ void __launch_bounds__(256) kv_append_kernel(const __grid_constant__ AppendArgs a) {
  constexpr int LPR = D / 8;        // lanes per row
  constexpr int RPP = 256 / LPR;    // rows per pass
  constexpr int UNROLL = 4;         // rows in flight per thread
  __shared__ float2 s_cs[D / 2];
  pdl_wait_prior_grids();
  pdl_launch_dependents();
  const int tok = blockIdx.x;
  const int lane8 = threadIdx.x % LPR, rsub = threadIdx.x / LPR;
  const int Hkv = a.c.Hkv, rows = a.Hq + 2 * Hkv;
  const int per = (rows + gridDim.y - 1) / gridDim.y;
  const int row_lo = blockIdx.y * per, row_hi = min(rows, row_lo + per);
  if (row_lo >= rows) return;

  const T* qb = static_cast<const T*>(a.q) + tok * a.q_ts + lane8 * 8;
  const T* kb = static_cast<const T*>(a.k) + tok * a.k_ts + lane8 * 8;
  const T* vb = static_cast<const T*>(a.v) + tok * a.v_ts + lane8 * 8;
  auto load = [&](int r, Pack8<T>& x) {
    x.u = make_uint4(0u, 0u, 0u, 0u);
    if (r < row_hi) {
      const T* p = r < a.Hq ? qb + r * a.q_hs : r < a.Hq + Hkv ? kb + (r - a.Hq) * a.k_hs : vb + (r - a.Hq - Hkv) * a.v_hs;
      x.u = __ldg(reinterpret_cast<const uint4*>(p));
    }
  };
  Pack8<T> x[UNROLL];
#pragma unroll
  for (int i = 0; i < UNROLL; ++i) load(row_lo + i * RPP + rsub, x[i]);

  const long long slot = a.slots[tok];
  const long long page = slot >> a.c.page_shift;
  const bool keep = slot >= 0 && page < a.c.num_pages;
  if (slot >= 0 && !keep && threadIdx.x == 0) record_status(a.status, kDevBadPage);
  const long long cache_off =
      keep ? page * a.c.page_stride + (slot & ((1ll << a.c.page_shift) - 1)) * a.c.token_stride : 0;

  const int half = a.rot / 2;
  for (int i = threadIdx.x; i < half; i += 256) {
    const double turns = static_cast<double>(a.positions[tok]) * a.inv_freq[i] * 0.15915494309189533577;
    float s, c;
    sincospif(2.0f * static_cast<float>(turns - rint(turns)), &s, &c);
    s_cs[i] = make_float2(c * a.rope_scale, s * a.rope_scale);
  }
  __syncthreads();

  const unsigned group_mask = 0xffffffffu;
  for (int r0 = row_lo; r0 < row_hi; r0 += UNROLL * RPP) {
    if (r0 != row_lo) {
#pragma unroll
      for (int i = 0; i < UNROLL; ++i) load(r0 + i * RPP + rsub, x[i]);
    }
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) {
      if (r0 + i * RPP >= row_hi) break;  // uniform over the CTA
      const int r = r0 + i * RPP + rsub;
      const bool there = r < row_hi;
      const bool is_q = r < a.Hq, is_v = r >= a.Hq + Hkv;
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = to_f32<T>(x[i].t[e]);
      const T* w = static_cast<const T*>(is_v ? nullptr : is_q ? a.q_norm : a.k_norm);
      // the shuffles run on every lane (a warp can hold rows of both kinds)
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(f[e], f[e], ss);
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(group_mask, ss, o);
      if (w != nullptr) {
        Pack8<T> wv;
        wv.u = __ldg(reinterpret_cast<const uint4*>(w + lane8 * 8));
        const float rstd = 1.0f / sqrtf(ss * (1.0f / D) + a.eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = f[e] * rstd * to_f32<T>(wv.t[e]);
      }
      if (half > 0) {
        const bool turn = lane8 * 8 < a.rot && !is_v;
        if (a.interleaved) {
          if (turn) {
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
              const float2 cs = s_cs[lane8 * 4 + e / 2];
              const float p = f[e], q = f[e + 1];
              f[e] = p * cs.x - q * cs.y;
              f[e + 1] = q * cs.x + p * cs.y;
            }
          }
        } else {
          // rot / 2 is a multiple of 8, so the pair of a lane's values is another lane's
          const int off = half / 8;
          const bool low = lane8 < off;
          const int from = turn ? (low ? lane8 + off : lane8 - off) : lane8;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float other = __shfl_sync(group_mask, f[e], from, LPR);
            if (turn) {
              const float2 cs = s_cs[(low ? lane8 : lane8 - off) * 8 + e];
              f[e] = low ? f[e] * cs.x - other * cs.y : f[e] * cs.x + other * cs.y;
            }
          }
        }
      }
      Pack8<T> o;
      if (w != nullptr || half > 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) o.t[e] = from_f32<T>(f[e]);
      } else {
        o = x[i];
      }
      if (is_v) o = x[i];
      if (is_q) {
        if (there) {
          T* dst = static_cast<T*>(a.q_out) + (static_cast<long long>(tok) * a.Hq + r) * D + lane8 * 8;
          *reinterpret_cast<uint4*>(dst) = o.u;
        }
      }
      const int h = is_v ? r - a.Hq - Hkv : r - a.Hq;
      if constexpr (!BITS4) {
        if (!is_q && there && keep) {
          uint8_t* dst = (is_v ? a.c.v : a.c.k) + cache_off + h * a.c.head_stride + lane8 * 16;
          *reinterpret_cast<uint4*>(dst) = o.u;
        }
      } else {
        float lo = f[0], hi = f[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) {
          lo = fminf(lo, f[e]);
          hi = fmaxf(hi, f[e]);
        }
#pragma unroll
        for (int s = 1; s < 4; s <<= 1) {
          lo = fminf(lo, __shfl_xor_sync(group_mask, lo, s));
          hi = fmaxf(hi, __shfl_xor_sync(group_mask, hi, s));
        }
        if (!is_q && there && keep) {
          T pair[2];
          pair[0] = from_f32<T>(__fdiv_rn(hi - lo, 15.0f));
          pair[1] = from_f32<T>(lo);
          const float scale = to_f32<T>(pair[0]), zero = to_f32<T>(pair[1]);
          uint32_t codes = 0;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float c = scale > 0.f ? fminf(fmaxf(rintf(__fdiv_rn(f[e] - zero, scale)), 0.f), 15.f) : 0.f;
            codes |= static_cast<uint32_t>(c) << (4 * e);
          }
          uint8_t* dst = (is_v ? a.c.v : a.c.k) + cache_off + h * a.c.head_stride;
          *reinterpret_cast<uint32_t*>(dst + lane8 * 4) = codes;
          if ((lane8 & 3) == 0) {
            T* sz = reinterpret_cast<T*>(dst + D / 2 + (lane8 >> 2) * 4);
            sz[0] = pair[0];
            sz[1] = pair[1];
          }
        }
      }
    }
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

template <typename A>
cudaError_t launch(const void* fn, dim3 grid, dim3 block, const A& a, cudaStream_t stream, bool pdl) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  void* params[] = {const_cast<A*>(&a)};
  return cudaLaunchKernelExC(&cfg, fn, params);
}

template <int D>
const void* append_fn(bool bf16, bool bits4) {
  if (bf16)
    return bits4 ? reinterpret_cast<const void*>(kv_append_kernel<D, __nv_bfloat16, true>)
                 : reinterpret_cast<const void*>(kv_append_kernel<D, __nv_bfloat16, false>);
  return bits4 ? reinterpret_cast<const void*>(kv_append_kernel<D, __half, true>)
               : reinterpret_cast<const void*>(kv_append_kernel<D, __half, false>);
}

template <int D>
const void* read_fn(bool bf16) {
  return bf16 ? reinterpret_cast<const void*>(kv4_read_kernel<D, __nv_bfloat16>)
              : reinterpret_cast<const void*>(kv4_read_kernel<D, __half>);
}

}  // namespace

cudaError_t launch_kv_append(const AppendArgs& a, int D, bool bf16, bool bits4, int sms, cudaStream_t stream, bool pdl) {
  const void* fn = D == 64 ? append_fn<64>(bf16, bits4) : D == 128 ? append_fn<128>(bf16, bits4) : append_fn<256>(bf16, bits4);
  // few tokens: a token's rows over several CTAs, one pass of rows each
  const int rows = a.Hq + 2 * a.c.Hkv, rpp = 2048 / D;
  int y = 1;
  if (a.N < 2 * sms) y = std::max(1, std::min((rows + rpp - 1) / rpp, 2 * sms / a.N));
  return launch(fn, dim3(a.N, y), dim3(256), a, stream, pdl);
}

cudaError_t launch_kv4_read(const Kv4ReadArgs& a, int D, bool bf16, cudaStream_t stream, bool pdl) {
  const void* fn = D == 64 ? read_fn<64>(bf16) : D == 128 ? read_fn<128>(bf16) : read_fn<256>(bf16);
  const long long threads = static_cast<long long>(a.M) * a.Hkv * (D / 8);
  return launch(fn, dim3(static_cast<unsigned>((threads + 255) / 256)), dim3(256), a, stream, pdl);
}

}  // namespace smb

// norm_rope_and_cache: what a layer does between its fused QKV projection and attention, in one pass over the rows. For
// every query and key head x of a token at position p
//   y = x rsqrt(mean(x^2) + eps) w                                 (w: the queries' or the keys' weights; left out: y = x)
//   (y_a, y_b) -> (y_a cos - y_b sin, y_b cos + y_a sin)          for the pairs (a, b) = (i, i + R/2), or (2i, 2i + 1), of
//                                                                  the first R elements, cos and sin from row p of the tables
// The queries go out, keys and values into the paged cache. All of it is fp32 and rounded once, where it is stored: the
// queries to their type, the keys to the cache's (16-bit, E4M3 or MXFP4).
//
// A lane holds a granule of 8 elements, a group of L = 8, 16 or 32 lanes a head (the power of two from D / 8 up): the sum
// of squares takes log2 L DPP steps, no LDS. The other half's elements of a pair (i, i + R/2) are loaded as a granule
// of their own, which the caches hold already, instead of moved between lanes. A thread keeps its place in the head over
// all of a token's heads, so that the table row and the weights are read once, and loads a pass ahead of what it computes
// (2048 tokens of 32 + 2 * 8 heads of 128, bf16, HBM-cold: 19.0 us, so 15.4; a copy of the projection takes 11.6). Bound by
// HBM (8192: 44.6 us, 4.5 TB/s) or, at a decode step's few tokens, by one launch.
#include "cache_rows.h"
#include "kvh_device.h"
#include "kvh_internal.h"

namespace kvh {
namespace {

constexpr int kThreads = 256;

template <int CTRL>
__device__ __forceinline__ float add_dpp(float x) {
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, false));
}

// The sum over this lane's group of L.
template <int L>
__device__ __forceinline__ float group_sum(float x) {
  x = add_dpp<0xB1>(x);   // lanes ^ 1
  x = add_dpp<0x4E>(x);   // lanes ^ 2
  x = add_dpp<0x141>(x);  // row_half_mirror: the other quad of 8
  if constexpr (L >= 16) x = add_dpp<0x140>(x);  // row_mirror: the other half of 16
  if constexpr (L == 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return x;
}

template <int DT>
__device__ __forceinline__ void store_e4m3(uint8_t* dst, const float (&x)[8], float scale) {
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = fp8_prep(x[i], scale);
  *(u32x2*)dst = u32x2{fp8_pack4(y[0], y[1], y[2], y[3]), fp8_pack4(y[4], y[5], y[6], y[7])};
}

// 8 elements as they lie in memory.
template <int DT>
struct Granule {
  u32x4 w[DT == 0 ? 2 : 1];
  __device__ __forceinline__ void load(const uint8_t* p) {
    w[0] = *(const u32x4*)p;
    if constexpr (DT == 0) w[1] = *(const u32x4*)(p + 16);
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (DT == 0) {
        x[i] = __uint_as_float(w[i / 4][i % 4]);
      } else {
        const uint16_t h = (uint16_t)(w[0][i / 2] >> (16 * (i & 1)));
        x[i] = DT == 2 ? BF16::to_f32(h) : F16::to_f32(h);
      }
    }
  }
};

// Workgroup (t, part) takes heads part * hpw .. of token t: query heads, then key heads, then value heads.
template <int DT, int CACHE, int L, bool PAIRS>
__global__ __launch_bounds__(kThreads) void norm_rope_kernel(NormRopeArgs a) {
  constexpr int EB = Rows<DT>::EB, HEADS = kThreads / L;
  const int64_t t = blockIdx.x;
  const int g = threadIdx.x % L, D = a.D, half = a.R / 2;  // granule of the head
  const bool in = 8 * g < D;
  const int d = in ? 8 * g : 0;
  const bool rot = d < a.R, low = d < half;
  const int d2 = rot && !PAIRS ? (low ? d + half : d - half) : d;  // the granule of the pairs' other elements
  const uint8_t* row = a.qkv + t * a.qkv_ts * EB;
  const int NH = a.H + 2 * a.Hkv, h0 = blockIdx.y * a.hpw, h1 = min(h0 + a.hpw, NH);
  // one pass ahead: this granule and the pairs' other one of the next head
  Granule<DT> xn, yn;
  auto load_head = [&](int hb) __attribute__((always_inline)) {
    const uint8_t* src = row + (int64_t)min(hb + (int)(threadIdx.x / L), h1 - 1) * D * EB;
    xn.load(src + d * EB);
    if (!PAIRS) yn.load(src + d2 * EB);
  };
  load_head(h0);
  Granule<DT> wq[2], wk[2];
  if (a.q_norm) {
    wq[0].load((const uint8_t*)a.q_norm + d * EB);
    wq[1].load((const uint8_t*)a.q_norm + d2 * EB);
  }
  if (a.k_norm) {
    wk[0].load((const uint8_t*)a.k_norm + d * EB);
    wk[1].load((const uint8_t*)a.k_norm + d2 * EB);
  }
  const int64_t pos = clamp64(a.positions[t], 0, a.max_pos - 1);
  const int64_t slot = a.slots[t];
  const bool in_pool = slot >= 0 && slot < a.num_slots;
  const int64_t blk = in_pool ? slot / a.BS : 0, off = in_pool ? slot % a.BS : 0;
  // the factors of this granule's own and other elements
  float c[8], s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = 1.f, s[i] = 0.f;
  if (rot) {
    const float* cr = a.cos_t + pos * half;
    const float* sr = a.sin_t + pos * half;
    if constexpr (PAIRS) {
      const f32x4 cv = *(const f32x4*)(cr + d / 2), sv = *(const f32x4*)(sr + d / 2);
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = cv[i / 2], s[i] = i & 1 ? sv[i / 2] : -sv[i / 2];
    } else {
      const int i0 = low ? d : d - half;
      Rows<0>::load8((const uint8_t*)(cr + i0), c);
      Rows<0>::load8((const uint8_t*)(sr + i0), s);
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] = low ? -s[i] : s[i];
    }
  }
  for (int hb = h0; hb < h1; hb += HEADS) {
    const int hw = hb + threadIdx.x / L;
    const int h = min(hw, h1 - 1);  // a group past the last head repeats it and stores nothing
    const bool is_q = h < a.H, is_v = h >= a.H + a.Hkv;
    float x[8], y[8];
    xn.get(x);
    if (!PAIRS) yn.get(y);
    if (hb + HEADS < h1) load_head(hb + HEADS);
    if (!is_v) {
      if (is_q ? a.q_norm : a.k_norm) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(x[i], x[i], ss);
        ss = group_sum<L>(in ? ss : 0.f);
        const float r = rsqrtf(ss / (float)D + a.eps);
        float wx[8], wy[8];
        (is_q ? wq : wk)[0].get(wx);
        if (!PAIRS) (is_q ? wq : wk)[1].get(wy);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] = x[i] * r * wx[i];
          if (!PAIRS) y[i] = y[i] * r * wy[i];
        }
      }
      if (rot) {
        float o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = x[i] * c[i] + (PAIRS ? x[i ^ 1] : y[i]) * s[i];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = o[i];
      }
    }
    uint32_t code = 0, e8m0 = 0;
    if constexpr (CACHE == 2) code = quantise8<DT>(x, e8m0);  // all four lanes of a quad are here
    if (!in || hw >= h1) continue;
    if (is_q) {
      Rows<DT>::store8(a.q_out + (t * a.q_ts + (int64_t)h * a.q_hs + d) * EB, x);
    } else if (in_pool) {
      const int kh = is_v ? h - a.H - a.Hkv : h - a.H;
      const Fp4Cache& kv = is_v ? a.vc : a.kc;
      const int64_t at = blk * kv.sb + off * kv.ss + (int64_t)kh * kv.sh;
      if constexpr (CACHE == 0) {
        Rows<DT>::store8(kv.c + (at + d) * EB, x);
      } else if constexpr (CACHE == 1) {
        store_e4m3<DT>(kv.c + at + d, x, is_v ? a.v_scale : a.k_scale);
      } else {
        *(uint32_t*)(kv.c + at + d / 2) = code;
        if ((g & 3) == 0) kv.x[blk * kv.xsb + off * kv.xss + (int64_t)kh * kv.xsh + g / 4] = (uint8_t)e8m0;
      }
    }
  }
}

template <int DT, int CACHE, int L>
int launch(NormRopeArgs a, bool pairs, int64_t T, hipStream_t s) {
  constexpr int heads = kThreads / L;
  const int NH = a.H + 2 * a.Hkv;
  // few tokens: a workgroup for each pass over `heads` heads, so that a step of a few sequences is one round of loads;
  // many: one for a token, whose table row and weights are read once (32 + 2 * 8 heads of 128, HBM-cold, us: 8 tokens 3.0
  // and 4.0, 256 4.4 and 5.0, 512 6.5 and 6.0, 2048 19.1 and 15.4, 8192 64.6 and 44.6; of 64: 256 3.7 and 4.1, 2048 12.8
  // and 11.0)
  a.hpw = T >= 512 ? NH : heads;
  const dim3 grid((unsigned)T, (NH + a.hpw - 1) / a.hpw);
  if (pairs)
    hipLaunchKernelGGL((norm_rope_kernel<DT, CACHE, L, true>), grid, dim3(kThreads), 0, s, a);
  else
    hipLaunchKernelGGL((norm_rope_kernel<DT, CACHE, L, false>), grid, dim3(kThreads), 0, s, a);
  return (int)hipGetLastError();
}

template <int DT, int CACHE>
int launch_l(const NormRopeArgs& a, bool pairs, int64_t T, hipStream_t s) {
  if (a.D <= 64) return launch<DT, CACHE, 8>(a, pairs, T, s);
  if (a.D <= 128) return launch<DT, CACHE, 16>(a, pairs, T, s);
  return launch<DT, CACHE, 32>(a, pairs, T, s);
}

template <int DT>
int launch_c(const NormRopeArgs& a, int32_t cache, bool pairs, int64_t T, hipStream_t s) {
  if (cache == KVH_CACHE_E4M3) return launch_l<DT, 1>(a, pairs, T, s);
  if (cache == KVH_CACHE_MXFP4) return launch_l<DT, 2>(a, pairs, T, s);
  return launch_l<DT, 0>(a, pairs, T, s);
}

}  // namespace

int launch_norm_rope(const NormRopeArgs& a, int64_t T, int32_t cache, bool pairs, int32_t dtype, hipStream_t s) {
  if (dtype == 2) return launch_c<2>(a, cache, pairs, T, s);
  return dtype == 1 ? launch_c<1>(a, cache, pairs, T, s) : launch_c<0>(a, cache, pairs, T, s);
}

}  // namespace kvh

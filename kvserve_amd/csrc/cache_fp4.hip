// Writing and reading an MXFP4 KV cache: E2M1 elements two to a byte with one E8M0 power of two for every 32 elements
// of a row (kvh_device.h). Three kernels over (token, head) rows, HBM-bound copies that convert on the way:
//
//   reshape_and_cache_fp4: this step's K/V rows quantised into the pool at their slots
//   rope_and_cache_fp4:    the split of the fused projection, RoPE, and that write
//   read_cache_fp4:        the rows at given slots back as 16-bit or fp32 values
//
// A block x[0..31] with the largest magnitude a (after a clamp to the largest value that the format and the rows' type
// both hold, which also takes the infinities; a NaN makes the block NaN) is stored under the smallest power of two 2^e
// with a < 7 * 2^e, i.e. e = floor(log2 a) - 2, one more where a's mantissa is 1.75 or more: no element is then off by
// more than half a step of its binade (with a <= 8 * 2^e, the usual rule, the largest could be off by a whole one).
// Elements are x / 2^e rounded to nearest even by v_cvt_scalef32_pk_fp4_f32. Every step before that is an integer
// operation on a's bits or exact, so the bytes are those of any fp32 implementation.
//
// A lane holds 8 consecutive elements (one or two 16-byte loads, a 4-byte store), a quad of lanes one block: its
// maximum takes two DPP steps, no LDS. The rows' 8-element granules are dealt out so that quads stay whole.
#include <type_traits>

#include "kvh_device.h"
#include "kvh_internal.h"

namespace kvh {
namespace {

constexpr int kThreads = 256;

template <int DT>  // KVH_DTYPE_*: 0 fp32, 1 fp16, 2 bf16
struct Rows {
  static constexpr int EB = DT == 0 ? 4 : 2;
  // 1.5 * 2^15 and 1.5 * 2^127: the next value of the format, 2^16 or 2^128, is past the type's range
  static __device__ __forceinline__ float largest() { return DT == 1 ? 49152.f : __uint_as_float(0x7f400000u); }
  static __device__ __forceinline__ void load8(const uint8_t* p, float (&x)[8]) {
    const u32x4 w = *(const u32x4*)p;
    if constexpr (DT == 0) {
      const u32x4 u = *(const u32x4*)(p + 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = __uint_as_float(w[i]);
        x[4 + i] = __uint_as_float(u[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint16_t h = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
        x[i] = DT == 2 ? BF16::to_f32(h) : F16::to_f32(h);
      }
    }
  }
  static __device__ __forceinline__ void store8(uint8_t* p, const float (&x)[8]) {
    if constexpr (DT == 0) {
      *(f32x4*)p = f32x4{x[0], x[1], x[2], x[3]};
      *(f32x4*)(p + 16) = f32x4{x[4], x[5], x[6], x[7]};
    } else {
      u32x4 w;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = DT == 2 ? BF16::pack2(x[2 * i], x[2 * i + 1]) : F16::pack2(x[2 * i], x[2 * i + 1]);
      *(u32x4*)p = w;
    }
  }
};

template <int CTRL>
__device__ __forceinline__ uint32_t quad_max(uint32_t x) {
  const uint32_t y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, false);
  return x > y ? x : y;
}

// 8 elements of this lane (a quad holds a block; all four lanes are here): their E2M1 codes, the block's E8M0 byte.
template <int DT>
__device__ __forceinline__ uint32_t quantise8(const float (&in)[8], uint32_t& e8m0) {
  const float big = Rows<DT>::largest();
  float x[8];
  uint32_t a = 0;  // magnitudes compare as integers, and a NaN's is above all
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = in[i] > big ? big : (in[i] < -big ? -big : in[i]);  // lets NaN through
    const uint32_t m = __float_as_uint(x[i]) & 0x7fffffffu;
    a = a > m ? a : m;
  }
  a = quad_max<0xB1>(a);  // lanes ^ 1
  a = quad_max<0x4E>(a);  // lanes ^ 2
  const int e = (int)((a + 0x200000u) >> 23) - 2;  // a mantissa of 1.75 or more carries into the exponent
  const uint32_t s = a > 0x7f800000u ? 255u : (uint32_t)(e < 2 ? 2 : e);  // at least 2^-125: every value is normal
  e8m0 = s;
  const float f = fp4_scale(s);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], f, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], f, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], f, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], f, 3);
  return w;
}

// Byte offset of a slot (in the pool) from a cache's first, and of its scales.
struct SlotAt {
  int64_t c, x;
};
__device__ __forceinline__ SlotAt slot_at(const Fp4Cache& k, int64_t slot, int64_t num_slots, int BS) {
  int64_t b, o;
  if (num_slots <= 0x7fffffffLL) {
    const uint32_t s = (uint32_t)slot, q = s / (uint32_t)BS;
    b = q;
    o = s - q * (uint32_t)BS;
  } else {
    b = slot / BS;
    o = slot % BS;
  }
  return SlotAt{b * k.sb + o * k.ss, b * k.xsb + o * k.xss};
}

// Granule g (8 elements) of head h of the row at `at`.
__device__ __forceinline__ void store_granule(const Fp4Cache& k, const SlotAt& at, int h, int g, uint32_t w,
                                              uint32_t e8m0) {
  *(uint32_t*)(k.c + at.c + (int64_t)h * k.sh + 4 * g) = w;
  if ((g & 3) == 0) k.x[at.x + (int64_t)h * k.xsh + g / 4] = (uint8_t)e8m0;
}

constexpr int kMaxTokens = kFp4TokensPerWg;

// Thread r of a workgroup takes granules r, r + 256, ... of each of its nt tokens' K|V rows (K heads, then V heads):
// the tokens' loads are issued together, the conversions and stores follow.
template <int DT>
__global__ __launch_bounds__(kThreads) void reshape_and_cache_fp4_kernel(
    const uint8_t* k, int64_t k_ts, int64_t k_hs, const uint8_t* v, int64_t v_ts, int64_t v_hs, Fp4Cache kc,
    Fp4Cache vc, const int64_t* slots, int64_t num_slots, int Hkv, int D, int BS, int64_t T, int tpw) {
  constexpr int EB = Rows<DT>::EB;
  const int gpr = D / 8;  // granules of a row, a multiple of 4
  const int per_tensor = Hkv * gpr;
  const int64_t t0 = (int64_t)blockIdx.x * tpw;
  const int nt = (int)min((int64_t)tpw, T - t0);
  int64_t slot[kMaxTokens];
#pragma unroll
  for (int j = 0; j < kMaxTokens; ++j) slot[j] = j < nt ? slots[t0 + j] : -1;
  for (int r0 = threadIdx.x; r0 < 2 * per_tensor; r0 += kThreads) {
    const bool is_v = r0 >= per_tensor;
    const int r = is_v ? r0 - per_tensor : r0;
    const int h = r / gpr, g = r % gpr;
    const int64_t ts = is_v ? v_ts : k_ts;
    const uint8_t* src = (is_v ? v : k) + (t0 * ts + (int64_t)h * (is_v ? v_hs : k_hs) + 8 * g) * EB;
    float f[kMaxTokens][8];
#pragma unroll
    for (int j = 0; j < kMaxTokens; ++j)
      if (j < nt) Rows<DT>::load8(src + j * ts * EB, f[j]);
#pragma unroll
    for (int j = 0; j < kMaxTokens; ++j) {
      if (j >= nt || slot[j] < 0 || slot[j] >= num_slots) continue;  // workgroup-uniform
      uint32_t s;
      const uint32_t w = quantise8<DT>(f[j], s);
      const Fp4Cache& c = is_v ? vc : kc;
      store_granule(c, slot_at(c, slot[j], num_slots, BS), h, g, w, s);
    }
  }
}

// One workgroup per token: items are 8 consecutive d of the first half of a query or key head with the matching 8 of
// the second half (a quad then holds a block of either half), and granules of the value heads. The rotation is
// computed in fp32 (two products and their sum, each rounded: no contraction) and rounded once, to q's type or to
// the format.
template <int DT>
__global__ __launch_bounds__(kThreads) void rope_and_cache_fp4_kernel(
    const uint8_t* qkv, int64_t qkv_ts, const int64_t* positions, const float* cos_t, const float* sin_t,
    int64_t max_pos, uint8_t* q_out, int64_t q_ts, int64_t q_hs, Fp4Cache kc, Fp4Cache vc, const int64_t* slots,
    int64_t num_slots, int H, int Hkv, int D, int BS) {
  constexpr int EB = Rows<DT>::EB;
  const int64_t t = blockIdx.x;
  const int half = D / 2, pv = half / 8, gpr = D / 8;
  const int n_rot = (H + Hkv) * pv, n_v = Hkv * gpr;
  const int64_t pos = clamp64(positions[t], 0, max_pos - 1);
  const float* cr = cos_t + pos * D;
  const float* sr = sin_t + pos * D;
  const int64_t slot = slots[t];
  const bool in_pool = slot >= 0 && slot < num_slots;
  const SlotAt k_at = slot_at(kc, in_pool ? slot : 0, num_slots, BS), v_at = slot_at(vc, in_pool ? slot : 0, num_slots, BS);
  const uint8_t* row = qkv + t * qkv_ts * EB;
  for (int it = threadIdx.x; it < n_rot + n_v; it += kThreads) {
    uint32_t s;
    if (it < n_rot) {
      const int h = it / pv, g = it % pv;  // query heads, then key heads
      const int d = 8 * g;
      const uint8_t* src = row + ((int64_t)h * D + d) * EB;
      float lo[8], hi[8], c_lo[8], c_hi[8], s_lo[8], s_hi[8], o_lo[8], o_hi[8];
      Rows<DT>::load8(src, lo);
      Rows<DT>::load8(src + half * EB, hi);
      Rows<0>::load8((const uint8_t*)(cr + d), c_lo);
      Rows<0>::load8((const uint8_t*)(cr + half + d), c_hi);
      Rows<0>::load8((const uint8_t*)(sr + d), s_lo);
      Rows<0>::load8((const uint8_t*)(sr + half + d), s_hi);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        o_lo[j] = lo[j] * c_lo[j] + -hi[j] * s_lo[j];
        o_hi[j] = hi[j] * c_hi[j] + lo[j] * s_hi[j];
      }
      if (h < H) {
        uint8_t* dst = q_out + (t * q_ts + (int64_t)h * q_hs + d) * EB;
        Rows<DT>::store8(dst, o_lo);
        Rows<DT>::store8(dst + half * EB, o_hi);
      } else if (in_pool) {
        uint32_t w = quantise8<DT>(o_lo, s);
        store_granule(kc, k_at, h - H, g, w, s);
        w = quantise8<DT>(o_hi, s);
        store_granule(kc, k_at, h - H, g + pv, w, s);
      }
    } else if (in_pool) {
      const int r = it - n_rot, h = r / gpr, g = r % gpr;
      float x[8];
      Rows<DT>::load8(row + ((int64_t)(H + Hkv + h) * D + 8 * g) * EB, x);
      const uint32_t w = quantise8<DT>(x, s);
      store_granule(vc, v_at, h, g, w, s);
    }
  }
}

// 8 elements of a lane from their codes.
template <int DT>
__device__ __forceinline__ void dequantise8(uint8_t* dst, uint32_t w, uint32_t e8m0) {
  const float f = fp4_scale(e8m0);
  if constexpr (DT == 0) {
    typedef float f32x2_t __attribute__((ext_vector_type(2)));
    const f32x2_t a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, f, 1),
                  c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, f, 3);
    *(f32x4*)dst = f32x4{a[0], a[1], b[0], b[1]};
    *(f32x4*)(dst + 16) = f32x4{c[0], c[1], d[0], d[1]};
  } else {
    using E = std::conditional_t<DT == 2, BF16, F16>;
    *(u32x4*)dst = u32x4{E::template from_fp4x2<0>(w, f), E::template from_fp4x2<1>(w, f),
                         E::template from_fp4x2<2>(w, f), E::template from_fp4x2<3>(w, f)};
  }
}

// As the write: granules of up to kMaxTokens tokens' K|V rows per thread, loads together, then conversions and stores.
// A slot outside the pool gives zeros.
template <int DT>
__global__ __launch_bounds__(kThreads) void read_cache_fp4_kernel(Fp4Cache kc, Fp4Cache vc, const int64_t* slots,
                                                                  int64_t num_slots, uint8_t* k, int64_t k_ts,
                                                                  int64_t k_hs, uint8_t* v, int64_t v_ts, int64_t v_hs,
                                                                  int Hkv, int D, int BS, int64_t T, int tpw) {
  constexpr int EB = Rows<DT>::EB;
  const int gpr = D / 8, per_tensor = Hkv * gpr;
  const int64_t t0 = (int64_t)blockIdx.x * tpw;
  const int nt = (int)min((int64_t)tpw, T - t0);
  int64_t slot[kMaxTokens];
#pragma unroll
  for (int j = 0; j < kMaxTokens; ++j) slot[j] = j < nt ? slots[t0 + j] : -1;
  for (int r0 = threadIdx.x; r0 < 2 * per_tensor; r0 += kThreads) {
    const bool is_v = r0 >= per_tensor;
    const int r = is_v ? r0 - per_tensor : r0;
    const int h = r / gpr, g = r % gpr;
    const Fp4Cache& c = is_v ? vc : kc;
    uint32_t w[kMaxTokens], s[kMaxTokens];
#pragma unroll
    for (int j = 0; j < kMaxTokens; ++j) {
      w[j] = s[j] = 0;
      if (slot[j] < 0 || slot[j] >= num_slots) continue;
      const SlotAt at = slot_at(c, slot[j], num_slots, BS);
      w[j] = *(const uint32_t*)(c.c + at.c + (int64_t)h * c.sh + 4 * g);
      s[j] = c.x[at.x + (int64_t)h * c.xsh + g / 4];
    }
    const int64_t ts = is_v ? v_ts : k_ts;
    uint8_t* dst = (is_v ? v : k) + (t0 * ts + (int64_t)h * (is_v ? v_hs : k_hs) + 8 * g) * EB;
#pragma unroll
    for (int j = 0; j < kMaxTokens; ++j)
      if (j < nt) dequantise8<DT>(dst + j * ts * EB, w[j], s[j]);
  }
}

// Tokens per workgroup: about 512 workgroups or more, at most kMaxTokens tokens each.
int tokens_per_wg(int64_t T) { return T >= 4 * 512 ? 4 : (T >= 2 * 512 ? 2 : 1); }

}  // namespace

int launch_reshape_and_cache_fp4(const void* k, int64_t k_ts, int64_t k_hs, const void* v, int64_t v_ts, int64_t v_hs,
                                 const Fp4Cache& kc, const Fp4Cache& vc, const int64_t* slots, int64_t T,
                                 int64_t num_blocks, int32_t Hkv, int32_t D, int32_t BS, int32_t dtype, hipStream_t s) {
  const int tpw = tokens_per_wg(T);
  const dim3 grid((unsigned)((T + tpw - 1) / tpw));
#define KVH_LAUNCH(DT)                                                                                             \
  hipLaunchKernelGGL((reshape_and_cache_fp4_kernel<DT>), grid, dim3(kThreads), 0, s, (const uint8_t*)k, k_ts, k_hs, \
                     (const uint8_t*)v, v_ts, v_hs, kc, vc, slots, num_blocks * BS, Hkv, D, BS, T, tpw)
  if (dtype == 2) KVH_LAUNCH(2); else if (dtype == 1) KVH_LAUNCH(1); else KVH_LAUNCH(0);
#undef KVH_LAUNCH
  return (int)hipGetLastError();
}

int launch_rope_and_cache_fp4(const void* qkv, int64_t qkv_ts, const int64_t* positions, const float* cos_t,
                              const float* sin_t, int64_t max_pos, void* q_out, int64_t q_ts, int64_t q_hs,
                              const Fp4Cache& kc, const Fp4Cache& vc, const int64_t* slots, int64_t T,
                              int64_t num_blocks, int32_t H, int32_t Hkv, int32_t D, int32_t BS, int32_t dtype,
                              hipStream_t s) {
#define KVH_LAUNCH(DT)                                                                                               \
  hipLaunchKernelGGL((rope_and_cache_fp4_kernel<DT>), dim3((unsigned)T), dim3(kThreads), 0, s, (const uint8_t*)qkv,   \
                     qkv_ts, positions, cos_t, sin_t, max_pos, (uint8_t*)q_out, q_ts, q_hs, kc, vc, slots,           \
                     num_blocks * BS, H, Hkv, D, BS)
  if (dtype == 2) KVH_LAUNCH(2); else if (dtype == 1) KVH_LAUNCH(1); else KVH_LAUNCH(0);
#undef KVH_LAUNCH
  return (int)hipGetLastError();
}

int launch_read_cache_fp4(const Fp4Cache& kc, const Fp4Cache& vc, const int64_t* slots, void* k, int64_t k_ts,
                          int64_t k_hs, void* v, int64_t v_ts, int64_t v_hs, int64_t T, int64_t num_blocks, int32_t Hkv,
                          int32_t D, int32_t BS, int32_t dtype, hipStream_t s) {
  const int tpw = tokens_per_wg(T);
  const dim3 grid((unsigned)((T + tpw - 1) / tpw));
#define KVH_LAUNCH(DT)                                                                                          \
  hipLaunchKernelGGL((read_cache_fp4_kernel<DT>), grid, dim3(kThreads), 0, s, kc, vc, slots, num_blocks * BS,      \
                     (uint8_t*)k, k_ts, k_hs, (uint8_t*)v, v_ts, v_hs, Hkv, D, BS, T, tpw)
  if (dtype == 2) KVH_LAUNCH(2); else if (dtype == 1) KVH_LAUNCH(1); else KVH_LAUNCH(0);
#undef KVH_LAUNCH
  return (int)hipGetLastError();
}

}  // namespace kvh

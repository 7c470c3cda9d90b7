// Rows of 8-element granules, and their MXFP4 form: what the kernels that write KV caches share.
#pragma once

#include "kvh_device.h"
#include "kvh_internal.h"

namespace kvh {
namespace {

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

}  // namespace
}  // namespace kvh

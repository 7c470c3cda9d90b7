// Products with weights held in 4 bits: y = x W^T, W[r][c] = s (q[r][c] - z), a scale s and a zero point z for every row and
// group of 32, 64 or 128 consecutive c; and the gated form SiLU(x G^T) (x U^T) of a weight whose first half of rows is G and
// whose second is U. bf16 or fp16, any number of rows of x, on v_mfma_f32_16x16x32 with fp32 sums, rounded once.
//
// A code becomes an operand in two instructions for two elements: its four bits are the mantissa's top four under the exponent
// of 16, so the MFMA multiplies by 16 + q, exact in either type, and nothing is rounded on the way. With ag the sum of
// x (16 + q) over a group and X the sum of x, the group adds s (ag - (16 + z) X) to a row: two FMAs on the accumulators
// a group, X once for all weight rows that a wave holds.
//
// The weight lies in blocks of 16 rows by 128 c, one wave-wide load of 16 bytes a lane: lane (j, r) holds of row r the
// elements 32 u + 8 j .. + 7 in dword u, the A operand of step u, element 2 p in nibble p and 2 p + 1 in nibble 4 + p.
// Beside each block lie its groups' 16 dwords: s in the low half and 16 + z in the high one, as elements of the type.
// Rows past the last and c past k are padded (c: s = 0, and x is taken as 0).
#include "kvh_device.h"
#include "kvh_internal.h"
#include "linear4.h"

namespace kvh {
namespace {

constexpr int kSteps = kW4Block / 32;  // MFMA steps of a block

template <class E>
struct Code;
template <>
struct Code<BF16> {
  static __device__ __forceinline__ u32x4 operand(uint32_t w) {
    const uint32_t m = 0x00780078u, o = 0x41804180u;
    return u32x4{((w << 3) & m) | o, ((w >> 1) & m) | o, ((w >> 5) & m) | o, ((w >> 9) & m) | o};
  }
};
template <>
struct Code<F16> {
  static __device__ __forceinline__ u32x4 operand(uint32_t w) {
    const uint32_t m = 0x03c003c0u, o = 0x4c004c00u;
    return u32x4{((w << 6) & m) | o, ((w << 2) & m) | o, ((w >> 2) & m) | o, ((w >> 6) & m) | o};
  }
};

// Accumulators of RT weight tiles by MT tiles of 16 rows of x. WK waves take slices of k and add theirs up in LDS. Workgroup
// (b, c): weight tiles from b RT (GLU: RT / 2 of each half), rows of x from 16 MT c.
template <class E, int G, int MT, int RT, int WK, bool GLU>
__global__ __launch_bounds__(64 * WK) void linear4_kernel(Linear4Args a) {
  constexpr int NG = kW4Block / G, SPG = G / 32;  // groups of a block, steps of a group
  constexpr int PH = RT * MT * WK > 32 ? (MT * WK > 32 ? 1 : 32 / (MT * WK)) : RT;  // tiles summed up at a time
  static_assert(!GLU || RT % 2 == 0);
  __shared__ f32x4 red[WK][(GLU ? 2 : 1) * PH][MT][64];
  const int lane = threadIdx.x & 63, j = lane >> 4, n = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row0 = 16 * MT * blockIdx.y;
  int tile[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    if (GLU) {
      const int t = blockIdx.x * (RT / 2) + r / 2, half = a.tiles / 2;
      tile[r] = min(t, half - 1) + (r & 1) * half;  // gate and up tiles in turn
    } else {
      tile[r] = min((int)blockIdx.x * RT + r, a.tiles - 1);
    }
  }
  const int b0 = (int)((int64_t)a.blocks * wave / WK), b1 = (int)((int64_t)a.blocks * (wave + 1) / WK);

  const uint16_t* xr[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) xr[t] = a.x + (int64_t)min(row0 + 16 * t + n, a.m - 1) * a.x_rs + 8 * j;

  f32x4 acc[RT][MT];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};

  struct Codes {
    u32x4 c[RT], s[RT][NG];
  } w[2];
  auto load_codes = [&](Codes& d, int b) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int64_t at = (int64_t)tile[r] * a.blocks + b;
      d.c[r] = __builtin_nontemporal_load((const u32x4*)(a.codes + at * 1024) + lane);
#pragma unroll
      for (int g = 0; g < NG; ++g) d.s[r][g] = __builtin_nontemporal_load((const u32x4*)(a.scales + (at * NG + g) * 16) + j);
    }
  };
  u32x4 x[kSteps][MT];
  auto load_x = [&](int b) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < kSteps; ++u)
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const int c = kW4Block * b + 32 * u;  // k is whole groups, so whole steps
        if (c < a.k)
          x[u][t] = *(const u32x4*)(xr[t] + c);
        else
          x[u][t] = u32x4{0u, 0u, 0u, 0u};
      }
  };
  auto compute = [&](const Codes& d) __attribute__((always_inline)) {
    float X[NG][MT];
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        float s = 0.f;
#pragma unroll
        for (int u = g * SPG; u < (g + 1) * SPG; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) s = E::dot2_ones(x[u][t][i], s);
        X[g][t] = sum_over_groups(s);
      }
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        f32x4 ag[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) ag[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = g * SPG; u < (g + 1) * SPG; ++u) {
          const u32x4 q = Code<E>::operand(d.c[r][u]);
#pragma unroll
          for (int t = 0; t < MT; ++t) ag[t] = E::mfma(q, x[u][t], ag[t]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float s = E::to_f32((uint16_t)(d.s[r][g][e] & 0xffffu)), z = E::to_f32((uint16_t)(d.s[r][g][e] >> 16));
#pragma unroll
          for (int t = 0; t < MT; ++t) acc[r][t][e] = __builtin_fmaf(s, __builtin_fmaf(-z, X[g][t], ag[t][e]), acc[r][t][e]);
        }
      }
  };
  if (b0 < b1) {
    load_codes(w[0], b0);
    int b = b0;
    while (true) {
      load_x(b);
      if (b + 1 < b1) load_codes(w[1], b + 1);
      compute(w[0]);
      if (++b == b1) break;
      load_x(b);
      if (b + 1 < b1) load_codes(w[0], b + 1);
      compute(w[1]);
      if (++b == b1) break;
    }
  }

  // the slices' sums in order, PH tiles at a time; output tile o is wave o % WK's
  constexpr int OT = GLU ? RT / 2 : RT, T2 = GLU ? 2 : 1;
#pragma unroll
  for (int p = 0; p < OT; p += PH) {
    if (p) __syncthreads();
#pragma unroll
    for (int q = 0; q < PH * T2; ++q)
      if (p * T2 + q < RT)
#pragma unroll
        for (int t = 0; t < MT; ++t) red[wave][q][t][lane] = acc[p * T2 + q][t];
    __syncthreads();
    for (int o = wave; o < PH * MT; o += WK) {
      const int q = o / MT, t = o % MT;
      if (p + q >= OT) break;
      f32x4 g = red[0][q * T2][t][lane], u{};
#pragma unroll
      for (int v = 1; v < WK; ++v) g += red[v][q * T2][t][lane];
      if constexpr (GLU) {
        u = red[0][q * T2 + 1][t][lane];
#pragma unroll
        for (int v = 1; v < WK; ++v) u += red[v][q * T2 + 1][t][lane];
#pragma unroll
        for (int e = 0; e < 4; ++e) g[e] = g[e] / (1.f + __expf(-g[e])) * u[e];
      }
      // lane (j, n): rows 4 j .. 4 j + 3 of the tile, row n of x's
      const int row = row0 + 16 * t + n, col = 16 * (blockIdx.x * OT + p + q) + 4 * j;
      if (row >= a.m) continue;
      uint16_t* dst = a.y + (int64_t)row * a.y_rs + col;
      const uint32_t lo = E::pack2(g[0], g[1]), hi = E::pack2(g[2], g[3]);
      if (col + 4 <= a.n && a.vec) {
        *(u32x2*)dst = u32x2{lo, hi};
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < a.n) dst[e] = (uint16_t)((e < 2 ? lo : hi) >> (16 * (e & 1)));
      }
    }
  }
}

template <class E, int G, int MT, int RT, int WK, bool GLU>
int launch(const Linear4Args& a, hipStream_t s) {
  constexpr int OT = GLU ? RT / 2 : RT;
  const int tiles = GLU ? a.tiles / 2 : a.tiles;
  hipLaunchKernelGGL((linear4_kernel<E, G, MT, RT, WK, GLU>), dim3((tiles + OT - 1) / OT, (a.m + 16 * MT - 1) / (16 * MT)),
                     dim3(64 * WK), 0, s, a);
  return (int)hipGetLastError();
}

template <class E, int G, bool GLU>
int launch_form(const Linear4Args& a, hipStream_t s) {
  const Linear4Form f = linear4_form(a.tiles, a.blocks, a.m);
#define KVH_FORM(MT, RT, WK) \
  if (f.mt == MT && f.rt == RT && f.wk == WK) return launch<E, G, MT, (GLU && RT < 2) ? 2 : RT, WK, GLU>(a, s);
  KVH_FORM(1, 1, 4) KVH_FORM(1, 1, 8) KVH_FORM(1, 2, 4) KVH_FORM(1, 2, 8)
  KVH_FORM(2, 1, 4) KVH_FORM(2, 1, 8) KVH_FORM(2, 2, 4) KVH_FORM(2, 2, 8)
  KVH_FORM(3, 2, 4) KVH_FORM(3, 2, 8) KVH_FORM(4, 2, 4) KVH_FORM(4, 2, 8)
#undef KVH_FORM
  return (int)hipErrorInvalidValue;
}

template <class E, bool GLU>
int launch_group(const Linear4Args& a, int32_t group, hipStream_t s) {
  if (group == 128) return launch_form<E, 128, GLU>(a, s);
  if (group == 64) return launch_form<E, 64, GLU>(a, s);
  return launch_form<E, 32, GLU>(a, s);
}

}  // namespace

int launch_linear4(const Linear4Args& a, int32_t group, bool glu, int32_t dtype, hipStream_t s) {
  if (glu) return dtype == 2 ? launch_group<BF16, true>(a, group, s) : launch_group<F16, true>(a, group, s);
  return dtype == 2 ? launch_group<BF16, false>(a, group, s) : launch_group<F16, false>(a, group, s);
}

}  // namespace kvh

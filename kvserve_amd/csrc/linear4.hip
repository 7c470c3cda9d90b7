// Products with weights held in 4 bits: y = x W^T, W[r][c] = s (q[r][c] - z), a scale s and a zero point z for every row and
// group of 32, 64 or 128 consecutive c; and the gated form SiLU(x G^T) (x U^T) of a weight whose first half of rows is G and
// whose second is U. bf16 or fp16, any number of rows of x, on v_mfma_f32_16x16x32 with fp32 sums, rounded once.
//
// A code becomes an operand in four instructions for four elements: its four bits are the mantissa's top four under the
// exponent of 16, so the MFMA multiplies by 16 + q, exact in either type, and nothing is rounded on the way. With ag the sum
// of x (16 + q) over a group and X the sum of x, the group adds s (ag - (16 + z) X) to a row. x is the A operand, the weight
// B: a lane then holds sums of one weight row alone, one dword of s and z serves its accumulators, and X, the product with
// a B operand of ones, comes out in the accumulators' places. bf16 operands have the exponents 2^12 lower and the sums are
// multiplied by 2^12 at the end, which rounds nothing else: 128 x (16 + q) 2^-12 stays in the range of fp32 for any finite x.
//
// The weight lies in blocks of 16 rows by 128 c, one wave-wide load of 16 bytes a lane: lane (j, r) holds of row r the
// elements 32 u + 8 j .. + 7 in dword u, the operand of step u, element 2 p in nibble p and 2 p + 1 in nibble 4 + p.
// Beside them lie 16 dwords for each of the block's groups: s in the low half and 16 + z in the high one, as elements of
// the type. Rows past the last and c past k are padded; there s = 0, and x is read again from its row's end.
//
// x goes through LDS a chunk at a time, one chunk ahead, for all waves of a workgroup: read by each wave from the caches it
// took the loads' path from the weight (8 rows against (28672, 4096), gated: 18.9 us, so 14.0; 64 rows 83 and 30.5). Where the
// weight has few rows its k is split over workgroups as well, whose sums a second launch adds in order: every further
// workgroup of rows reads all of x. Few rows are bound by the codes (those 8: 4.3 TB/s),
// many by the vector instructions beside the MFMAs, about four to one (64 rows of x and 64 of the weight, a block in one
// group: 68 MFMAs, 128 instructions that convert, 64 that multiply by s, 64 that take out z), of which two would hide: 1000 rows
// against (8192, 4096) 0.77 PFLOP/s, in groups of 64 and 32, whose part grows with their number, 0.68 and 0.55.
#include "kvh_device.h"
#include "kvh_internal.h"
#include "linear4.h"

namespace kvh {
namespace {

constexpr int kSteps = kW4Block / 32;  // MFMA steps of a block

// The weight operand of one step, in units of 1 / kUnit, and such a unit twice.
template <class E>
struct Code;
template <>
struct Code<BF16> {
  static constexpr uint32_t kOne = 0x39803980u, kMask = 0x00780078u, k16 = 0x3b803b80u;
  static constexpr float kUnit = 4096.f;
  static __device__ __forceinline__ u32x4 operand(uint32_t w, uint32_t o) {
    return u32x4{((w << 3) & kMask) | o, ((w >> 1) & kMask) | o, ((w >> 5) & kMask) | o, ((w >> 9) & kMask) | o};
  }
};
template <>
struct Code<F16> {
  static constexpr uint32_t kOne = 0x3c003c00u, kMask = 0x03c003c0u, k16 = 0x4c004c00u;
  static constexpr float kUnit = 1.f;
  static __device__ __forceinline__ u32x4 operand(uint32_t w, uint32_t o) {
    return u32x4{((w << 6) & kMask) | o, ((w << 2) & kMask) | o, ((w >> 2) & kMask) | o, ((w >> 6) & kMask) | o};
  }
};

__device__ __forceinline__ float silu(float g) { return g / (1.f + __expf(-g)); }

// Four sums of rows of W, as they are accumulated, as elements of y (GLU: those of a gate, and of its up rows in u).
template <class E, bool GLU>
__device__ __forceinline__ f32x4 finish(f32x4 v, const f32x4& u) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e] *= Code<E>::kUnit;
    if constexpr (GLU) v[e] = silu(v[e]) * (u[e] * Code<E>::kUnit);
  }
  return v;
}

// Four neighbouring elements of y, of which some may lie past its last column.
template <class E>
__device__ __forceinline__ void store_y(const Linear4Args& a, int row, int col, const f32x4& v) {
  uint16_t* dst = a.y + (int64_t)row * a.y_rs + col;
  const uint32_t lo = E::pack2(v[0], v[1]), hi = E::pack2(v[2], v[3]);
  if (col + 4 <= a.n && a.vec) {
    *(u32x2*)dst = u32x2{lo, hi};
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (col + e < a.n) dst[e] = (uint16_t)((e < 2 ? lo : hi) >> (16 * (e & 1)));
  }
}

// Workgroup (b, c, z): weight tiles from b WR RT (GLU: RT / 2 of each half), rows of x from MT 16 c, chunks of split z.
// PD blocks of codes a wave in flight, two where the registers hold them.
template <class E, int G, int ROWS, int RT, int WR, int WK, int S, bool GLU>
__global__ __launch_bounds__(64 * WR * WK) void linear4_kernel(Linear4Args a) {
  constexpr int NG = kW4Block / G, SPG = G / 32;  // groups of a block, steps of a group
  constexpr int W = WR * WK, MT = (ROWS + 15) / 16, KB = S * WK;
  constexpr int XB = ROWS * 2 * kW4Block;  // bytes of a block of x
  constexpr int PD = RT * MT <= 8 ? 2 : 1, U = PD > S ? PD / S : 1;
  constexpr int TOTAL = KB * ROWS * 16, PIECES = (TOTAL + 64 * W - 1) / (64 * W);  // of 16 bytes, in a chunk, a thread
  static_assert(!GLU || RT % 2 == 0);
  static_assert(S % PD == 0 || PD % S == 0);
  constexpr Linear4Form kForm{ROWS, RT, WR, WK, S, 1};
  constexpr bool SHARE = linear4_shares(kForm);
  static_assert(!SHARE || ROWS % 16 == 0);
  __shared__ __attribute__((aligned(16))) char lds[linear4_lds(kForm)];
  const int lane = threadIdx.x & 63, j = lane >> 4, n = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wave % WR, wk = wave / WR;
  const int row0 = 16 * MT * blockIdx.y;
  const u32x4* codes[RT];
  const uint32_t* scales[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    int tile;
    if (GLU) {  // gate and up tiles in turn
      const int t = (blockIdx.x * WR + wr) * (RT / 2) + r / 2, half = a.tiles / 2;
      tile = min(t, half - 1) + (r & 1) * half;
    } else {
      tile = min(((int)blockIdx.x * WR + wr) * RT + r, a.tiles - 1);
    }
    codes[r] = (const u32x4*)a.codes + (int64_t)tile * a.blocks * 64;
    scales[r] = a.scales + (int64_t)tile * a.blocks * NG * 16;
  }
  f32x4 acc[RT][MT];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};

  struct Codes {
    u32x4 c[RT];
    uint32_t s[RT][NG];
  } w[PD];
  auto load_codes = [&](Codes& d, int b) __attribute__((always_inline)) {
    b = min(b, a.blocks - 1);  // past the end: read again, not used
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      d.c[r] = __builtin_nontemporal_load(codes[r] + b * 64 + lane);
#pragma unroll
      for (int g = 0; g < NG; ++g) d.s[r][g] = scales[r][(b * NG + g) * 16 + n];
    }
  };
  // Piece p of a chunk: 8 elements of block p / 16 / ROWS, row p / 16 % ROWS. A row's 16 pieces of a block are put in places
  // xored with the row, so that the operands' reads (one piece of 16 rows) take all banks.
  u32x4 st[PIECES];
  auto stage_load = [&](int c) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < PIECES; ++q) {
      const int p = q * 64 * W + threadIdx.x, row = (p >> 4) % ROWS, b = (p >> 4) / ROWS;
      if (TOTAL % (64 * W) != 0 && p >= TOTAL) continue;
      const int k0 = (c * KB + b) * kW4Block + 8 * (p & 15);
      st[q] = *(const u32x4*)(a.x + (int64_t)min(row0 + row, a.m - 1) * a.x_rs + min(k0, a.k - 8));
    }
  };
  auto stage_store = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < PIECES; ++q) {
      const int p = q * 64 * W + threadIdx.x, row = (p >> 4) % ROWS, b = (p >> 4) / ROWS;
      if (TOTAL % (64 * W) != 0 && p >= TOTAL) continue;
      *(u32x4*)(lds + (buf * KB + b) * XB + row * 2 * kW4Block + 16 * ((p ^ row) & 15)) = st[q];
    }
  };
  uint32_t k16 = Code<E>::k16;
  asm("" : "+v"(k16));  // in a register: an instruction takes one constant
  // SHARE: X of block i of a chunk in buffer `buf`, [group][row], written by the waves of a slice in turn and read a
  // chunk later, behind the barrier that is there; minus s z of the blocks that it is for meanwhile in sz.
  float sz[SHARE ? S : 1][RT][NG];
  auto sums_of = [&](int buf, int i) __attribute__((always_inline)) {
    return (float*)(lds + linear4_x(kForm)) + (buf * KB + wk * S + i) * NG * ROWS;
  };
  auto write_sums = [&](const char* xb, float* X) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < (MT + WR - 1) / WR; ++q) {
      const int t = q * WR + wr;
      if (t >= MT) break;
      const char* row = xb + (16 * t + n) * 2 * kW4Block;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = g * SPG; u < (g + 1) * SPG; ++u)
          v = E::mfma(*(const u32x4*)(row + 16 * ((4 * u + j) ^ n)),
                      u32x4{Code<E>::kOne, Code<E>::kOne, Code<E>::kOne, Code<E>::kOne}, v);
        if (n == 0) *(f32x4*)(X + g * ROWS + 16 * t + 4 * j) = v;
      }
    }
  };
  auto subtract = [&](int i, const float* X) __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const f32x4 v = *(const f32x4*)(X + g * ROWS + 16 * t + 4 * j);
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[r][t][e] = __builtin_fmaf(sz[i][r][g], v[e], acc[r][t][e]);
      }
  };
  auto step = [&](const Codes& d, const char* xb, int i) __attribute__((always_inline)) {
    u32x4 x[kSteps][MT];
#pragma unroll
    for (int u = 0; u < kSteps; ++u)
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const int row = ROWS < 16 ? n % ROWS : 16 * t + n;
        x[u][t] = *(const u32x4*)(xb + row * 2 * kW4Block + 16 * ((4 * u + j) ^ (row & 15)));
      }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      f32x4 X[MT];
#pragma unroll
      for (int t = 0; t < MT && !SHARE; ++t) {
        X[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = g * SPG; u < (g + 1) * SPG; ++u)
          X[t] = E::mfma(x[u][t], u32x4{Code<E>::kOne, Code<E>::kOne, Code<E>::kOne, Code<E>::kOne}, X[t]);
      }
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        f32x4 ag[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) ag[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = g * SPG; u < (g + 1) * SPG; ++u) {
          const u32x4 q = Code<E>::operand(d.c[r][u], k16);
#pragma unroll
          for (int t = 0; t < MT; ++t) ag[t] = E::mfma(x[u][t], q, ag[t]);
        }
        const float s = E::to_f32((uint16_t)(d.s[r][g] & 0xffffu)), z = E::to_f32((uint16_t)(d.s[r][g] >> 16));
        if constexpr (SHARE) sz[i][r][g] = -s * z;  // exact
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            acc[r][t][e] = __builtin_fmaf(s, SHARE ? ag[t][e] : __builtin_fmaf(-z, X[t][e], ag[t][e]), acc[r][t][e]);
      }
    }
  };

  const int all = (a.blocks + KB - 1) / KB;
  const int c_lo = (int)((int64_t)all * blockIdx.z / a.splits), c_hi = (int)((int64_t)all * (blockIdx.z + 1) / a.splits);
  stage_load(c_lo);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < PD; ++i) load_codes(w[i], (c_lo + i / S) * KB + wk * S + i % S);
  __builtin_amdgcn_sched_barrier(0);
  stage_store(0);
  for (int c0 = c_lo; c0 < c_hi; c0 += U) {
#pragma unroll
    for (int cc = 0; cc < U; ++cc) {
      const int c = c0 + cc;
      if (c >= c_hi) break;
      __syncthreads();  // chunk c is in its buffer, the other one free
      const bool more = c + 1 < c_hi;
      if (more) stage_load(c + 1);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (SHARE)
#pragma unroll
        for (int i = 0; i < S; ++i)
          if (c > c_lo) subtract(i, sums_of((c - 1 - c_lo) & 1, i));  // (an earlier chunk is whole)
#pragma unroll
      for (int i = 0; i < S; ++i) {
        const int b = c * KB + wk * S + i;
        Codes& wi = w[(cc * S + i) % PD];
        if (b < a.blocks) {
          const char* xb = lds + (((c - c_lo) & 1) * KB + wk * S + i) * XB;
          if constexpr (SHARE) write_sums(xb, sums_of((c - c_lo) & 1, i));
          step(wi, xb, i);
        }
        __builtin_amdgcn_sched_barrier(0);
        load_codes(wi, (c + (i + PD) / S) * KB + wk * S + (i + PD) % S);  // the block PD steps on
        __builtin_amdgcn_sched_barrier(0);
      }
      if (more) stage_store((c + 1 - c_lo) & 1);
    }
  }

  // the slices' sums in order: lane l of a wave takes row l / 4 and columns 4 (l % 4) .. of an output tile
  float* red = (float*)lds;
  __syncthreads();
  if constexpr (SHARE) {
#pragma unroll
    for (int i = 0; i < S; ++i)
      if ((c_hi - 1) * KB + wk * S + i < a.blocks) subtract(i, sums_of((c_hi - 1 - c_lo) & 1, i));
    __syncthreads();
  }
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int t = 0; t < MT; ++t) *(f32x4*)(red + (((wave * RT + r) * MT + t) * 64 + lane) * 4) = acc[r][t];
  __syncthreads();
  constexpr int OT = GLU ? RT / 2 : RT, T2 = GLU ? 2 : 1;
  const int lr = lane >> 2, lc = lane & 3, at = ((lr >> 2) * 16 + 4 * lc) * 4 + (lr & 3);
  auto sum = [&](int g0, int r, int t) __attribute__((always_inline)) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < WK; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += red[(((k * WR + g0) * RT + r) * MT + t) * 256 + at + 4 * i];
    return v;
  };
  for (int o = wave; o < WR * OT * MT; o += W) {
    const int g0 = o / (OT * MT), q = o / MT % OT, t = o % MT;
    const int row = row0 + 16 * t + lr, tile = (blockIdx.x * WR + g0) * OT + q, col = 16 * tile + 4 * lc;
    f32x4 v = sum(g0, q * T2, t), u{};
    if constexpr (GLU) u = sum(g0, q * T2 + 1, t);
    if (row >= a.m) continue;
    if (a.splits > 1) {  // sums of 16-row tiles, gate tiles ahead of up tiles
      const int half = a.tiles / T2;
      if (tile >= half) continue;
      float* dst = a.ws + (((int64_t)blockIdx.z * a.m + row) * a.tiles + tile) * 16 + 4 * lc;
      *(f32x4*)dst = v;
      if constexpr (GLU) *(f32x4*)(dst + (int64_t)half * 16) = u;
      continue;
    }
    store_y<E>(a, row, col, finish<E, GLU>(v, u));
  }
}

// The splits' sums in order, a thread for four columns of a row.
template <class E, bool GLU>
__global__ __launch_bounds__(256) void linear4_sum_kernel(Linear4Args a) {
  const int quads = (GLU ? a.tiles / 2 : a.tiles) * 4;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= (int64_t)a.m * quads) return;
  const int row = (int)(id / quads), c = (int)(id % quads);
  const float* src = a.ws + (int64_t)row * a.tiles * 16 + 4 * c;
  const int64_t step = (int64_t)a.m * a.tiles * 16;
  f32x4 v = *(const f32x4*)src, u{};
  for (int z = 1; z < a.splits; ++z) v += *(const f32x4*)(src + z * step);
  if constexpr (GLU) {
    src += a.tiles * 8;
    u = *(const f32x4*)src;
    for (int z = 1; z < a.splits; ++z) u += *(const f32x4*)(src + z * step);
  }
  store_y<E>(a, row, 4 * c, finish<E, GLU>(v, u));
}

template <class E, int G, int ROWS, int RT, int WR, int WK, int S, bool GLU>
int launch(const Linear4Args& a, hipStream_t s) {
  constexpr int OT = (GLU ? RT / 2 : RT) * WR, MT = (ROWS + 15) / 16;
  const int tiles = GLU ? a.tiles / 2 : a.tiles;
  const dim3 grid((tiles + OT - 1) / OT, (a.m + 16 * MT - 1) / (16 * MT), a.splits);
  hipLaunchKernelGGL((linear4_kernel<E, G, ROWS, RT, WR, WK, S, GLU>), grid, dim3(64 * WR * WK), 0, s, a);
  int err = (int)hipGetLastError();
  if (err || a.splits == 1) return err;
  const int64_t work = (int64_t)a.m * tiles * 4;
  hipLaunchKernelGGL((linear4_sum_kernel<E, GLU>), dim3((unsigned)((work + 255) / 256)), dim3(256), 0, s, a);
  return (int)hipGetLastError();
}

template <class E, int G, bool GLU>
int launch_form(const Linear4Args& a, const Linear4Form& f, hipStream_t s) {
#define KVH_FORM(ROWS, RT, WR, WK, S)                                       \
  if (f.rows == ROWS && f.rt == RT && f.wr == WR && f.wk == WK && f.s == S) \
    return launch<E, G, ROWS, RT, WR, WK, S, GLU>(a, s);
  if constexpr (!GLU) {
    KVH_FORM(8, 1, 1, 8, 2)
    KVH_FORM(8, 1, 1, 16, 2)
    KVH_FORM(16, 1, 1, 8, 2)
    KVH_FORM(16, 2, 1, 8, 2)
    KVH_FORM(32, 1, 1, 8, 1)
    KVH_FORM(32, 1, 2, 8, 1)
    KVH_FORM(32, 1, 2, 4, 1)
    KVH_FORM(48, 1, 2, 4, 1)
    KVH_FORM(64, 1, 2, 4, 1)
  }
  KVH_FORM(16, 2, 2, 4, 2)
  KVH_FORM(16, 2, 4, 4, 2)
  KVH_FORM(32, 2, 2, 4, 1)
  KVH_FORM(48, 2, 2, 4, 1)
  KVH_FORM(64, 2, 2, 4, 1)
  KVH_FORM(32, 2, 4, 2, 1)
  KVH_FORM(48, 2, 4, 2, 1)
  KVH_FORM(64, 2, 4, 2, 1)
  KVH_FORM(32, 4, 2, 4, 1)
  KVH_FORM(48, 4, 2, 4, 1)
  KVH_FORM(64, 4, 4, 2, 1)
#undef KVH_FORM
  return (int)hipErrorInvalidValue;
}

template <class E, bool GLU>
int launch_group(const Linear4Args& a, const Linear4Form& f, int32_t group, hipStream_t s) {
  if (group == 128) return launch_form<E, 128, GLU>(a, f, s);
  if (group == 64) return launch_form<E, 64, GLU>(a, f, s);
  return launch_form<E, 32, GLU>(a, f, s);
}

}  // namespace

size_t linear4_workspace(int64_t m, int32_t tiles, int32_t blocks, bool glu) {
  const Linear4Form f = linear4_form(tiles, blocks, m, glu);
  return f.splits > 1 ? (size_t)f.splits * m * tiles * 16 * sizeof(float) : 0;
}

int launch_linear4(const Linear4Args& args, int32_t group, bool glu, int32_t dtype, hipStream_t s) {
  const Linear4Form f = linear4_form(args.tiles, args.blocks, args.m, glu);
  Linear4Args a = args;
  a.splits = f.splits;
  if (glu) return dtype == 2 ? launch_group<BF16, true>(a, f, group, s) : launch_group<F16, true>(a, f, group, s);
  return dtype == 2 ? launch_group<BF16, false>(a, f, group, s) : launch_group<F16, false>(a, f, group, s);
}

}  // namespace kvh

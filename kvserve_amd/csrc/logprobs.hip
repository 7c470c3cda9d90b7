// token_logprobs: for every row x[0..V) of a step's logits the log probability of one given token, the entropy of the
// row's distribution and its `top` largest entries with their log probabilities, in one pass over the logits:
//
//   m = max_j x_j,  s = sum_j e^(x_j - m),  t = sum_j e^(x_j - m) (x_j - m) / ln 2
//   log p_j = (x_j - m) - ln s,   entropy = -sum_j p_j log p_j = ln s - ln 2 t / s
//
// m, s, t are running values of a thread (fp32), rescaled where its maximum moves, then joined over lanes, waves and
// segments. With c = log2 e a term's exponent is d_j = c x_j - r, one FMA against the rounded r = fl(c m): rounded
// once relative to itself. What r is off by, delta = c m - r, is exact in one FMA and taken out at the end. Where |m| is
// above kFar, delta would be no small number: there d_j = c (x_j - m).
//
// HBM-bound on the logits, with the vector units close behind (8 issue slots an element: widening, maximum, FMA,
// exponential, two sums). A row is cut into S segments of 128 vectors or more (the last has what is left, down to
// none), a workgroup each, so that few rows fill the chip too; a second launch joins the segments (S = 1: none).
//
// The largest entries: the pass keeps the maxima of up to 16 x 64 cells, a cell being what four neighbouring threads read
// in a sixteenth of it (one more maximum a vector). The `top`-th largest of the 64 maxima over a quad of threads each
// is a lower bound thr of the segment's `top`-th largest entry, and rarely many more than `top` entries reach it (24
// expected of 20 asked for). They lie in cells whose maximum does, so those cells alone are read again (20 cells of a
// 256 KB row: 10 KB), and the entries found are ranked by counting, ties by the lower index. Where entries equal to thr
// abound (a row of few values, or masked with -inf but for fewer than `top`), the larger ones are ranked and the
// equal ones taken in index order; where more than kList are larger than thr (the largest entries all in few
// cells), `top` rounds of a whole maximum take their place.
//
// NaN counts as -inf in the order and makes the row's s and t NaN; an infinite or all -inf row gives NaN as well. A
// segment whose s is NaN takes its cells' maxima in a second pass, entry by entry: the first one's may lack what a signalling
// NaN stood beside.
#include <type_traits>

#include "kvh_device.h"
#include "kvh_internal.h"

// on a lambda: what it captures stays in registers
#define INLINE __attribute__((always_inline))

namespace kvh {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kGroups = 64, kSpans = 16;  // quads of threads, parts of the pass
constexpr int kCellsRead = 512;           // cells at or above thr, beyond which ties are taken in index order
// kList: a segment of fewer than 64 x 4 vectors leaves quads empty and may list all its entries
constexpr int kList = 2048, kJoinList = kMaxLogprobSplits * kMaxLogprobTop;
static_assert(kList >= kThreads * 8 && kJoinList <= kList, "rank_list holds an eighth of a list's 2048 in each thread");
constexpr int kUnroll = 4;

struct LogprobArgs {
  const uint8_t* x;
  int64_t row_bytes;
  const int64_t* tokens;
  float* logprobs;
  float* entropy;
  float* top_logprobs;
  int64_t* top_ids;
  int32_t V, top, S, vps;  // vps: vectors of a segment
  float4* part;            // [rows, S]: m, s, t
  uint64_t* keys;          // [rows, S, top], descending, 0 past a segment's entries
};

template <int DT>  // KVH_DTYPE_*
struct Vec {
  static constexpr int EB = DT == 0 ? 4 : 2, N = 16 / EB;
  static __device__ __forceinline__ void unpack(const u32x4& w, float (&f)[N]) {
    if constexpr (DT == 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint16_t h = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
        f[i] = DT == 2 ? BF16::to_f32(h) : F16::to_f32(h);
      }
    }
  }
  static __device__ __forceinline__ float one(const uint8_t* p) {
    if constexpr (DT == 0) return *(const float*)p;
    const uint16_t h = *(const uint16_t*)p;
    return DT == 2 ? BF16::to_f32(h) : F16::to_f32(h);
  }
};

// The order of entries: value (NaN as -inf, -0 as 0), then the lower index.
__device__ __forceinline__ uint64_t entry_key(float x, uint32_t index) {
  const uint32_t b = __float_as_uint((x == x ? x : -INFINITY) + 0.f);
  const uint32_t o = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
  return (uint64_t)o << 32 | (0xffffffffu - index);
}
__device__ __forceinline__ float key_value(uint64_t k) {
  const uint32_t o = (uint32_t)(k >> 32);
  return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
__device__ __forceinline__ uint32_t key_index(uint64_t k) { return 0xffffffffu - (uint32_t)k; }

__device__ __forceinline__ uint64_t max64(uint64_t a, uint64_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint64_t shfl_xor64(uint64_t x, int o) {
  return (uint64_t)(uint32_t)__shfl_xor((int)(x >> 32), o) << 32 | (uint32_t)__shfl_xor((int)(uint32_t)x, o);
}

constexpr float kLn2 = 0.6931471805599453f;
constexpr float kFar = 1048576.f;

struct Sums {
  float m, s, t;
};
// Both relative to the larger maximum (0 while that is -inf).
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
  const float m = fmaxf(a.m, b.m), ref = m == -INFINITY ? 0.f : m;
  const float da = (a.m - ref) * kLog2e, db = (b.m - ref) * kLog2e;
  const float wa = fast_exp2(da), wb = fast_exp2(db);
  Sums v;
  v.m = m;
  v.s = wa * a.s + wb * b.s;
  // an empty side weighs nothing (its d is -inf)
  v.t = (wa > 0.f ? wa * __builtin_fmaf(da, a.s, a.t) : 0.f) + (wb > 0.f ? wb * __builtin_fmaf(db, b.s, b.t) : 0.f);
  return v;
}
__device__ __forceinline__ Sums wave_join(Sums v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = join(v, Sums{__shfl_xor(v.m, o), __shfl_xor(v.s, o), __shfl_xor(v.t, o)});
  return v;
}

// The logit of the row's token, NaN for one outside the vocabulary: read ahead of the sums, two loads one after the other.
template <int DT>
__device__ __forceinline__ float token_logit(const LogprobArgs& a, int64_t row) {
  const int64_t tok = a.tokens[row];
  const bool in = tok >= 0 && tok < a.V;
  const float x = Vec<DT>::one(a.x + row * a.row_bytes + (in ? tok : 0) * Vec<DT>::EB);
  return in ? x : __uint_as_float(0x7fc00000u);
}

// The row's outputs but for the alternatives, from one thread.
__device__ __forceinline__ void write_row(const LogprobArgs& a, int64_t row, float x, const Sums& v, float ln_s) {
  a.logprobs[row] = x - v.m - ln_s;
  a.entropy[row] = ln_s - kLn2 * (v.t / v.s);
}

// max / min of three with no canonicalisation of the operands first. A quiet NaN among them is dropped. A signalling one
// comes out quieted where it meets another operand, and is dropped after that with what it met: logprob_kernel takes the
// cells of a row with a NaN again.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
  float r;
  asm("v_min3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// Ranks the n keys of `list` (distinct, n <= kList; the list is used up): emit(rank, key) for the first `top`. Many are
// thinned out first: the `top`-th largest of the threads' maxima is a lower bound, and few keys reach it.
template <class F>
__device__ __forceinline__ void rank_list(uint64_t* list, int n, int top, uint64_t* maxima, int* count, F&& emit) {
  if (n > kThreads) {
    uint64_t own[kList / kThreads], best = 0;
#pragma unroll
    for (int i = 0; i < kList / kThreads; ++i) {
      const int e = (int)threadIdx.x + i * kThreads;
      own[i] = e < n ? list[e] : 0;
      best = max64(best, own[i]);
    }
    maxima[threadIdx.x] = best;
    __syncthreads();
    if (threadIdx.x == 0) *count = 0;
    int above = 0;
#pragma unroll 8
    for (int i = 0; i < kThreads; ++i) above += maxima[i] > best;
    __syncthreads();
    if (above == top - 1) maxima[0] = best;
    __syncthreads();
    const uint64_t low = maxima[0];
#pragma unroll
    for (int i = 0; i < kList / kThreads; ++i)
      if (own[i] >= low) list[atomicAdd(count, 1)] = own[i];
    __syncthreads();
    n = *count;
  }
  for (int e = threadIdx.x; e < n; e += kThreads) {
    const uint64_t k = list[e];
    int r = 0;
#pragma unroll 8
    for (int i = 0; i < n; ++i) r += list[i] > k;
    if (r < top) emit(r, k);
  }
}

template <int DT, bool FINAL>
__global__ __launch_bounds__(kThreads, 6) void logprob_kernel(LogprobArgs a) {
  using X = Vec<DT>;
  constexpr int N = X::N, EB = X::EB;
  __shared__ Sums s_sums[kWaves];
  __shared__ alignas(8) float s_cell[kSpans][kGroups];  // (the keys' maxima of the threads once the entries are listed)
  static_assert(sizeof(s_cell) >= kThreads * sizeof(uint64_t), "");
  __shared__ float s_group[kGroups], s_thr;
  __shared__ uint64_t s_best[kWaves], s_list[kList];
  __shared__ uint16_t s_cand[kSpans * kGroups];
  __shared__ int s_n, s_nc, s_count[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = FINAL ? blockIdx.x : blockIdx.x / (unsigned)a.S;
  const int seg = FINAL ? 0 : (int)(blockIdx.x % (unsigned)a.S);
  const uint8_t* x = a.x + row * a.row_bytes;
  const int head = min(a.V, (int)((16 - ((uintptr_t)x & 15)) & 15) / EB);
  const int nvec = (a.V - head) / N, tail = a.V - head - nvec * N;
  const int v0 = min(nvec, seg * a.vps), v1 = FINAL || seg == a.S - 1 ? nvec : min(nvec, v0 + a.vps);
  const bool has_head = seg == 0 && tid < head, has_tail = (FINAL || seg == a.S - 1) && tid < tail;
  const u32x4* mid = (const u32x4*)(x + head * EB);
  const int tail0 = head + nvec * N;

  // the sums' reference is r = c m - delta (0 while m is -inf); entries below lo take the careful sum
  float m = -INFINITY, r = 0.f, delta = 0.f, lo = -kFar, s = 0.f, t = 0.f;
  float cell = -INFINITY;  // the thread's maximum in this span
  // an entry or vector whose maximum is mx: moves m
  auto raise = [&](float mx) INLINE {
    cell = fmaxf(cell, mx);
    if (__builtin_amdgcn_ballot_w64(mx > m)) {
      const float mn = fmaxf(m, mx);
      const bool none = mn == -INFINITY, far = fabsf(mn) > kFar && !none;
      const float rn = none ? 0.f : mn * kLog2e, dn = none || far ? 0.f : __builtin_fmaf(mn, kLog2e, -rn);
      // (an m that was -inf: nothing to rescale, d = -inf)
      const float d = none ? 0.f : (m - mn) * kLog2e - delta + dn, w = fast_exp2(d);
      t = w > 0.f ? w * __builtin_fmaf(d, s, t) : 0.f;
      s *= w;
      m = mn;
      r = rn;
      delta = dn;
      lo = far ? INFINITY : -kFar;
    }
  };
  auto add = [&](float v) INLINE {
    const float d = __builtin_fmaf(v, kLog2e, -r);
    const float e = fast_exp2(d);  // NaN stays
    s += e;
    t = __builtin_fmaf(e, d, t);
  };
  // also for -inf, the types' lowest values and maxima far from 0: an exponential of 0 meets a finite d
  auto add_careful = [&](float v) INLINE {
    const float d = lo == INFINITY ? (v - m) * kLog2e : __builtin_fmaf(v, kLog2e, -r);
    const float e = fast_exp2(d);
    s += e;
    t = __builtin_fmaf(e, fmaxf(d, -1000.f), t);
  };
  auto vector = [&](const u32x4& w) INLINE {
    float f[N];
    X::unpack(w, f);
    float mx = max3(f[0], f[1], f[2]), mn = min3(f[0], f[1], f[2]);
#pragma unroll
    for (int i = 3; i < N; i += 2) {
      mx = max3(mx, f[i], i + 1 < N ? f[i + 1] : f[i]);
      mn = min3(mn, f[i], i + 1 < N ? f[i + 1] : f[i]);
    }
    raise(mx);
    if (__builtin_amdgcn_ballot_w64(mn < lo)) {
#pragma unroll
      for (int i = 0; i < N; ++i) add_careful(f[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) add(f[i]);
    }
  };
  // spans of `quads` rounds of kUnroll vectors a thread; the last has the rest
  const int quads = (v1 - v0) / (kThreads * kUnroll) / kSpans + 1;
  int span = 0, left = quads;
  auto end_span = [&]() INLINE {
    float q = fmaxf(cell, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(cell), 0xB1, 0xf, 0xf, false)));
    q = fmaxf(q, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(q), 0x4E, 0xf, 0xf, false)));
    if ((tid & 3) == 0) s_cell[span][tid >> 2] = q;
    cell = -INFINITY;
    ++span;
    left = quads;
  };
  if (has_head) {
    const float v = X::one(x + tid * EB);
    raise(v);
    add_careful(v);
  }
  // rounds of kUnroll vectors, the next one's loads in flight under this one's sums
  const int rounds = (v1 - v0) / (kThreads * kUnroll);
  u32x4 even[kUnroll], odd[kUnroll];
  auto load = [&](u32x4 (&w)[kUnroll], int round) INLINE {
    const u32x4* src = mid + v0 + round * (kThreads * kUnroll) + tid;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) w[u] = __builtin_nontemporal_load(src + kThreads * u);
    __builtin_amdgcn_sched_barrier(0);
  };
  auto sum = [&](const u32x4 (&w)[kUnroll]) INLINE {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) vector(w[u]);
    if (--left == 0) end_span();
  };
  if (rounds > 0) load(even, 0);
  float target = 0.f;
  if constexpr (FINAL) target = token_logit<DT>(a, row);
  int round = 0;
  for (; round + 2 <= rounds; round += 2) {
    load(odd, round + 1);
    sum(even);
    load(even, min(round + 2, rounds - 1));
    sum(odd);
  }
  if (round < rounds) sum(even);
  if (const int i = v0 + rounds * (kThreads * kUnroll) + tid; v0 + rounds * (kThreads * kUnroll) < v1) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) odd[u] = mid[min(i + kThreads * u, v1 - 1)];
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (i + kThreads * u < v1) vector(odd[u]);
  }
  if (has_tail) {
    const float v = X::one(x + (tail0 + tid) * EB);
    raise(v);
    add_careful(v);
  }
  end_span();

  const float back = fast_exp2(-delta);  // from r to c m
  const Sums ws = wave_join(Sums{m, s * back, back * __builtin_fmaf(-delta, s, t)});
  if (lane == 0) s_sums[wave] = ws;
  if (tid == 0) s_n = s_nc = 0;
  __syncthreads();
  Sums v = s_sums[0];
#pragma unroll
  for (int k = 1; k < kWaves; ++k) v = join(v, s_sums[k]);
  const float ln_s = logf(v.s);
  if (tid == 0) {
    if constexpr (FINAL)
      write_row(a, row, target, v, ln_s);
    else
      a.part[row * a.S + seg] = float4{v.m, v.s, v.t, 0.f};
  }
  if (a.top == 0) return;
  if (v.s != v.s) {  // uniform: a NaN or a +inf. The cells again, entry by entry
    span = 0, left = quads;
    auto keep = [&](float e) INLINE { cell = e > cell ? e : cell; };  // no NaN is above
    auto keep_vector = [&](int i) INLINE {
      float f[N];
      X::unpack(mid[i], f);
#pragma unroll
      for (int j = 0; j < N; ++j) keep(f[j]);
    };
    if (has_head) keep(X::one(x + tid * EB));
    for (int i = v0 + tid, k = 0; k < rounds; ++k) {
      for (int u = 0; u < kUnroll; ++u, i += kThreads) keep_vector(i);
      if (--left == 0) end_span();
    }
    for (int i = v0 + rounds * (kThreads * kUnroll) + tid; i < v1; i += kThreads) keep_vector(i);
    if (has_tail) keep(X::one(x + (tail0 + tid) * EB));
    end_span();
    __syncthreads();
  }
  if (wave == 0) {
    float g = s_cell[0][lane];
    for (int k = 1; k < span; ++k) g = fmaxf(g, s_cell[k][lane]);
    s_group[lane] = g;
    if (lane == 0) s_thr = -INFINITY;
    __builtin_amdgcn_wave_barrier();
    int above = 0, reach = 0;
#pragma unroll 16
    for (int k = 0; k < kGroups; ++k) {
      above += s_group[k] > g;
      reach += s_group[k] >= g;
    }
    if (above < a.top && a.top <= reach) s_thr = g;  // of lanes of one value
  }
  __syncthreads();
  const float thr = s_thr;

  // which of a vector's entries are above, or at, low
  auto hits = [&](const u32x4& w, float low, bool equal) INLINE {
    float e[N];
    X::unpack(w, e);
    uint32_t hit = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float v = e[j] == e[j] ? e[j] : -INFINITY;
      hit |= (uint32_t)(v > low || (equal && v == low)) << j;
    }
    return hit;
  };
  auto edge_hit = [&](int j, float low, bool equal) INLINE {
    const float e = X::one(x + j * EB), v = e == e ? e : -INFINITY;
    return v > low || (equal && v == low);
  };
  auto key_of = [&](int j) INLINE { return entry_key(X::one(x + (int64_t)j * EB), j); };
  // this thread's share of the listed cells' vectors, then its own head and tail
  auto walk = [&](float low, bool equal, auto&& f) INLINE {
    const int len = 4 * kUnroll * quads, items = s_nc * len;
    for (int w0 = tid; w0 < items; w0 += kThreads * kUnroll) {
      u32x4 w[kUnroll];
      int i[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int q = min(w0 + kThreads * u, items - 1), c = q / len, k = q - c * len, cell = s_cand[c];
        i[u] = v0 + (cell / kGroups * kUnroll * quads + k / 4) * kThreads + cell % kGroups * 4 + k % 4;
        w[u] = mid[min(i[u], v1 - 1)];
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        uint32_t hit = w0 + kThreads * u < items && i[u] < v1 ? hits(w[u], low, equal) : 0;
        for (; hit; hit &= hit - 1) f(key_of(head + i[u] * N + __builtin_ctz(hit)));
      }
    }
    if (has_head && edge_hit(tid, low, equal)) f(key_of(tid));
    if (has_tail && edge_hit(tail0 + tid, low, equal)) f(key_of(tail0 + tid));
  };
  // lists the cells (of a segment with vectors) whose maximum is above, or at, thr
  auto list_cells = [&](bool equal) INLINE {
    for (int c = tid; c < span * kGroups && v0 < v1; c += kThreads) {
      const float g = s_cell[c / kGroups][c % kGroups];
      if (g > thr || (equal && g == thr)) s_cand[atomicAdd(&s_nc, 1)] = (uint16_t)c;
    }
    __syncthreads();
  };
  auto list_entries = [&](bool equal) INLINE {
    walk(thr, equal, [&](uint64_t k) INLINE {
      const int p = atomicAdd(&s_n, 1);
      if (p < kList) s_list[p] = k;
    });
    __syncthreads();
    return s_n;
  };
  auto emit = [&](int r, uint64_t k) INLINE {
    if constexpr (FINAL) {
      a.top_logprobs[row * a.top + r] = key_value(k) - v.m - ln_s;
      a.top_ids[row * a.top + r] = key_index(k);
    } else {
      a.keys[(row * a.S + seg) * a.top + r] = k;
    }
  };
  list_cells(true);
  int n = s_nc > kCellsRead ? kList + 1 : list_entries(true);
  if (n <= kList) {
    rank_list(s_list, n, a.top, (uint64_t*)s_cell, &s_nc, emit);
    if constexpr (!FINAL)
      for (int r = n + tid; r < a.top; r += kThreads) emit(r, 0);
    return;
  }
  __syncthreads();
  if (tid == 0) s_n = s_nc = 0;
  __syncthreads();
  list_cells(false);
  n = list_entries(false);
  if (n <= kList) {
    rank_list(s_list, n, a.top, (uint64_t*)s_cell, &s_nc, emit);
    // the rest: entries equal to thr (there are enough) in index order
    int found = n;
    auto take = [&](uint32_t hit, int first) INLINE {  // bit j: entry first + j is such a one
      const int count = __builtin_popcount(hit);
      int before = count;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(before, o);
        before += lane >= o ? y : 0;
      }
      if (lane == 63) s_count[wave] = before;
      before -= count;
      __syncthreads();
      int all = 0;
#pragma unroll
      for (int k = 0; k < kWaves; ++k) {
        before += k < wave ? s_count[k] : 0;
        all += s_count[k];
      }
      __syncthreads();
      for (int r = found + before; hit && r < a.top; ++r, hit &= hit - 1)
        emit(r, entry_key(thr, first + __builtin_ctz(hit)));
      found += all;
    };
    auto equals = [&](uint32_t at_or_above, uint32_t above) INLINE { return at_or_above & ~above; };
    take(has_head ? equals(edge_hit(tid, thr, true), edge_hit(tid, thr, false)) : 0, tid);
    for (int b = v0; b < v1 && found < a.top; b += kThreads) {
      const u32x4 w = mid[min(b + tid, v1 - 1)];
      take(b + tid < v1 ? equals(hits(w, thr, true), hits(w, thr, false)) : 0, head + (b + tid) * N);
    }
    if (found < a.top)
      take(has_tail ? equals(edge_hit(tail0 + tid, thr, true), edge_hit(tail0 + tid, thr, false)) : 0, tail0 + tid);
    if constexpr (!FINAL)
      for (int r = found + tid; r < a.top; r += kThreads) emit(r, 0);
    return;
  }
  uint64_t last = ~0ull;
  for (int r = 0; r < a.top; ++r) {  // the largest key below the last one
    uint64_t best = 0;
    walk(thr, false, [&](uint64_t k) INLINE { best = k < last ? max64(best, k) : best; });
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) best = max64(best, shfl_xor64(best, o));
    if (lane == 0) s_best[wave] = best;
    __syncthreads();
    last = max64(max64(s_best[0], s_best[1]), max64(s_best[2], s_best[3]));
    if (tid == 0) emit(r, last);
    __syncthreads();
  }
}

// Joins a row's segments: the sums over lanes, the alternatives as above (the segments' largest keys in the place of
// the cells' maxima).
template <int DT>
__global__ __launch_bounds__(kThreads) void logprob_join_kernel(LogprobArgs a) {
  __shared__ Sums s_sums;
  __shared__ uint64_t s_first[kMaxLogprobSplits], s_thr;
  __shared__ uint64_t s_list[kJoinList], s_maxima[kThreads];
  __shared__ int s_n;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  const uint64_t* keys = a.keys + row * a.S * a.top;
  if (tid == 0) {
    s_n = 0;
    s_thr = 1;
  }
  const float target = token_logit<DT>(a, row);
  // every load of the row's before the first is used
  uint64_t own[kJoinList / kThreads];
#pragma unroll
  for (int i = 0; i < kJoinList / kThreads; ++i) {
    const int k = tid + i * kThreads;
    own[i] = k < a.S * a.top ? keys[k] : 0;
  }
  // the segments' q-th largest keys: the (top / q)-th largest of them has `top` keys at or above it
  const int q = min(a.top, (2 * a.top + a.S - 1) / a.S);
  if (tid < 64) {
    Sums v{-INFINITY, 0.f, 0.f};
    if (tid < a.S) {
      const float4 p = a.part[row * a.S + tid];
      v = Sums{p.x, p.y, p.z};
    }
    if (a.top > 0 && tid < kMaxLogprobSplits) s_first[tid] = tid < a.S ? keys[(int64_t)tid * a.top + q - 1] : 0;
    v = wave_join(v);
    if (tid == 0) {
      s_sums = v;
      write_row(a, row, target, v, logf(v.s));
    }
  }
  if (a.top == 0) return;
  __syncthreads();
  if (tid < kMaxLogprobSplits) {
    const uint64_t g = s_first[tid];
    int r = 0;
#pragma unroll
    for (int k = 0; k < kMaxLogprobSplits; ++k) r += s_first[k] > g;
    if (r == (a.top + q - 1) / q - 1 && g != 0) s_thr = g;
  }
  __syncthreads();
  const uint64_t thr = s_thr;
#pragma unroll
  for (int i = 0; i < kJoinList / kThreads; ++i)
    if (own[i] >= thr) s_list[atomicAdd(&s_n, 1)] = own[i];
  __syncthreads();
  const Sums v = s_sums;
  const float ln_s = logf(v.s);
  rank_list(s_list, s_n, a.top, s_maxima, &s_n, [&](int r, uint64_t k) {
    a.top_logprobs[row * a.top + r] = key_value(k) - v.m - ln_s;
    a.top_ids[row * a.top + r] = key_index(k);
  });
}

int vec_elems(int32_t dtype) { return dtype == 0 ? 4 : 8; }

}  // namespace

// Segments of a row, one for every 256 vectors at most: up to kTarget workgroups in all, where a row to itself leaves the
// chip idle. A segment pays for its own alternatives and the joining launch, so no more (bf16, 128256 entries, 5
// alternatives, us by segments: 512 rows 1: 28.8, 2: 34.1; 300 rows 27.1, 27.5; 128 rows 1: 20.1, 2: 18.4, 4: 17.8,
// 8: 18.2; 64 rows 2: 17.7, 4: 15.1, 8: 14.5, 16: 15.0; 8 rows 8: 11.9, 32: 11.5).
int32_t logprob_splits(int64_t rows, int32_t V, int32_t dtype) {
  constexpr int64_t kTarget = 512;
  const int64_t chunks = (V / vec_elems(dtype) + kThreads - 1) / kThreads;
  int64_t s = rows > 0 ? kTarget / rows : 1;
  if (s > chunks) s = chunks;
  if (s > kMaxLogprobSplits) s = kMaxLogprobSplits;
  return s < 1 ? 1 : (int32_t)s;
}

int launch_token_logprobs(const void* logits, int64_t row_stride, const int64_t* tokens, float* logprobs,
                          float* entropy, float* top_logprobs, int64_t* top_ids, int64_t rows, int32_t V, int32_t top,
                          int32_t dtype, void* ws, hipStream_t st) {
  LogprobArgs a{};
  a.x = (const uint8_t*)logits;
  a.row_bytes = row_stride * (dtype == 0 ? 4 : 2);
  a.tokens = tokens;
  a.logprobs = logprobs;
  a.entropy = entropy;
  a.top_logprobs = top_logprobs;
  a.top_ids = top_ids;
  a.V = V;
  a.top = top;
  a.S = logprob_splits(rows, V, dtype);
  // shares in 8 vectors, whole 128-byte lines of rows that begin on one; the last segment takes the rest
  const int64_t nvec = V / vec_elems(dtype);
  a.vps = (int32_t)((nvec + a.S - 1) / a.S + 7) / 8 * 8;
  a.part = (float4*)ws;
  a.keys = (uint64_t*)((char*)ws + rows * a.S * sizeof(float4));
  const dim3 block(kThreads);
#define KVH_LAUNCH(DT)                                                                                       \
  if (a.S == 1) {                                                                                            \
    hipLaunchKernelGGL((logprob_kernel<DT, true>), dim3((unsigned)rows), block, 0, st, a);                  \
  } else {                                                                                                   \
    hipLaunchKernelGGL((logprob_kernel<DT, false>), dim3((unsigned)(rows * a.S)), block, 0, st, a);         \
    const int err = (int)hipGetLastError();                                                                  \
    if (err) return err;                                                                                     \
    hipLaunchKernelGGL((logprob_join_kernel<DT>), dim3((unsigned)rows), block, 0, st, a);                   \
  }
  if (dtype == 2) {
    KVH_LAUNCH(2)
  } else if (dtype == 1) {
    KVH_LAUNCH(1)
  } else {
    KVH_LAUNCH(0)
  }
#undef KVH_LAUNCH
  return (int)hipGetLastError();
}

}  // namespace kvh

// token_logprobs: for every row x[0..V) of a step's logits the log probability of one given token, the entropy of the
// row's distribution and its `top` largest entries with their log probabilities, in one pass over the logits:
//
//   m = max_j x_j,  s = sum_j e^(x_j - m),  t = sum_j e^(x_j - m) (x_j - m)
//   log p_j = (x_j - m) - ln s,   entropy = -sum_j p_j log p_j = ln s - t / s
//
// m, s, t are running values of a thread (fp32), rescaled where its maximum moves, then joined over lanes, waves
// and segments; x_j - m is taken before the product with log2 e, so the terms near the maximum are exact.
//
// HBM-bound on the logits. A row is cut into S segments of whole 256-vector chunks, a workgroup each, so that few rows
// fill the chip too; a second launch joins the segments (S = 1: none).
//
// The largest entries cost the pass one select per vector: a thread only remembers where its maximum was first seen.
// Entries are ordered by a 64-bit key, value first, then the lower index, so keys differ and the order is total. The
// `top`-th largest of the 64 maxima over four threads each is a lower bound of the segment's `top`-th largest key, and
// at least `top` entries, rarely many more (24 expected of 20 asked for), lie at or above it, all of them in threads
// whose maximum does: those threads walk their entries again (in the caches), the entries found are ranked by
// counting. Where more than kList are found (the largest entries all in few threads' strides), `top` rounds of a
// whole maximum take their place.
//
// NaN counts as -inf in the order and makes the row's m, s, t NaN; an infinite or all -inf row gives NaN as well.
#include "kvh_device.h"
#include "kvh_internal.h"

namespace kvh {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kGroups = 64;  // threads' maxima are ranked in groups of four
constexpr int kList = 2048, kJoinList = kMaxLogprobSplits * kMaxLogprobTop;
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

struct Sums {
  float m, s, t;
};
// Both relative to the larger maximum (0 while that is -inf).
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
  const float m = fmaxf(a.m, b.m), ref = m == -INFINITY ? 0.f : m;
  const float da = a.m - ref, db = b.m - ref;
  const float wa = fast_exp2(da * kLog2e), wb = fast_exp2(db * kLog2e);
  Sums r;
  r.m = m;
  r.s = wa * a.s + wb * b.s;
  // an empty side weighs nothing (its d is -inf)
  r.t = (wa > 0.f ? wa * __builtin_fmaf(da, a.s, a.t) : 0.f) + (wb > 0.f ? wb * __builtin_fmaf(db, b.s, b.t) : 0.f);
  return r;
}
__device__ __forceinline__ Sums wave_join(Sums v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = join(v, Sums{__shfl_xor(v.m, o), __shfl_xor(v.s, o), __shfl_xor(v.t, o)});
  return v;
}

// The row's outputs but for the alternatives, from one thread.
template <int DT>
__device__ __forceinline__ void write_row(const LogprobArgs& a, int64_t row, const Sums& v, float ln_s) {
  const int64_t tok = a.tokens[row];
  const bool in = tok >= 0 && tok < a.V;
  const float x = Vec<DT>::one(a.x + row * a.row_bytes + (in ? tok : 0) * Vec<DT>::EB);
  a.logprobs[row] = in ? x - v.m - ln_s : __uint_as_float(0x7fc00000u);
  a.entropy[row] = ln_s - v.t / v.s;
}

// Ranks the n keys of `list` (distinct): emit(rank, key) for the first `top`.
template <class F>
__device__ __forceinline__ void rank_list(const uint64_t* list, int n, int top, F&& emit) {
  for (int e = threadIdx.x; e < n; e += kThreads) {
    const uint64_t k = list[e];
    int r = 0;
    for (int i = 0; i < n; ++i) r += list[i] > k;
    if (r < top) emit(r, k);
  }
}

// A thread's entries in the order of their indexes: an element of the row's unaligned head, vectors v0 + tid,
// v0 + tid + 256, ... of its aligned middle, an element of its tail.
constexpr int kNone = -3, kTail = -2, kHead = -1;

template <int DT, bool FINAL>
__global__ __launch_bounds__(kThreads) void logprob_kernel(LogprobArgs a) {
  using X = Vec<DT>;
  constexpr int N = X::N, EB = X::EB;
  __shared__ Sums s_sums[kWaves];
  __shared__ uint64_t s_group[kGroups], s_thr, s_best[kWaves];
  __shared__ uint64_t s_list[kList];
  __shared__ int s_n;
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

  float m = -INFINITY, s = 0.f, t = 0.f;
  int at = has_head ? kHead : (v0 + tid < v1 ? v0 + tid : (has_tail ? kTail : kNone));
  // an entry or vector whose maximum is mx, first at `where`: moves m
  auto raise = [&](float mx, int where) {
    at = mx > m ? where : at;
    if (__builtin_amdgcn_ballot_w64(mx > m)) {
      const float mn = fmaxf(m, mx), d = m - mn;
      const float w = mn == -INFINITY ? 1.f : fast_exp2(d * kLog2e);
      t = w > 0.f ? w * __builtin_fmaf(mx > m ? d : 0.f, s, t) : 0.f;
      s *= w;
      m = mn;
    }
  };
  auto add = [&](float v, float ref) {
    const float d = v - ref;
    const float e = fast_exp2(d * kLog2e);  // NaN stays
    s += e;
    t = __builtin_fmaf(e, fmaxf(d, -1000.f), t);  // e is 0 there: -inf adds nothing
  };
  auto vector = [&](const u32x4& w, int where) {
    float f[N];
    X::unpack(w, f);
    float mx = fmaxf(f[0], f[1]);
#pragma unroll
    for (int i = 2; i < N; ++i) mx = fmaxf(mx, f[i]);
    raise(mx, where);
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < N; ++i) add(f[i], ref);
  };
  if (has_head) {
    const float v = X::one(x + tid * EB);
    raise(v, kHead);
    add(v, m == -INFINITY ? 0.f : m);
  }
  int i = v0 + tid;
  for (; i - tid + kThreads * kUnroll <= v1; i += kThreads * kUnroll) {
    u32x4 w[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) w[u] = mid[i + kThreads * u];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) vector(w[u], i + kThreads * u);
  }
  for (; i < v1; i += kThreads) vector(mid[i], i);
  if (has_tail) {
    const float v = X::one(x + (tail0 + tid) * EB);
    raise(v, kTail);
    add(v, m == -INFINITY ? 0.f : m);
  }

  const Sums ws = wave_join(Sums{m, s, t});
  if (lane == 0) s_sums[wave] = ws;
  if (tid == 0) {
    s_n = 0;
    s_thr = 1;
  }
  // the key of the thread's maximum at its first place
  uint64_t mine = 0;
  if (a.top > 0) {
    if (at == kHead) {
      mine = entry_key(m, tid);
    } else if (at == kTail) {
      mine = entry_key(m, tail0 + tid);
    } else if (at >= 0) {
      float f[N];
      X::unpack(mid[at], f);
      int k = 0;
#pragma unroll
      for (int j = N - 1; j >= 0; --j) k = f[j] == m ? j : k;
      if (m == -INFINITY) k = 0;  // nothing above -inf, NaNs among it
      mine = entry_key(m, head + at * N + k);
    }
    uint64_t g = max64(mine, shfl_xor64(mine, 1));
    g = max64(g, shfl_xor64(g, 2));
    if ((tid & 3) == 0) s_group[tid >> 2] = g;
  }
  __syncthreads();
  Sums v = s_sums[0];
#pragma unroll
  for (int k = 1; k < kWaves; ++k) v = join(v, s_sums[k]);
  const float ln_s = logf(v.s);
  if (tid == 0) {
    if constexpr (FINAL)
      write_row<DT>(a, row, v, ln_s);
    else
      a.part[row * a.S + seg] = float4{v.m, v.s, v.t, 0.f};
  }
  if (a.top == 0) return;
  if (wave == 0) {
    const uint64_t g = s_group[lane];
    int r = 0;
    for (int k = 0; k < kGroups; ++k) r += s_group[k] > g;
    if (r == a.top - 1 && g != 0) s_thr = g;  // of distinct keys one at most
  }
  __syncthreads();
  const uint64_t thr = s_thr;
  const float thr_x = thr == 1 ? -INFINITY : key_value(thr);

  // f(key) for every entry of the thread at or above `low` in value
  auto walk = [&](float low, auto&& f) {
    if (has_head) f(entry_key(X::one(x + tid * EB), tid));
    for (int i = v0 + tid; i < v1; i += kThreads * kUnroll) {
      u32x4 w[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) w[u] = mid[min(i + kThreads * u, v1 - 1)];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        if (i + kThreads * u >= v1) continue;
        float e[N];
        X::unpack(w[u], e);
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (!(e[j] < low)) f(entry_key(e[j], head + (i + kThreads * u) * N + j));
      }
    }
    if (has_tail) f(entry_key(X::one(x + (tail0 + tid) * EB), tail0 + tid));
  };
  if (mine >= thr)
    walk(thr_x, [&](uint64_t k) {
      if (k < thr) return;
      const int p = atomicAdd(&s_n, 1);
      if (p < kList) s_list[p] = k;
    });
  __syncthreads();
  const int n = s_n;
  auto emit = [&](int r, uint64_t k) {
    if constexpr (FINAL) {
      a.top_logprobs[row * a.top + r] = key_value(k) - v.m - ln_s;
      a.top_ids[row * a.top + r] = key_index(k);
    } else {
      a.keys[(row * a.S + seg) * a.top + r] = k;
    }
  };
  if (n <= kList) {
    rank_list(s_list, n, a.top, emit);
    if constexpr (!FINAL)
      for (int r = n + tid; r < a.top; r += kThreads) emit(r, 0);
    return;
  }
  // more entries than the list holds: each round takes the largest key below the last one
  uint64_t last = ~0ull;
  for (int r = 0; r < a.top; ++r) {
    uint64_t best = 0;
    if (mine >= thr)  // the others' entries lie below thr
      walk(thr_x, [&](uint64_t k) { best = k < last ? max64(best, k) : best; });
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
// the threads' maxima).
template <int DT>
__global__ __launch_bounds__(kThreads) void logprob_join_kernel(LogprobArgs a) {
  __shared__ Sums s_sums;
  __shared__ uint64_t s_first[kMaxLogprobSplits], s_thr;
  __shared__ uint64_t s_list[kJoinList];
  __shared__ int s_n;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  const uint64_t* keys = a.keys + row * a.S * a.top;
  if (tid == 0) {
    s_n = 0;
    s_thr = 1;
  }
  if (tid < kMaxLogprobSplits) {
    Sums v{-INFINITY, 0.f, 0.f};
    if (tid < a.S) {
      const float4 p = a.part[row * a.S + tid];
      v = Sums{p.x, p.y, p.z};
    }
    if (a.top > 0) s_first[tid] = tid < a.S ? keys[(int64_t)tid * a.top] : 0;
    v = wave_join(v);
    if (tid == 0) {
      s_sums = v;
      write_row<DT>(a, row, v, logf(v.s));
    }
  }
  if (a.top == 0) return;
  __syncthreads();
  if (tid < kMaxLogprobSplits) {
    const uint64_t g = s_first[tid];
    int r = 0;
    for (int k = 0; k < kMaxLogprobSplits; ++k) r += s_first[k] > g;
    if (r == a.top - 1 && g != 0) s_thr = g;
  }
  __syncthreads();
  const uint64_t thr = s_thr;
  for (int k = tid; k < a.S * a.top; k += kThreads) {
    const uint64_t key = keys[k];
    if (key >= thr) s_list[atomicAdd(&s_n, 1)] = key;
  }
  __syncthreads();
  const Sums v = s_sums;
  const float ln_s = logf(v.s);
  rank_list(s_list, s_n, a.top, [&](int r, uint64_t k) {
    a.top_logprobs[row * a.top + r] = key_value(k) - v.m - ln_s;
    a.top_ids[row * a.top + r] = key_index(k);
  });
}

int vec_elems(int32_t dtype) { return dtype == 0 ? 4 : 8; }

}  // namespace

// Segments of a row: about kTarget workgroups in all (eight of a CU's, all resident), whole chunks of 256 vectors each.
int32_t logprob_splits(int64_t rows, int32_t V, int32_t dtype) {
  constexpr int64_t kTarget = 2048;
  const int64_t chunks = (V / vec_elems(dtype) + kThreads - 1) / kThreads;
  int64_t s = rows > 0 ? (kTarget + rows - 1) / rows : 1;
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
  const int64_t chunks = (V / vec_elems(dtype) + kThreads - 1) / kThreads;
  a.vps = (int32_t)((chunks + a.S - 1) / a.S) * kThreads;
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

// Log probabilities of given tokens, with the entropy of each row and its k likeliest alternatives.
//
//   z = x / tau,  m = max z,  S = sum exp(z - m),  W = sum exp(z - m)(z - m)
//   logp_t = z_t - m - log S,   H = log S - W / S
//   dx_j = (gl (1[j=t] - p_j) - gH p_j (logp_j + H) + sum_i gk_i (1[j=id_i] - p_j)) / tau
//
// Bound by memory: the forward reads the logits once, the backward reads them and writes the gradient.  A row is
// read by a cluster of 1 to 8 CTAs (several where there are fewer rows than the GPU has room for CTAs); each thread
// keeps a running maximum, sum and weighted sum over its 16-byte vectors, and they are joined by shuffles, shared
// memory and, across the cluster, distributed shared memory.  Exponentials are base 2 of differences to the running
// maximum, subtracted before they are scaled, so that a row of the type's lowest values stays uniform.
//
// The alternatives cost no second pass: the maximum of each group of 4 threads is known after the first.  With k
// groups' maxima at or above the k-th largest of them, every value of the top k lies in one of these groups, so only
// their vectors are read again (from L2) and compared.  Values order by (value, lowest index) as one 64-bit key, so
// there are no ties.
#include <cooperative_groups.h>

#include "decoder_ops.h"
#include "vec.cuh"

namespace mtorus {

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 512;
constexpr int kGroups = kThreads / 4;
constexpr int kMaxTop = 64;
constexpr int kCandidates = 1024;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLowest = -3.402823466e38f;  // finite, so that differences to it are never NaN
constexpr long long kNoKey = LLONG_MIN;

// 2^x to 2 steps of fp32; results below 2^-126 are 0 (a probability there no longer reaches any output's type).
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// Orders by value, then by lowest index; -0 equals 0 and NaN ranks with -inf.
__device__ __forceinline__ long long key_of(float x, int64_t index) {
  const int b = __float_as_int(isnan(x) ? -INFINITY : x);
  const int o = b < 0 ? -(b & 0x7fffffff) : b;
  return (long long)o * 0x100000000ll + (0xffffffffll - index);
}
__device__ __forceinline__ float key_value(long long k) {
  const int o = (int)(k >> 32);
  return __int_as_float(o < 0 ? (int)(0x80000000u | (unsigned)(-o)) : o);
}
__device__ __forceinline__ int64_t key_index(long long k) { return 0xffffffffll - (k & 0xffffffffll); }

struct Running {
  float m, s, w;  // maximum; sums of 2^t and 2^t t with t = (x - m) c
};

__device__ __forceinline__ void rescale(Running& a, float m, float c) {
  const float t = fmaxf((a.m - m) * c, -200.f);
  const float f = ex2(t);
  a.w = f * fmaf(t, a.s, a.w);
  a.s *= f;
  a.m = m;
}

__device__ __forceinline__ void join(Running& a, Running b, float c) {
  const float m = fmaxf(a.m, b.m);
  rescale(a, m, c);
  rescale(b, m, c);
  a.s += b.s;
  a.w += b.w;
}

// One value, whatever it is: NaN and inf - inf go on into the sums, a masked value adds 2^-200 * -200 = 0.
template <bool ENT>
__device__ __forceinline__ void add(Running& a, float x, float c) {
  if (x > a.m) rescale(a, x, c);
  const float t = ENT ? max_nan((x - a.m) * c, -200.f) : (x - a.m) * c;
  const float e = ex2(t);
  a.s += e;
  if (ENT) a.w = fmaf(e, t, a.w);
}

// Packed maximum of two 16-bit values each: a NaN loses, or wins.
template <typename T>
__device__ __forceinline__ uint32_t max_pair(uint32_t a, uint32_t b) {
  uint32_t y;
  if constexpr (std::is_same_v<T, bf16>)
    asm("max.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
  else
    asm("max.f16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
  return y;
}
template <typename T>
__device__ __forceinline__ uint32_t max_pair_nan(uint32_t a, uint32_t b) {
  uint32_t y;
  if constexpr (std::is_same_v<T, bf16>)
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
  else
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
  return y;
}

template <typename T>
__device__ __forceinline__ float largest(const Vec<T, 16 / sizeof(T)>& v) {
  if constexpr (sizeof(T) == 2) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&v);
    const float2 f = widen_pair<T>(max_pair<T>(max_pair<T>(w[0], w[1]), max_pair<T>(w[2], w[3])));
    return fmaxf(f.x, f.y);
  } else {
    return fmaxf(fmaxf(v.v[0], v.v[1]), fmaxf(v.v[2], v.v[3]));
  }
}

// A thread's sums over its vectors with few instructions per value: exponents x c - r with the reference r = m c,
// two values at a time. r is rounded; that shifts all exponents alike and fast_done() takes it out again. For the
// weighted sum, values are kept at -1e30 or above (fp16: at its lowest), so that an exponent is finite and a masked
// value adds 0 * finite. Good for maxima from -2^26 / c to 2^26 / c that lie well above that; fast_done() says so.
struct Fast {
  float m, r, best;  // m >= the lower limit; best: the largest value
  float2 s, w;
};

constexpr float kFastLimit = 67108864.f;  // 2^26: r is rounded by at most 2

__device__ __forceinline__ Fast fast_start(float c) {
  return Fast{-kFastLimit / c, -kFastLimit, -INFINITY, both(0.f), both(0.f)};
}

// A vector with a value above `best`.
template <bool ENT>
__device__ __forceinline__ void fast_raise(Fast& a, float vm, float c) {
  a.best = vm;
  if (vm <= a.m) return;
  const float r = vm * c, d = a.r - r, f = ex2(d);
  if (ENT) a.w = mul2(fma2(a.s, both(d), a.w), both(f));
  a.s = mul2(a.s, both(f));
  a.m = vm;
  a.r = r;
}

template <typename T>
__device__ __forceinline__ constexpr float kept_above() {
  return std::is_same_v<T, __half> ? -65504.f : -1e30f;
}

template <typename T, bool ENT>
__device__ __forceinline__ void fast_add(Fast& a, const Vec<T, 16 / sizeof(T)>& v, float c) {
  constexpr int N = 16 / sizeof(T) / 2;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float2 x;
    if constexpr (sizeof(T) == 2) {
      uint32_t w = reinterpret_cast<const uint32_t*>(&v)[i];
      if (ENT) w = max_pair_nan<T>(w, std::is_same_v<T, bf16> ? 0xf149f149u : 0xfbfffbffu);  // kept_above<T>()
      x = widen_pair<T>(w);
    } else {
      x = make_float2(v.v[2 * i], v.v[2 * i + 1]);
      if (ENT) x = make_float2(max_nan(x.x, kept_above<T>()), max_nan(x.y, kept_above<T>()));
    }
    const float2 t = fma2(x, both(c), both(-a.r));
    const float2 e = make_float2(ex2(t.x), ex2(t.y));
    a.s = add2(a.s, e);
    if (ENT) a.w = fma2(e, t, a.w);
  }
}

// The sums relative to the maximum itself; false where the values were out of range (a NaN or +inf among them shows
// in the sums and needs no second look).
template <typename T, bool ENT>
__device__ __forceinline__ bool fast_done(const Fast& a, float c, Running& out) {
  const float s = a.s.x + a.s.y, w = a.w.x + a.w.y;
  out = Running{kLowest, 0.f, 0.f};
  if (isnan(s)) {
    out.s = s;
    return true;
  }
  if (a.best == -INFINITY) return true;  // nothing, or masked values only
  if (a.best < a.m || fabsf(a.r) > kFastLimit) return false;
  if (ENT && (kept_above<T>() - a.m) * c > -200.f) return false;
  const float d = fmaf(a.m, c, -a.r), f = ex2(-d);
  out = Running{a.m, s * f, f * fmaf(-d, s, w)};
  return true;
}

__device__ __forceinline__ Running shuffle_join(Running a, float c) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Running b;
    b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
    b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
    b.w = __shfl_xor_sync(0xffffffffu, a.w, o);
    join(a, b, c);
  }
  return a;
}

// A row of V values as single values up to the first 16-byte boundary, vectors, and single values to its end.
template <typename T>
struct RowParts {
  static constexpr int VEC = 16 / sizeof(T);
  int64_t head, vectors, tail0;
  __device__ __forceinline__ RowParts(const T* row, int64_t V) {
    const int64_t off = (16 - reinterpret_cast<uintptr_t>(row) % 16) % 16 / sizeof(T);
    head = off < V ? off : V;
    vectors = (V - head) / VEC;
    tail0 = head + vectors * VEC;
  }
};

struct FwdParams {
  const void* logits;
  const int64_t* tokens;
  float *logprob, *stats, *entropy, *top_lp;
  int64_t* top_ids;
  int64_t ld, V;
  float c, inv_tau;
  int top, cluster;
};

struct TopShared {
  long long group[kGroups];
  long long cand[kCandidates];
  long long best[kMaxTop];  // this CTA's largest keys in falling order, kNoKey behind them
  int winners[kGroups];
  int n_cand, n_winners;
  long long threshold, red[kThreads / 32];
};

// Writes the `top` largest of keys[0, n) to out in falling order. The keys differ, but for kNoKey, which is left
// out; with fewer than `top` keys, kNoKey follows them where n < top.
__device__ __forceinline__ void rank_keys(const long long* keys, int n, long long* out, int top) {
  for (int i = n + threadIdx.x; i < top; i += kThreads) out[i] = kNoKey;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const long long k = keys[i];
    if (k == kNoKey) continue;
    int r = 0;
    for (int j = 0; j < n; ++j) r += keys[j] > k;
    if (r < top) out[r] = k;
  }
}

template <typename T, bool ENT, bool TOP>
__global__ void __launch_bounds__(kThreads) token_logprobs_fwd(const __grid_constant__ FwdParams p) {
  constexpr int VEC = 16 / sizeof(T);
  constexpr int UNROLL = 4;
  using V16 = Vec<T, VEC>;
  __shared__ Running warps[kThreads / 32];
  __shared__ Running all;
  __shared__ TopShared ts;  // left out where TOP is false
  const int C = p.cluster, rank = blockIdx.x % C;
  const int64_t row = blockIdx.x / C;
  const T* x = static_cast<const T*>(p.logits) + row * p.ld;
  const RowParts<T> parts(x, p.V);
  const V16* xv = reinterpret_cast<const V16*>(x + parts.head);
  const int tid = threadIdx.x;
  const int64_t step = (int64_t)kThreads * C, first = (int64_t)rank * kThreads + tid;

  // one pass: vector j of the row belongs to thread j % (kThreads C) of the cluster
  Fast sums = fast_start(p.c);
  int64_t best_at = first;
  auto take = [&](const V16& v, int64_t j) {
    const float vm = largest<T>(v);
    if (vm > sums.best) {
      best_at = j;
      fast_raise<ENT>(sums, vm, p.c);
    }
    fast_add<T, ENT>(sums, v, p.c);
  };
  int64_t j = first;
  for (; j + (UNROLL - 1) * step < parts.vectors; j += UNROLL * step) {
    V16 v[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) v[u] = xv[j + u * step];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) take(v[u], j + u * step);
  }
  for (; j < parts.vectors; j += step) take(xv[j], j);
  Running a;
  if (!fast_done<T, ENT>(sums, p.c, a)) {
    for (j = first; j < parts.vectors; j += step) {
      float f[VEC];
      widen(xv[j], f);
#pragma unroll
      for (int i = 0; i < VEC; ++i) add<ENT>(a, f[i], p.c);
    }
  }
  // the row's ends: at most 2 (VEC - 1) values, one each for the first threads of the cluster
  const int64_t ends = parts.head + (p.V - parts.tail0);
  const int64_t end_at = first < parts.head ? first : parts.tail0 + (first - parts.head);
  if (first < ends) add<ENT>(a, to_f<T>(x[end_at]), p.c);

  a = shuffle_join(a, p.c);
  if ((tid & 31) == 0) warps[tid >> 5] = a;
  if constexpr (TOP) {
    // the largest key of each group of 4 threads
    long long k = kNoKey;
    if (first < parts.vectors) {
      const V16 v = xv[best_at];
#pragma unroll
      for (int i = 0; i < VEC; ++i) k = max(k, key_of(to_f<T>(v.v[i]), parts.head + best_at * VEC + i));
    }
    k = max(k, __shfl_xor_sync(0xffffffffu, k, 1));
    k = max(k, __shfl_xor_sync(0xffffffffu, k, 2));
    if ((tid & 3) == 0) ts.group[tid >> 2] = k;
    if (tid == 0) {
      ts.n_cand = ts.n_winners = 0;
      ts.threshold = kNoKey;
    }
  }
  __syncthreads();
  if (tid < 32) {
    a = tid < kThreads / 32 ? warps[tid] : Running{kLowest, 0.f, 0.f};
    a = shuffle_join(a, p.c);
    if (tid == 0) all = a;
  }
  if constexpr (TOP) {
    if (tid < kGroups) {  // the k-th largest group maximum bounds the k-th largest value from below
      const long long k = ts.group[tid];
      int r = 0;
      for (int i = 0; i < kGroups; ++i) r += ts.group[i] > k;
      if (r == p.top - 1 && k != kNoKey) ts.threshold = k;
    }
    __syncthreads();
    const long long threshold = ts.threshold;
    if (tid < kGroups) {
      const long long k = ts.group[tid];
      if (k != kNoKey && k >= threshold) ts.winners[atomicAdd(&ts.n_winners, 1)] = tid;
    }
    __syncthreads();
    const float floor_value = threshold == kNoKey ? -INFINITY : key_value(threshold);
    auto offer = [&](float f, int64_t index) {
      if (f < floor_value) return;
      const long long k = key_of(f, index);
      if (k < threshold) return;
      const int at = atomicAdd(&ts.n_cand, 1);
      if (at < kCandidates) ts.cand[at] = k;
    };
    // every vector of the winners: 4 threads each, one round of the first pass after the other
    const unsigned won = ts.n_winners, rounds = (unsigned)((parts.vectors + step - 1) / step);
    for (unsigned i = tid; i < rounds * 4 * won; i += kThreads) {
      const unsigned round = i / 4 / won, owner = ts.winners[i / 4 - round * won] * 4 + (i & 3);
      const int64_t jj = round * step + rank * kThreads + owner;
      if (jj >= parts.vectors) continue;
      const V16 v = xv[jj];
#pragma unroll
      for (int e = 0; e < VEC; ++e) offer(to_f<T>(v.v[e]), parts.head + jj * VEC + e);
    }
    if (first < ends) offer(to_f<T>(x[end_at]), end_at);
    __syncthreads();
    const int n = ts.n_cand;
    if (n <= kCandidates) {
      rank_keys(ts.cand, n, ts.best, p.top);
    } else {
      // More values above the bound than there is room for: rows whose largest values all lie in a few threads'
      // vectors.  Takes the largest key below the last one, k times over.
      long long last = LLONG_MAX;
      for (int r = 0; r < p.top; ++r) {
        long long k = kNoKey;
        for (int64_t jj = first; jj < parts.vectors; jj += step) {
          const V16 v = xv[jj];
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const long long q = key_of(to_f<T>(v.v[e]), parts.head + jj * VEC + e);
            if (q < last) k = max(k, q);
          }
        }
        if (first < ends) {
          const long long q = key_of(to_f<T>(x[end_at]), end_at);
          if (q < last) k = max(k, q);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) k = max(k, __shfl_xor_sync(0xffffffffu, k, o));
        __syncthreads();
        if ((tid & 31) == 0) ts.red[tid >> 5] = k;
        __syncthreads();
        for (int w = 0; w < kThreads / 32; ++w) k = max(k, ts.red[w]);
        if (tid == 0) ts.best[r] = k;
        last = k;
      }
    }
  }
  if (C > 1) {  // the cluster's first CTA joins what the others hold
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    if (rank == 0) {
      if (tid == 0) {
        a = all;
        for (int r = 1; r < C; ++r) join(a, *cluster.map_shared_rank(&all, r), p.c);
      }
      if constexpr (TOP) {
        for (int i = tid; i < C * p.top; i += kThreads)
          ts.cand[i] = *cluster.map_shared_rank(&ts.best[i % p.top], i / p.top);
        __syncthreads();
        rank_keys(ts.cand, C * p.top, ts.best, p.top);  // V >= top: every place is filled
      }
    }
    cluster.sync();  // the others' shared memory lives until it has been read
    if (rank != 0) return;
  }
  if (TOP) __syncthreads();
  if (tid == 0) {
    all = a;
    const int64_t t = p.tokens[row];
    // a row without any possible token has S = 0
    const bool none = a.s == 0.f;
    const float l2s = none ? -INFINITY : log2f(a.s);
    float lp = 0.f;
    if (t >= 0 && t < p.V) lp = none ? -INFINITY : (to_f<T>(x[t]) - a.m) * p.inv_tau - l2s * kLn2;
    p.logprob[row] = lp;
    p.stats[2 * row] = a.m;
    p.stats[2 * row + 1] = l2s;
    if (ENT) p.entropy[row] = none ? 0.f : (l2s - a.w / a.s) * kLn2;
  }
  if constexpr (TOP) {
    __syncthreads();
    const float m = all.m, s = all.s;
    const float l2s = s == 0.f ? -INFINITY : log2f(s);
    for (int i = tid; i < p.top; i += kThreads) {
      const int64_t id = key_index(ts.best[i]);
      p.top_ids[row * p.top + i] = id;
      p.top_lp[row * p.top + i] = s == 0.f ? -INFINITY : (to_f<T>(x[id]) - m) * p.inv_tau - l2s * kLn2;
    }
  }
}

struct BwdParams {
  const void* logits;
  void* dlogits;
  const int64_t *tokens, *top_ids;
  const float *stats, *entropy, *g_logprob, *g_entropy, *g_top;
  int64_t ld, V;
  float c, inv_tau;
  int top, splits;
};

// One CTA per row, or per one of `splits` parts of a row.
template <typename T, bool ENT>
__global__ void __launch_bounds__(kThreads) token_logprobs_bwd(const __grid_constant__ BwdParams p) {
  constexpr int VEC = 16 / sizeof(T);
  using V16 = Vec<T, VEC>;
  const int64_t row = blockIdx.x / p.splits;
  const int part = blockIdx.x % p.splits, tid = threadIdx.x;
  const T* x = static_cast<const T*>(p.logits) + row * p.ld;
  T* dx = static_cast<T*>(p.dlogits) + row * p.V;
  const int64_t token = p.tokens[row];
  const bool use = p.g_logprob != nullptr && token >= 0 && token < p.V;
  const float m = p.stats[2 * row], l2s = p.stats[2 * row + 1];
  const float gl = use ? p.g_logprob[row] * p.inv_tau : 0.f;
  const float gh = ENT ? p.g_entropy[row] * p.inv_tau : 0.f;
  const float h = ENT ? p.entropy[row] : 0.f;
  float total = gl;
  if (p.g_top != nullptr) {
    for (int i = 0; i < p.top; ++i) total += p.g_top[row * p.top + i] * p.inv_tau;
  }
  const bool none = l2s == -INFINITY;  // no possible token: no gradient
  auto grad = [&](float v) {
    const float t = max_nan(fmaf(v - m, p.c, -l2s), -200.f);  // log2 of the probability
    const float e = ex2(t);
    return none ? 0.f : ENT ? -e * fmaf(gh, fmaf(t, kLn2, h), total) : -e * total;
  };
  // the gradient has no stride of its own: its rows may lie on other 16-byte offsets than the logits'
  const bool same = (reinterpret_cast<uintptr_t>(x) - reinterpret_cast<uintptr_t>(dx)) % 16 == 0;
  const RowParts<T> parts(x, p.V);
  const int64_t step = (int64_t)kThreads * p.splits, first = (int64_t)part * kThreads + tid;
  const V16* xv = reinterpret_cast<const V16*>(x + parts.head);
  for (int64_t j = first; j < parts.vectors; j += step) {
    float f[VEC];
    widen(load_stream(xv + j), f);
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = grad(f[i]);
    if (same) {
      store_stream(reinterpret_cast<V16*>(dx + parts.head) + j, narrow<T, VEC>(f));
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) dx[parts.head + j * VEC + i] = from_f<T>(f[i]);
    }
  }
  const int64_t ends = parts.head + (p.V - parts.tail0);
  const int64_t end_at = first < parts.head ? first : parts.tail0 + (first - parts.head);
  if (first < ends) dx[end_at] = from_f<T>(grad(to_f<T>(x[end_at])));
  // The token's own value and the alternatives', each whole and rounded once, by the CTA that wrote their vector.
  __syncthreads();
  for (int i = tid; i <= (p.g_top != nullptr ? p.top : 0); i += kThreads) {
    const int64_t id = i == 0 ? token : p.top_ids[row * p.top + i - 1];
    if (i == 0 && !use) continue;
    const int64_t owner = id < parts.head ? id
                          : id >= parts.tail0 ? parts.head + id - parts.tail0
                                              : (id - parts.head) / VEC % step;
    if (owner / kThreads != part) continue;
    float d = grad(to_f<T>(x[id]));
    if (!none) {
      if (use && id == token) d += gl;
      if (p.g_top != nullptr) {
        for (int q = 0; q < p.top; ++q) {
          if (p.top_ids[row * p.top + q] == id) d += p.g_top[row * p.top + q] * p.inv_tau;
        }
      }
    }
    dx[id] = from_f<T>(d);
  }
}

}  // namespace

void token_logprobs_fwd_launch(const at::Tensor& logits, const at::Tensor& tokens, double inv_tau, int64_t top,
                               const at::Tensor& logprob, const at::Tensor& stats, const at::Tensor& entropy,
                               const at::Tensor& top_lp, const at::Tensor& top_ids) {
  const int64_t rows = logits.size(0), V = logits.size(1);
  if (rows == 0) return;
  FwdParams p{};
  p.logits = logits.data_ptr();
  p.tokens = tokens.data_ptr<int64_t>();
  p.logprob = logprob.data_ptr<float>();
  p.stats = stats.data_ptr<float>();
  if (entropy.defined()) p.entropy = entropy.data_ptr<float>();
  if (top > 0) {
    p.top_lp = top_lp.data_ptr<float>();
    p.top_ids = top_ids.data_ptr<int64_t>();
  }
  p.ld = rows > 1 ? logits.stride(0) : V;
  p.V = V;
  p.inv_tau = (float)inv_tau;
  p.c = (float)(inv_tau * 1.4426950408889634);
  p.top = (int)top;
  // clusters until every SM has work, as long as each thread has a vector to read
  const int64_t vectors = V * logits.element_size() / 16;
  int C = 1;
  while (C < 8 && rows * C < num_sms() && vectors > (int64_t)kThreads * C) C *= 2;
  p.cluster = C;
  MT_CHECK(rows * C < (int64_t(1) << 31), "token_logprobs: too many rows: ", rows);
  auto launch = [&](auto kernel) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(rows * C));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = cur_stream();
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)C;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, p));
    MT_LAUNCH_CHECK();
  };
  dispatch_act(logits.scalar_type(), [&](auto t) {
    using T = decltype(t);
    const bool ent = entropy.defined();
    if (ent && top > 0)
      launch(token_logprobs_fwd<T, true, true>);
    else if (ent)
      launch(token_logprobs_fwd<T, true, false>);
    else if (top > 0)
      launch(token_logprobs_fwd<T, false, true>);
    else
      launch(token_logprobs_fwd<T, false, false>);
  });
}

void token_logprobs_bwd_launch(const at::Tensor& logits, const at::Tensor& tokens, double inv_tau, int64_t top,
                               const at::Tensor& stats, const at::Tensor& entropy, const at::Tensor& top_ids,
                               const at::Tensor& g_logprob, const at::Tensor& g_entropy, const at::Tensor& g_top,
                               const at::Tensor& dlogits) {
  const int64_t rows = logits.size(0), V = logits.size(1);
  if (rows == 0) return;
  BwdParams p{};
  p.logits = logits.data_ptr();
  p.dlogits = dlogits.data_ptr();
  p.tokens = tokens.data_ptr<int64_t>();
  p.stats = stats.data_ptr<float>();
  p.top = (int)top;
  if (g_logprob.defined()) p.g_logprob = g_logprob.data_ptr<float>();
  if (g_entropy.defined()) {
    p.g_entropy = g_entropy.data_ptr<float>();
    p.entropy = entropy.data_ptr<float>();
  }
  if (g_top.defined()) {
    p.g_top = g_top.data_ptr<float>();
    p.top_ids = top_ids.data_ptr<int64_t>();
  }
  p.ld = rows > 1 ? logits.stride(0) : V;
  p.V = V;
  p.inv_tau = (float)inv_tau;
  p.c = (float)(inv_tau * 1.4426950408889634);
  const int64_t vectors = V * logits.element_size() / 16;
  p.splits = 1;
  while (rows * p.splits < 4 * num_sms() && vectors > (int64_t)kThreads * p.splits) p.splits *= 2;
  MT_CHECK(rows * p.splits < (int64_t(1) << 31), "token_logprobs: too many rows: ", rows);
  dispatch_act(logits.scalar_type(), [&](auto t) {
    using T = decltype(t);
    const unsigned grid = (unsigned)(rows * p.splits);
    if (g_entropy.defined())
      token_logprobs_bwd<T, true><<<grid, kThreads, 0, cur_stream()>>>(p);
    else
      token_logprobs_bwd<T, false><<<grid, kThreads, 0, cur_stream()>>>(p);
    MT_LAUNCH_CHECK();
  });
}

}  // namespace mtorus

// Log probabilities of given tokens, with the entropy of each row and its k likeliest alternatives.
//
//   z = x / tau,  m = max z,  S = sum exp(z - m),  W = sum exp(z - m)(z - m)
//   logp_t = z_t - m - log S,   H = log S - W / S
//   dx_j = (gl (1[j=t] - p_j) - gH p_j (logp_j + H) + sum_i gk_i (1[j=id_i] - p_j)) / tau
//
// Bound by memory: the forward reads the logits once, the backward reads them and writes the gradient.  A row is read by
// a CTA, a cluster of 2 to 8 (where there are fewer rows than the GPU has room for CTAs) or, where it is short, a warp.
// Each thread keeps a running maximum, sum and weighted sum over its 16-byte vectors; shuffles, shared memory and
// distributed shared memory join them.  Exponentials are base 2, in pairs and with one multiply-add per exponent; a
// thread whose values are out of range for that goes over them again with differences to the maximum, subtracted
// before they are scaled, so that a row of the type's lowest values stays uniform.  8192 x 50304 bf16: forward 135 us (with
// the entropy 140 - 150 us; the special-function unit is then busy for most of it), backward 268 us, where the copy's
// rate allows 126 us and 252 us.
//
// The alternatives are picked afterwards, by a second, small kernel.  The first leaves the maxima of small groups of
// neighbouring values.  The k-th largest of them bounds the k-th largest value from below, and only a group whose
// maximum reaches it can hold one of the k: these few groups are read again and their values from the bound on are
// ranked.  Values order by (value, lowest index) as one 64-bit key, so there are no ties.  (2048 x 50257, k = 20: 44 + 17
// us.  In one kernel with the pass over the logits, many rows at once, each step waits for memory behind the loads of
// the other rows on its SM: 67 us.)
#include <cooperative_groups.h>

#include <ATen/cuda/EmptyTensor.h>

#include "decoder_ops.h"
#include "vec.cuh"

namespace mtorus {

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 256;  // of a CTA of the first pass and of the backward
constexpr int kUnroll = 4;     // vectors of a thread in flight
constexpr int kTopThreads = 128;  // of a CTA that picks the alternatives of a row
constexpr int kColumns = 256;
constexpr int kManyWinners = 128;
constexpr int kMaxTop = 64;
constexpr int kHits = 256, kCandidates = 640;
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

// Whole numbers in the order of the values; -0 equals 0 and NaN ranks with -inf.
__device__ __forceinline__ int order_of(float x) {
  const int b = __float_as_int(isnan(x) ? -INFINITY : x);
  return b < 0 ? -(b & 0x7fffffff) : b;
}
// Keys order by value, then by lowest index.
__device__ __forceinline__ long long key_of(float x, int64_t index) {
  return (long long)order_of(x) * 0x100000000ll + (0xffffffffll - index);
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

// The largest value of N vectors.
template <typename T, int N>
__device__ __forceinline__ float largest(const Vec<T, 16 / sizeof(T)> (&v)[N]) {
  if constexpr (sizeof(T) == 2) {
    uint32_t m = reinterpret_cast<const uint32_t*>(&v[0])[0];
#pragma unroll
    for (int i = 1; i < 4 * N; ++i) m = max_pair<T>(m, reinterpret_cast<const uint32_t*>(&v[i / 4])[i % 4]);
    const float2 f = widen_pair<T>(m);
    return fmaxf(f.x, f.y);
  } else {
    float m = v[0].v[0];
#pragma unroll
    for (int i = 1; i < 4 * N; ++i) m = fmaxf(m, v[i / 4].v[i % 4]);
    return m;
  }
}

// A thread's sums over its vectors with few instructions per value: exponents x c - r with the reference r = m c,
// two values at a time. m follows the maximum only when that is 2^8 times likelier, so that hardly any vector after
// the first has to rescale the sums (a warp does when one of its lanes does). r is rounded; that shifts all exponents
// alike and fast_done() takes it out again. For the weighted sum, values are kept at -1e30 or above (fp16: at its
// lowest), so that an exponent is finite and a masked value adds 0 * finite. Good for maxima from -2^26 / c to
// 2^26 / c that lie well above that; fast_done() says so. No value may lie above the reference by more than the slack,
// the lifted ones that come before any other among them: so the reference starts at -2^26 / c, or, where it is higher, at
// the value that masked ones are lifted to (1 each, until the first possible value scales them away).
struct Fast {
  float m, minus_r, limit, best;  // limit: the maximum up to which m stays; best: the maximum
  float2 s, w;
};

constexpr float kFastLimit = 67108864.f;  // 2^26: r is rounded by at most 2
constexpr float kSlack = 8.f;

template <typename T>
__device__ __forceinline__ constexpr float kept_above() {
  return std::is_same_v<T, __half> ? -65504.f : -1e30f;
}

template <typename T, bool ENT>
__device__ __forceinline__ Fast fast_start(float c) {
  const float least = -kFastLimit / c;
  const bool lifted = ENT && kept_above<T>() > least;
  const float m = lifted ? kept_above<T>() : least;
  return Fast{m, lifted ? -(m * c) : kFastLimit, m, -INFINITY, both(0.f), both(0.f)};
}

template <bool ENT>
__device__ __forceinline__ void fast_raise(Fast& a, float vm, float c) {
  const float minus_r = -(vm * c), d = minus_r - a.minus_r, f = ex2(d);
  if (ENT) a.w = mul2(fma2(a.s, both(d), a.w), both(f));
  a.s = mul2(a.s, both(f));
  a.m = vm;
  a.minus_r = minus_r;
  a.limit = vm + kSlack / c;
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
    const float2 t = fma2(x, both(c), both(a.minus_r));
    const float2 e = make_float2(ex2(t.x), ex2(t.y));
    a.s = add2(a.s, e);
    if (ENT) a.w = fma2(e, t, a.w);
  }
}

// The sums relative to the maximum itself; false where the values were out of range, on the way to which the sums may
// have overflowed. The reference only rises, so where it ended in range a NaN in the sums is one among the values.
template <typename T, bool ENT>
__device__ __forceinline__ bool fast_done(const Fast& a, float c, Running& out) {
  const float s = a.s.x + a.s.y, w = a.w.x + a.w.y;
  out = Running{kLowest, 0.f, 0.f};
  if (fabsf(a.minus_r) > kFastLimit) return false;  // above the upper limit
  if (isnan(s)) {
    out.s = s;
    return true;
  }
  if (a.best == -INFINITY) return true;  // nothing, or masked values only
  if (a.best < a.m) return false;        // below the start
  if (ENT && (kept_above<T>() - a.m) * c > -200.f) return false;
  const float d = fmaf(a.m, c, a.minus_r), f = ex2(-d);
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
  int64_t head, vectors, tail0, end;
  __device__ __forceinline__ RowParts(const T* row, int64_t V) : end(V) {
    const int64_t off = (16 - reinterpret_cast<uintptr_t>(row) % 16) % 16 / sizeof(T);
    head = off < V ? off : V;
    vectors = (V - head) / VEC;
    tail0 = head + vectors * VEC;
  }
};

// How the first kernel's maxima cut up a row for the second. A tile is kUnroll vectors for each of 2^threads_log threads,
// thread i's being i, i + 2^threads_log, ...; a group is the vectors of 2^lanes_log neighbouring threads in a tile, or
// (single) one vector.
struct Groups {
  uint32_t stride;  // groups of the row with the most
  int threads_log, lanes_log;
  bool single;
};

// All values -inf: what a thread without a vector takes in its place.
template <typename T>
__device__ __forceinline__ Vec<T, 16 / sizeof(T)> masked_vector() {
  const uint32_t w = std::is_same_v<T, bf16> ? 0xff80ff80u : std::is_same_v<T, __half> ? 0xfc00fc00u : 0xff800000u;
  const uint4 v = make_uint4(w, w, w, w);
  return *reinterpret_cast<const Vec<T, 16 / sizeof(T)>*>(&v);
}

struct FwdParams {
  const void* logits;
  const int64_t* tokens;
  float *logprob, *stats, *entropy;
  float* maxima;  // [rows, groups], or nullptr; -inf for a group without values
  int64_t rows, ld, V;
  float c, inv_tau;
  int cluster;
  Groups groups;
};

struct TopParams {
  const float* maxima;  // as the first kernel's
  float* top_lp;
  int64_t* top_ids;
  float inv_tau;
  int top;
  Groups groups;
};

struct TopShared {
  int4 group[kColumns / 4];  // maxima of columns, or of a few together
  uint4 hit[kHits];             // vectors with a value from the bound on
  int hit_at[kHits];
  long long cand[kCandidates];
  int winners[kColumns];
  int n_hit, n_cand, n_won, floor, larger;
  long long threshold, red[kThreads / 32];
};

// Appends `column` to the winners where `win`.
__device__ __forceinline__ void push_winner(TopShared& ts, bool win, int column) {
  const unsigned all = __ballot_sync(0xffffffffu, win), lane = threadIdx.x & 31;
  int base = 0;
  if (lane == 0 && all != 0) base = atomicAdd(&ts.n_won, __popc(all));
  const int at = __shfl_sync(0xffffffffu, base, 0) + __popc(all & ((1u << lane) - 1));
  if (win) ts.winners[at] = column;
}

// The alternatives of a row, by a CTA of NT threads; m and l2s as in the statistics. The groups c, c + kColumns, ... of
// the row are its column c; a thread looks after columns tid, tid + NT, ...
template <typename T, int NT>
__device__ __forceinline__ void pick_top(const TopParams& p, const T* x, const RowParts<T>& parts, int64_t row, float m,
                                         float l2s, TopShared& ts) {
  constexpr int VEC = 16 / sizeof(T), PER = kColumns / NT;
  constexpr unsigned kAll = 0xffffffffu;
  using V16 = Vec<T, VEC>;
  const int tid = threadIdx.x;
  const V16* xv = reinterpret_cast<const V16*>(x + parts.head);
  static_assert(kUnroll == 4, "the shifts here");
  const int log = p.groups.lanes_log, threads_log = p.groups.threads_log;
  const bool single = p.groups.single;
  const unsigned vectors = (unsigned)parts.vectors;
  const unsigned full = vectors >> (threads_log + 2), rest = vectors - (full << (threads_log + 2));  // tiles, vectors
  const unsigned groups = single ? vectors : (full + (rest != 0)) << (threads_log - log);
  // groups with values, and the columns that hold them
  const unsigned real = single ? vectors
                               : (full << (threads_log - log)) + ((min(rest, 1u << threads_log) + (1u << log) - 1) >> log);
  const int columns = (int)min(real, (unsigned)kColumns);
  int value[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) value[i] = INT_MIN;
  for (unsigned g = tid; g < groups; g += kColumns) {
    const float* most = p.maxima + row * p.groups.stride + g;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (g + i * NT < groups) value[i] = max(value[i], order_of(most[i * NT]));
    }
  }
  int column_log = single ? 0 : 2 + log;  // vectors of a column
  const int group_log = column_log;
  while ((unsigned)kColumns << (column_log - group_log) < groups) ++column_log;
  // the r-th vector of a column, in the order of the row; `vectors` or more for none
  auto vector_of = [&](unsigned column, unsigned r) {
    if (single) return column + r * kColumns;
    const unsigned round = r >> log, g = column + (round >> 2) * kColumns, tile = g >> (threads_log - log);
    return (tile << (threads_log + 2)) + ((round & 3) << threads_log) +
           ((g << log) & ((1u << threads_log) - 1)) + (r & ((1u << log) - 1));
  };
  if (tid == 0) {
    ts.n_hit = ts.n_cand = ts.n_won = ts.larger = 0;
    ts.floor = INT_MAX;
    ts.threshold = kNoKey;  // stays where fewer equal values are left than needed
  }

  // The bound: the k-th largest of the columns' maxima, or, where there are many more columns than that, of the maxima of
  // 2 or 4 columns: fewer comparisons, shared by the threads that hold these columns, for a few more values to rank.
  const int merged = columns >= 6 * p.top ? 4 : columns >= 3 * p.top ? 2 : 1;
  int low = INT_MAX;  // smallest maximum that fewer than k others exceed
  int* list = reinterpret_cast<int*>(ts.group);
  if (merged < PER || (PER == 1 && merged == 1)) {
    int above[PER] = {};
#pragma unroll
    for (int k = 0; k < PER; ++k) list[tid + k * NT] = value[k];
    __syncthreads();
#pragma unroll 4
    for (int i = 0; i < kColumns / 4; ++i) {
      const int4 q = ts.group[i];
#pragma unroll
      for (int k = 0; k < PER; ++k)
        above[k] += (q.x > value[k]) + (q.y > value[k]) + (q.z > value[k]) + (q.w > value[k]);
    }
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      if (value[k] != INT_MIN && above[k] < p.top) low = min(low, value[k]);
    }
  } else {
    const int share = merged / PER;  // threads of a maximum: 1, 2 or 4
    int best = value[0], above = 0;
#pragma unroll
    for (int k = 1; k < PER; ++k) best = max(best, value[k]);
    for (int o = 1; o < share; o *= 2) best = max(best, __shfl_xor_sync(kAll, best, o));
    if (tid % share == 0) list[tid / share] = best;
    __syncthreads();
    const int n = NT / share / share / 4;
    const int4* o = ts.group + tid % share * n;
#pragma unroll 8
    for (int i = 0; i < n; ++i) {
      const int4 q = o[i];
      above += (q.x > best) + (q.y > best) + (q.z > best) + (q.w > best);
    }
    for (int o = 1; o < share; o *= 2) above += __shfl_xor_sync(kAll, above, o);
    if (best != INT_MIN && above < p.top) low = best;
  }
  low = __reduce_min_sync(kAll, low);
  if ((tid & 31) == 0) atomicMin(&ts.floor, low);
  __syncthreads();
  // with fewer columns than alternatives every value counts
  const int floor = columns < p.top ? INT_MIN + 1 : ts.floor;
  long long threshold = columns < p.top ? kNoKey : (long long)floor * 0x100000000ll;
#pragma unroll
  for (int i = 0; i < PER; ++i) push_winner(ts, value[i] >= floor, tid + i * NT);
  __syncthreads();
  int won = ts.n_won;
  if (won > kManyWinners) {
    // Many columns share the bound (equal or masked logits): of these, those with the lowest indexes win.
    long long k[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int column = tid + i * NT;
      k[i] = kNoKey;
      if (value[i] == floor) {
        for (unsigned q = 0; q >> column_log == 0 && k[i] == kNoKey; ++q) {
          const unsigned j = vector_of(column, q);
          if (j >= vectors) continue;
          const V16 v = xv[j];
#pragma unroll
          for (int e = VEC - 1; e >= 0; --e) {
            const float f = to_f<T>(v.v[e]);
            if (order_of(f) == floor) k[i] = key_of(f, parts.head + (int64_t)j * VEC + e);
          }
        }
      }
      ts.cand[column] = k[i];
      const unsigned more = __ballot_sync(kAll, value[i] > floor);
      if ((tid & 31) == 0) atomicAdd(&ts.larger, __popc(more));
    }
    __syncthreads();
    if (tid == 0) ts.n_won = 0;
    const int need = p.top - ts.larger;  // so many of the equal ones
    int r[PER] = {};
    for (int i = 0; i < kColumns; ++i) {
#pragma unroll
      for (int n = 0; n < PER; ++n) r[n] += ts.cand[i] > k[n];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      push_winner(ts, value[i] > floor || (k[i] != kNoKey && r[i] < need), tid + i * NT);
      if (k[i] != kNoKey && r[i] == need - 1) ts.threshold = k[i];
    }
    __syncthreads();
    won = ts.n_won;
    threshold = need > 0 ? ts.threshold : (long long)(floor + 1) * 0x100000000ll;
  }

  const float floor_value = threshold == kNoKey ? -INFINITY : key_value(threshold);
  auto offer = [&](float f, int64_t index) {
    if (f < floor_value) return;
    const long long k = key_of(f, index);
    if (k < threshold) return;
    const int at = atomicAdd(&ts.n_cand, 1);
    if (at < kCandidates) ts.cand[at] = k;
  };
  const int64_t last_equal = key_index(threshold);  // values that equal the bound count up to here
  const unsigned todo = (unsigned)won << column_log;
  for (unsigned i = tid; i < todo; i += kUnroll * NT) {
    V16 v[kUnroll];
    unsigned at[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const unsigned q = i + u * NT;
      at[u] = q < todo ? vector_of(ts.winners[q >> column_log], q & ((1u << column_log) - 1)) : vectors;
      if (at[u] < vectors) v[u] = xv[at[u]];
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (at[u] >= vectors) continue;
      const V16 one[1] = {v[u]};
      const float vm = largest<T>(one);
      if (vm < floor_value || (vm == floor_value && parts.head + (int64_t)at[u] * VEC > last_equal)) continue;
      const int h = atomicAdd(&ts.n_hit, 1);
      if (h >= kHits) continue;
      ts.hit[h] = *reinterpret_cast<const uint4*>(&v[u]);
      ts.hit_at[h] = (int)at[u];
    }
  }
  __syncthreads();
  const int hits = ts.n_hit;
  for (int i = tid; i < min(hits, kHits) * VEC; i += NT)
    offer(to_f<T>(reinterpret_cast<const T*>(ts.hit)[i]), parts.head + (int64_t)ts.hit_at[i / VEC] * VEC + i % VEC);
  // the row's ends, at most 2 (VEC - 1) values
  const int64_t end_at = tid < parts.head ? tid : parts.tail0 + (tid - parts.head);
  const bool end = tid < parts.head + (parts.end - parts.tail0);
  if (end) offer(to_f<T>(x[end_at]), end_at);
  __syncthreads();

  auto put = [&](int i, long long k) {
    p.top_ids[row * p.top + i] = key_index(k);
    p.top_lp[row * p.top + i] = l2s == -INFINITY ? -INFINITY : (key_value(k) - m) * p.inv_tau - l2s * kLn2;
  };
  const int n = ts.n_cand;
  if (hits <= kHits && n <= kCandidates) {
    // each candidate's place is the number of larger ones, which 4 threads count
    const int part = tid & 3;
    for (int i0 = 0; i0 < n; i0 += NT / 4) {
      const int i = i0 + (tid >> 2);
      const long long k = i < n ? ts.cand[i] : kNoKey;
      int r = 0;
#pragma unroll 4
      for (int j = part; j < n; j += 4) r += ts.cand[j] > k;
      r += __shfl_xor_sync(kAll, r, 1);
      r += __shfl_xor_sync(kAll, r, 2);
      if (part == 0 && i < n && r < p.top) put(r, k);
    }
    return;
  }
  // More values above the bound than there is room for: rows whose largest values all lie in a few columns. Takes the
  // largest key below the last one, k times over.
  long long last = LLONG_MAX;
  for (int i = 0; i < p.top; ++i) {
    long long k = kNoKey;
    for (int64_t j = tid; j < parts.vectors; j += NT) {
      const V16 v = xv[j];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const long long q = key_of(to_f<T>(v.v[e]), parts.head + j * VEC + e);
        if (q < last) k = max(k, q);
      }
    }
    if (end) {
      const long long q = key_of(to_f<T>(x[end_at]), end_at);
      if (q < last) k = max(k, q);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) k = max(k, __shfl_xor_sync(kAll, k, o));
    __syncthreads();
    if ((tid & 31) == 0) ts.red[tid >> 5] = k;
    __syncthreads();
    for (int w = 0; w < NT / 32; ++w) k = max(k, ts.red[w]);
    if (tid == 0) put(i, k);
    last = k;
  }
}

template <typename T>
__global__ void __launch_bounds__(kTopThreads, 14)
    token_logprobs_top(const __grid_constant__ TopParams p, const T* logits, int64_t ld, int64_t V, const float* stats) {
  __shared__ TopShared ts;
  const int64_t row = blockIdx.x;
  const T* x = logits + row * ld;
  pick_top<T, kTopThreads>(p, x, RowParts<T>(x, V), row, stats[2 * row], stats[2 * row + 1], ts);
}

enum Top : int { kNoTop, kTopMaxima, kTopHere };

// NT: threads that share a row, a CTA (or one of a cluster) or a warp. TOP: the maxima for the alternatives are written,
// or the alternatives picked at once, by the row's first CTA.
template <typename T, bool ENT, int TOP, int NT>
__global__ void __launch_bounds__(kThreads, NT == 32 ? 4 : TOP == kTopHere ? 2 : 5)
    token_logprobs_fwd(const __grid_constant__ FwdParams p, const __grid_constant__ TopParams top) {
  constexpr int VEC = 16 / sizeof(T), TILE = NT * kUnroll;
  constexpr bool WARP = NT == 32;
  using V16 = Vec<T, VEC>;
  __shared__ Running warps[kThreads / 32];
  __shared__ Running all;
  const int C = WARP ? 1 : p.cluster, rank = WARP ? 0 : blockIdx.x % C;
  const int tid = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int64_t row = WARP ? (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5) : blockIdx.x / C;
  if (WARP && row >= p.rows) return;
  const T* x = static_cast<const T*>(p.logits) + row * p.ld;
  const RowParts<T> parts(x, p.V);
  const V16* xv = reinterpret_cast<const V16*>(x + parts.head);
  int64_t token = -1;
  if (rank == 0 && tid == 0) token = p.tokens[row];  // looked at after the loop: nothing may wait before its loads

  // one pass, a tile after the other
  const int64_t tiles = (parts.vectors + TILE - 1) / TILE;
  Fast sums = fast_start<T, ENT>(p.c);
  auto take = [&](const auto& v) {  // the values of one or more vectors; their maximum
    const float vm = largest<T>(v);
    sums.best = fmaxf(sums.best, vm);
    if (vm > sums.limit) fast_raise<ENT>(sums, vm, p.c);
#pragma unroll
    for (const V16& u : v) fast_add<T, ENT>(sums, u, p.c);
    return vm;
  };
  auto keep = [&](const V16(&v)[kUnroll], int64_t tile, float vm) {  // the tile's maxima
    float* most = p.maxima + row * p.groups.stride;
    if (WARP && p.groups.single) {
      const int64_t j = tile * TILE + tid;
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const V16 one[1] = {v[u]};
        if (j + u * NT < parts.vectors) most[j + u * NT] = fmaxf(-INFINITY, largest<T>(one));
      }
    } else {
      const int lanes = 1 << p.groups.lanes_log;
      vm = fmaxf(-INFINITY, vm);
      for (int o = 1; o < lanes; o *= 2) vm = fmaxf(vm, __shfl_xor_sync(0xffffffffu, vm, o));
      if ((tid & (lanes - 1)) == 0) most[(tile * NT + tid) >> p.groups.lanes_log] = vm;
    }
  };
  int64_t tile = rank;
  for (; (tile + 1) * TILE <= parts.vectors; tile += C) {
    const V16* from = xv + tile * TILE + tid;
    V16 v[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) v[u] = from[u * NT];
    const float vm = take(v);
    if constexpr (TOP != kNoTop) keep(v, tile, vm);
  }
  T token_value = from_f<T>(0.f);
  if (token >= 0 && token < p.V) token_value = x[token];
  if (tile < tiles) {  // the last one, where it is not full
    const int64_t j = tile * TILE + tid;
    V16 v[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) v[u] = j + u * NT < parts.vectors ? xv[j + u * NT] : masked_vector<T>();
    float vm = -INFINITY;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const V16 one[1] = {v[u]};
      if (tile * TILE + u * NT < parts.vectors) vm = fmaxf(vm, take(one));
    }
    if constexpr (TOP != kNoTop) keep(v, tile, vm);
  }
  Running a;
  if (!fast_done<T, ENT>(sums, p.c, a)) {
    for (tile = rank; tile < tiles; tile += C) {
      for (int u = 0; u < kUnroll; ++u) {
        const int64_t j = tile * TILE + u * NT + tid;
        if (j >= parts.vectors) break;
        float f[VEC];
        widen(xv[j], f);
#pragma unroll
        for (int i = 0; i < VEC; ++i) add<ENT>(a, f[i], p.c);
      }
    }
  }
  // the row's ends: at most 2 (VEC - 1) values, one each for the first threads of the row
  const int64_t end_at = tid < parts.head ? tid : parts.tail0 + (tid - parts.head);
  if (rank == 0 && tid < parts.head + (p.V - parts.tail0)) add<ENT>(a, to_f<T>(x[end_at]), p.c);

  a = shuffle_join(a, p.c);
  if constexpr (!WARP) {
    if ((tid & 31) == 0) warps[tid >> 5] = a;
    __syncthreads();
    if (tid < 32) {
      a = tid < kThreads / 32 ? warps[tid] : Running{kLowest, 0.f, 0.f};
      a = shuffle_join(a, p.c);
    }
    if (C > 1) {  // the cluster's first CTA joins what the others hold
      cg::cluster_group cluster = cg::this_cluster();
      if (tid == 0) all = a;
      cluster.sync();
      if (rank == 0 && tid == 0) {
        for (int r = 1; r < C; ++r) join(a, *cluster.map_shared_rank(&all, r), p.c);
      }
      cluster.sync();  // the others' shared memory lives until it has been read
    }
  }
  if (rank != 0) return;
  if (tid == 0) {
    // a row without any possible token has S = 0
    const bool none = a.s == 0.f;
    const float l2s = none ? -INFINITY : log2f(a.s);
    float lp = 0.f;
    if (token >= 0 && token < p.V) lp = none ? -INFINITY : (to_f<T>(token_value) - a.m) * p.inv_tau - l2s * kLn2;
    p.logprob[row] = lp;
    p.stats[2 * row] = a.m;
    p.stats[2 * row + 1] = l2s;
    if (ENT) p.entropy[row] = none ? 0.f : (l2s - a.w / a.s) * kLn2;
    all.m = a.m;
    all.s = l2s;
  }
  if constexpr (TOP == kTopHere) {
    __shared__ TopShared ts;
    __syncthreads();
    pick_top<T, NT>(top, x, parts, row, all.m, all.s, ts);
  }
}

struct BwdParams {
  const void* logits;
  void* dlogits;
  const int64_t *tokens, *top_ids;
  const float *stats, *entropy, *g_logprob, *g_entropy, *g_top;
  int64_t rows, ld, V;
  float c, inv_tau;
  int top, splits;
};

// NT threads share a row: a CTA, or one of `splits` for parts of the row, or a warp.
template <typename T, bool ENT, int NT>
__global__ void __launch_bounds__(kThreads) token_logprobs_bwd(const __grid_constant__ BwdParams p) {
  constexpr int VEC = 16 / sizeof(T);
  constexpr bool WARP = NT == 32;
  using V16 = Vec<T, VEC>;
  const int splits = WARP ? 1 : p.splits, part = WARP ? 0 : blockIdx.x % splits;
  const int tid = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int64_t row = WARP ? (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5) : blockIdx.x / splits;
  if (WARP && row >= p.rows) return;
  const T* x = static_cast<const T*>(p.logits) + row * p.ld;
  T* dx = static_cast<T*>(p.dlogits) + row * p.V;
  const int64_t token = p.tokens[row];
  const bool use = p.g_logprob != nullptr && token >= 0 && token < p.V;
  const float m = p.stats[2 * row], l2s = p.stats[2 * row + 1];
  const float gl = use ? p.g_logprob[row] * p.inv_tau : 0.f;
  const float gh = ENT ? p.g_entropy[row] * p.inv_tau : 0.f;
  const float h = ENT ? p.entropy[row] : 0.f;
  float total = gl;
  bool any = use || gh != 0.f;
  if (p.g_top != nullptr) {
    for (int i = 0; i < p.top; ++i) {
      const float g = p.g_top[row * p.top + i];
      any = any || g != 0.f;
      total += g * p.inv_tau;
    }
  }
  // No gradient: no possible token, or an ignored one and nothing else comes in (then the logits may be anything, such as
  // NaN in the rows that pad a batch).
  const bool none = l2s == -INFINITY || !any;
  auto grad = [&](float v) {
    const float t = max_nan(fmaf(v - m, p.c, -l2s), -200.f);  // log2 of the probability
    const float e = ex2(t);
    return none ? 0.f : ENT ? -e * fmaf(gh, fmaf(t, kLn2, h), total) : -e * total;
  };
  // the gradient has no stride of its own: its rows may lie on other 16-byte offsets than the logits'
  const bool same = (reinterpret_cast<uintptr_t>(x) - reinterpret_cast<uintptr_t>(dx)) % 16 == 0;
  const RowParts<T> parts(x, p.V);
  const int64_t step = (int64_t)NT * splits, first = (int64_t)part * NT + tid;
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
  if (WARP)
    __syncwarp();
  else
    __syncthreads();
  for (int i = tid; i <= (p.g_top != nullptr ? p.top : 0); i += NT) {
    const int64_t id = i == 0 ? token : p.top_ids[row * p.top + i - 1];
    if (i == 0 && !use) continue;
    const int64_t owner = id < parts.head ? id
                          : id >= parts.tail0 ? parts.head + id - parts.tail0
                                              : (id - parts.head) / VEC % step;
    if (owner / NT != part) continue;
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

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Short rows leave most of a CTA idle, so a warp takes each, where there are enough of them.
bool warp_per_row(int64_t rows, int64_t vectors) { return vectors <= 512 && rows >= 2 * num_sms(); }

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
  p.ld = rows > 1 ? logits.stride(0) : V;
  p.V = V;
  p.inv_tau = (float)inv_tau;
  p.c = (float)(inv_tau * 1.4426950408889634);
  p.rows = rows;
  const int64_t vectors = V * logits.element_size() / 16;
  const bool warp = warp_per_row(rows, vectors);
  const int64_t threads = warp ? 32 : kThreads, tiles = std::max<int64_t>(1, ceil_div(vectors, threads * kUnroll));
  // Clusters while all CTAs are resident at once (5 on an SM) and each has a tile: 257 x 131072 fp32 45 us with one
  // CTA for a row, 33 us with two, 37 us with four; 4 x 50304 bf16 6.6, 5.5, 4.7 and (eight) 4.2 us.
  int C = 1;
  while (!warp && C < 8 && rows * C * 2 <= 5 * num_sms() && tiles > C) C *= 2;
  p.cluster = C;
  MT_CHECK(rows * C < (int64_t(1) << 31), "token_logprobs: too many rows: ", rows);
  at::Tensor maxima;
  if (top > 0) {
    // groups as large as leave 128 at least in a long row; in a short one single vectors where there are too few others
    Groups& g = p.groups;
    g.threads_log = warp ? 5 : 8;
    while (g.lanes_log < 5 && tiles * threads >> g.lanes_log > kColumns) ++g.lanes_log;
    g.single = warp && tiles * threads < 3 * top;
    g.stride = (uint32_t)(g.single ? std::max<int64_t>(1, vectors) : tiles * threads >> g.lanes_log);
    maxima = at::Tensor(at::detail::empty_cuda({rows, (int64_t)g.stride}, at::kFloat, logits.device(), c10::nullopt));
    p.maxima = maxima.data_ptr<float>();
  }
  // With a CTA or less on each SM the alternatives are picked where the row was read: a launch less (4 x 50304 bf16,
  // k = 8: 6.6 us on the device, as two kernels 7.8 us, and 3.5 us less on the host). With more, they would wait behind the other rows' loads.
  const bool here = top > 0 && !warp && rows * C <= num_sms();
  TopParams q{p.maxima, nullptr, nullptr, p.inv_tau, (int)top, p.groups};
  if (top > 0) {
    q.top_lp = top_lp.data_ptr<float>();
    q.top_ids = top_ids.data_ptr<int64_t>();
  }
  auto launch = [&](auto kernel) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(warp ? ceil_div(rows, kThreads / 32) : rows * C));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = cur_stream();
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)C;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = C > 1 ? 1 : 0;
    C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, p, q));
    MT_LAUNCH_CHECK();
  };
  dispatch_act(logits.scalar_type(), [&](auto t) {
    using T = decltype(t);
    const bool ent = entropy.defined();
    auto with = [&](auto nt, auto what) {
      constexpr int NT = decltype(nt)::value, TOP = decltype(what)::value;
      if (ent)
        launch(token_logprobs_fwd<T, true, TOP, NT>);
      else
        launch(token_logprobs_fwd<T, false, TOP, NT>);
    };
    using std::integral_constant;
    if (warp && top > 0)
      with(integral_constant<int, 32>{}, integral_constant<int, kTopMaxima>{});
    else if (warp)
      with(integral_constant<int, 32>{}, integral_constant<int, kNoTop>{});
    else if (here)
      with(integral_constant<int, kThreads>{}, integral_constant<int, kTopHere>{});
    else if (top > 0)
      with(integral_constant<int, kThreads>{}, integral_constant<int, kTopMaxima>{});
    else
      with(integral_constant<int, kThreads>{}, integral_constant<int, kNoTop>{});
    if (top == 0 || here) return;
    token_logprobs_top<T><<<(unsigned)rows, kTopThreads, 0, cur_stream()>>>(q, static_cast<const T*>(p.logits), p.ld, V,
                                                                          p.stats);
    MT_LAUNCH_CHECK();
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
  p.rows = rows;
  const int64_t vectors = V * logits.element_size() / 16;
  const bool warp = warp_per_row(rows, vectors);
  p.splits = 1;
  while (!warp && rows * p.splits < 4 * num_sms() && vectors > (int64_t)kThreads * p.splits) p.splits *= 2;
  MT_CHECK(rows * p.splits < (int64_t(1) << 31), "token_logprobs: too many rows: ", rows);
  dispatch_act(logits.scalar_type(), [&](auto t) {
    using T = decltype(t);
    const unsigned grid = (unsigned)(warp ? ceil_div(rows, kThreads / 32) : rows * p.splits);
    auto with = [&](auto nt) {
      constexpr int NT = decltype(nt)::value;
      if (g_entropy.defined())
        token_logprobs_bwd<T, true, NT><<<grid, kThreads, 0, cur_stream()>>>(p);
      else
        token_logprobs_bwd<T, false, NT><<<grid, kThreads, 0, cur_stream()>>>(p);
      MT_LAUNCH_CHECK();
    };
    if (warp)
      with(std::integral_constant<int, 32>{});
    else
      with(std::integral_constant<int, kThreads>{});
  });
}

}  // namespace mtorus

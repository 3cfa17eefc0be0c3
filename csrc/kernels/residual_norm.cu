// Residual update of a block with its norms, in one pass each way:
//   rh = 1/sqrt(mean h^2 + eps),  b = h rh post,   y = beta x + alpha g b     (post norm, gate, scales)
//   ry = 1/sqrt(mean y^2 + eps),  n = y ry pre                               (pre norm of the next block)
// Backward, with u = dn pre, yh = y ry, hh = h rh and e = alpha g post (a gate per row stays out of e, as r):
//   Y = dy + ry (u - yh mean(u yh));  dx = beta Y;  dg = alpha b Y;  dpre = sum dn yh;  dpost = sum alpha g Y hh
//   dh = rh (r e Y - hh mean(r e hh Y))
// y is computed again from x and h in 32 bits (reading x instead of y costs the same bytes), so the statistics
// and the weight gradients see the value before its rounding.
//
// Bound by memory: forward 2 reads and 2 writes of [T, d], backward 4 and 2.  One CTA of d / 8 threads (or
// d / 16) walks a strided set of rows; a thread owns the same 8 (16) columns of every row, so the weights and the sums
// of weight gradients stay in its registers.  Its vectors of the next rows are on their way through a ring in shared memory;
// each thread reads back only what it copied itself, so the ring needs no barrier. Rows of up to 128 columns (the norm
// of a head) share a warp.
//
// The backward needs little more than the memory's time in instructions, so it is written to need few: one row
// reduction, not two (mean(e hh Y) follows from sums of e hh with dy + ry u and with yh), one column sum q = sum r Y hh for
// both dpost = alpha g q and dgate = alpha post q, pairs of values per instruction, and 6 shuffles for 3 row sums.
//
// 16384 x 2048 bf16, both norms and a gate per channel: forward 45 us (a bare stream of its reads and writes takes as
// long), backward 71 us (63 us) and 4.5 us for the weights' sums; the copy's rate allows 41 us and 62 us.
#include <ATen/cuda/EmptyTensor.h>

#include "decoder_ops.h"
#include "vec.cuh"

namespace mtorus {

namespace {

constexpr int kMaxWarps = 32;
constexpr int kSmemBudget = 200 * 1024;  // of 227 KB per SM: the CTAs' static part and the system's 1 KB each fit too

// Tensors that are read row by row.
enum In : int { kX = 0, kH = 1, kGate = 2, kDy = 3, kDn = 4, kIns = 5 };

struct NormParams {
  const void* in[kIns];  // nullptr: not there
  uint32_t ld[kIns];
  int slot[kIns];  // where an input lies in a row's slots, bytes
  const float *pre, *post, *gate;  // gate: per channel or per row
  void *y, *n, *dx, *dh, *dgate;
  float *rstd_h, *rstd_y, *part;
  uint32_t rows;
  int d, gate_kind, depth, stage;  // ring: rows in flight, bytes of one row's slots
  float beta, alpha, eps;
  bool want_dpre, want_q;
};

// How rows are read and written. kAligned: all start on 16 bytes, so that a thread takes vectors. kShifted: all tensors'
// rows lie alike, but off 16 bytes; a CTA whose rows are a multiple of 16 / sizeof(T) rows apart sees the same offset in
// each, takes the vectors that cover its rows, and leaves what lies before and behind them alone. kSingle: anything else,
// value by value.
enum Mode : int { kSingle, kAligned, kShifted };

// Place in its row, counted from the first vector's start, of a thread's i-th value in a group of 256: vectors, or single
// values 32 apart, so that each load of the warp is contiguous. LANES < 32: lanes of a warp that share a row of at most
// 8 LANES columns, in one group.
template <typename T, int MODE, int LANES>
__device__ __forceinline__ int place_of(int group, int lane, int i) {
  constexpr int VEC = 16 / sizeof(T);
  if constexpr (MODE == kSingle) return group * 256 + i * 32 + lane;
  return group * 256 + (i / VEC) * (LANES * VEC) + lane * VEC + i % VEC;
}

// The rows that a thread has asked for, and their values. The slots of one row lie one input after another, each
// with one 16-byte vector of every thread after the other. INPUTS: a bit for each input, or 0 where the kernel looks
// at its parameters for which ones there are.
template <typename T, int MODE, int NG, int LANES, unsigned INPUTS>
struct Rows {
  static_assert(LANES == 32 || (MODE == kAligned && NG == 1), "several rows to a warp");
  static constexpr int VEC = 16 / sizeof(T), NV = 8 / VEC, PER = 32 / LANES;  // PER: rows at a time
  const NormParams& p;
  const unsigned char* mine;  // this thread's first vector in the ring
  uint32_t address;           // the same as a shared-memory address
  int lane, g0, pitch;        // pitch: from a thread's vector to its next
  int shift;                  // kShifted: values of the first vector that lie before the row

  __device__ __forceinline__ Rows(const NormParams& p, const unsigned char* ring)
      : p(p),
        mine(ring + threadIdx.x * 16),
        address(static_cast<uint32_t>(__cvta_generic_to_shared(mine))),
        lane(threadIdx.x & (LANES - 1)),
        g0((threadIdx.x >> 5) * NG),
        pitch(blockDim.x * 16),
        shift(MODE == kShifted ? (int)((uint64_t)blockIdx.x * p.d % VEC) : 0) {}

  // column of a thread's i-th value; below 0 or from d on: none
  __device__ __forceinline__ int column(int g, int i) const { return place_of<T, MODE, LANES>(g0 + g, lane, i) - shift; }

  // the CTA's first rows, and from one set of rows to the next; `mine`: the thread's row of a set, which may lie behind
  // the last one where PER > 1
  __device__ __forceinline__ uint32_t first() const { return blockIdx.x * PER; }
  __device__ __forceinline__ uint32_t step() const { return gridDim.x * PER; }
  __device__ __forceinline__ uint32_t mine_of(uint32_t set) const {
    return LANES == 32 ? set : set + (threadIdx.x & 31) / LANES;
  }
  __device__ __forceinline__ bool there(uint32_t row) const { return LANES == 32 || row < p.rows; }
  __device__ __forceinline__ bool leads(uint32_t row) const {  // the thread that writes the row's scalars
    return LANES == 32 ? threadIdx.x == 0 : lane == 0 && row < p.rows;
  }

  __device__ __forceinline__ bool has(int t) const { return INPUTS != 0 ? INPUTS >> t & 1 : p.in[t] != nullptr; }

  __device__ __forceinline__ const T* row_of(int t, uint32_t row) const {
    return static_cast<const T*>(p.in[t]) + (uint64_t)row * p.ld[t];
  }

  __device__ __forceinline__ void ask(uint32_t row, int stage) const {
    if constexpr (MODE != kSingle) {
      if (LANES < 32 || row < p.rows) {
#pragma unroll
        for (int t = 0; t < kIns; ++t) {
          if (!has(t)) continue;
          // a row that is not there is zeros, so that the other rows' column sums stay clean
          const T* src = row_of(t, there(row) ? row : 0) - shift;
#pragma unroll
          for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int k = 0; k < NV; ++k) {
              // what lies behind the row is not read: zeros take its place
              const int at = place_of<T, MODE, LANES>(g0 + g, lane, k * VEC),
                        left = there(row) ? p.d + shift - at : 0;
              const int bytes = MODE == kAligned ? (left > 0 ? 16 : 0) : max(0, min(16, left * (int)sizeof(T)));
              copy_async16(address + stage * p.stage + p.slot[t] + (g * NV + k) * pitch, src + (left > 0 ? at : 0),
                           bytes);
            }
        }
      }
      copy_async_commit();
    }
  }

  // the 8 values of group g as pairs; 0 beyond d and where the input is not there
  __device__ __forceinline__ void get(int input, uint32_t row, int stage, int g, float2 (&f)[4]) const {
    if (!has(input)) {
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = both(0.f);
    } else if constexpr (MODE != kSingle) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const uint4 w = *reinterpret_cast<const uint4*>(mine + stage * p.stage + p.slot[input] + (g * NV + k) * pitch);
        if constexpr (sizeof(T) == 2) {
          f[0] = widen_pair<T>(w.x);
          f[1] = widen_pair<T>(w.y);
          f[2] = widen_pair<T>(w.z);
          f[3] = widen_pair<T>(w.w);
        } else {
          f[2 * k] = make_float2(__uint_as_float(w.x), __uint_as_float(w.y));
          f[2 * k + 1] = make_float2(__uint_as_float(w.z), __uint_as_float(w.w));
        }
      }
      if (MODE == kShifted && column(g, 0) < 0) {  // what lies before the row
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          if (column(g, i) < 0) (i & 1 ? f[i / 2].y : f[i / 2].x) = 0.f;
        }
      }
    } else {
      const T* src = row_of(input, row);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = column(g, i);
        const float v = c < p.d ? to_f<T>(src[c]) : 0.f;
        if (i & 1)
          f[i / 2].y = v;
        else
          f[i / 2].x = v;
      }
    }
  }

  __device__ __forceinline__ void put(void* out, uint32_t row, int g, const float2 (&f)[4]) const {
    T* dst = static_cast<T*>(out) + (uint64_t)row * (uint32_t)p.d;
    if constexpr (MODE != kSingle) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = column(g, k * VEC);
        uint4 w;
        if constexpr (sizeof(T) == 2) {
          w = make_uint4(narrow_pair<T>(f[0]), narrow_pair<T>(f[1]), narrow_pair<T>(f[2]), narrow_pair<T>(f[3]));
        } else {
          w = make_uint4(__float_as_uint(f[2 * k].x), __float_as_uint(f[2 * k].y), __float_as_uint(f[2 * k + 1].x),
                         __float_as_uint(f[2 * k + 1].y));
        }
        if (MODE == kAligned ? c < p.d && there(row) : c >= 0 && c + VEC <= p.d) {
          __stcs(reinterpret_cast<uint4*>(dst + c), w);
        } else if (MODE == kShifted) {  // the row's ends
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            if (c + i >= 0 && c + i < p.d) dst[c + i] = reinterpret_cast<const T*>(&w)[i];
          }
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = column(g, i);
        if (c < p.d) dst[c] = from_f<T>(i & 1 ? f[i / 2].y : f[i / 2].x);
      }
    }
  }

  // fp32 weights [d]; `none` where there are none or beyond d
  __device__ __forceinline__ void weight(const float* w, int g, float none, float2 (&f)[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c0 = column(g, 2 * i), c1 = column(g, 2 * i + 1);
      f[i].x = w != nullptr && c0 >= 0 && c0 < p.d ? w[c0] : none;
      f[i].y = w != nullptr && c1 >= 0 && c1 < p.d ? w[c1] : none;
    }
  }

  // e = alpha g post without a gate per row or per element
  __device__ __forceinline__ void branch_weight(int g, float2 (&e)[4]) const {
    float2 w[4];
    weight(p.post, g, 1.f, e);
    weight(p.gate_kind == kGateChannel ? p.gate : nullptr, g, 1.f, w);
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = mul2(mul2(e[i], w[i]), both(p.alpha));
  }
};

// Sum of one value over the CTA (LANES < 32: over the lanes of a row) for every thread. `red` holds [2][kMaxWarps]
// floats; `par` alternates between its halves, so that one barrier per call is enough.
template <int LANES>
__device__ __forceinline__ float cta_sum(float v, float* red, int& par) {
  if constexpr (LANES < 32) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  }
  v = warp_sum(v);
  const int nw = blockDim.x >> 5, lane = threadIdx.x & 31;
  if (nw == 1) return v;
  float* r = red + par * kMaxWarps;
  par ^= 1;
  if (lane == 0) r[threadIdx.x >> 5] = v;
  __syncthreads();
  return warp_sum(lane < nw ? r[lane] : 0.f);
}

// The same for three values; `red` holds [2][kMaxWarps] float4. Halves and quarters of the warp first share the values
// out among them, so that 6 shuffles do; then a lane adds one value of every 8th warp.
template <int LANES>
__device__ __forceinline__ float3 cta_sum3(float3 v, float4* red, int& par) {
  constexpr unsigned kAll = 0xffffffffu;
  if constexpr (LANES < 32) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
      v.x += __shfl_xor_sync(kAll, v.x, o);
      v.y += __shfl_xor_sync(kAll, v.y, o);
      v.z += __shfl_xor_sync(kAll, v.z, o);
    }
    return v;
  }
  const int lane = threadIdx.x & 31;
  const bool up = lane & 16, odd = lane & 8;
  const float a = (up ? v.z : v.x) + __shfl_xor_sync(kAll, up ? v.x : v.z, 16);
  const float b = v.y + __shfl_xor_sync(kAll, v.y, 16);
  float s = (odd ? b : a) + __shfl_xor_sync(kAll, odd ? a : b, 8);
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) s += __shfl_xor_sync(kAll, s, o);
  // lanes 0, 8, 16 hold the sums of x, y, z
  const int nw = blockDim.x >> 5;
  int step = 8;
  if (nw > 1) {
    float* r = reinterpret_cast<float*>(red + par * kMaxWarps);
    par ^= 1;
    if ((lane & 7) == 0) r[(threadIdx.x >> 5) * 4 + (lane >> 3)] = s;
    __syncthreads();
    s = 0.f;
    for (int i = lane; i < 4 * nw; i += 32) s += r[i];
#pragma unroll
    for (int o = 16; o > 2; o >>= 1) s += __shfl_xor_sync(kAll, s, o);
    step = 1;  // lanes 0, 1, 2
  }
  return make_float3(__shfl_sync(kAll, s, 0), __shfl_sync(kAll, s, step), __shfl_sync(kAll, s, 2 * step));
}

// ALL: there are a branch and a pre norm, and no gate per element -- what a training step calls; with this known, and
// the rest done by arithmetic (no post norm is rh = 1), a row takes two thirds of the instructions.
template <typename T, int MODE, int NG, int LANES, bool ALL, int MAXT, int MINB>
__global__ void __launch_bounds__(MAXT, MINB) residual_norm_fwd(const __grid_constant__ NormParams p) {
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ float red[2 * kMaxWarps];
  const Rows<T, MODE, NG, LANES, ALL ? 1u << kX | 1u << kH : 0u> in(p, ring);
  const float inv_d = 1.f / p.d;
  const bool branch = in.has(kH);
  int par = 0, stage = 0;
  float2 e[NG][4], pre[NG][4];
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    in.branch_weight(g, e[g]);
    in.weight(p.pre, g, 0.f, pre[g]);
  }
  float gates = 1.f;  // of the CTA's next 32 rows, one row per lane
  int turn = 0;
  for (int k = 0; k < p.depth - 1; ++k) in.ask(in.mine_of(in.first() + k * in.step()), k);
  for (uint32_t set = in.first(); set < p.rows; set += in.step()) {
    const uint32_t row = in.mine_of(set);
    in.ask(row + (p.depth - 1) * in.step(), stage == 0 ? p.depth - 1 : stage - 1);
    float gate = 1.f;
    if (p.gate_kind == kGateRow) {
      const uint64_t mine = row + (uint64_t)in.lane * in.step();
      if (turn == 0 && mine < p.rows) gates = p.gate[mine];
      gate = __shfl_sync(0xffffffffu, gates, turn, LANES);
      turn = (turn + 1) & (LANES - 1);
    }
    if constexpr (MODE != kSingle) copy_async_wait(p.depth - 1);
    float2 y[NG][4];
    if (branch) {
      float rh = 1.f;
#pragma unroll
      for (int g = 0; g < NG; ++g) in.get(kH, row, stage, g, y[g]);
      if (p.post != nullptr) {
        float2 s = both(0.f);
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
          for (int i = 0; i < 4; ++i) s = fma2(y[g][i], y[g][i], s);
        rh = rsqrtf(cta_sum<LANES>(s.x + s.y, red, par) * inv_d + p.eps);
        if (in.leads(row) && p.rstd_h != nullptr) p.rstd_h[row] = rh;
      }
      const float2 r = both(rh * gate), beta = both(p.beta);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float2 x[4];
        in.get(kX, row, stage, g, x);
#pragma unroll
        for (int i = 0; i < 4; ++i) y[g][i] = mul2(y[g][i], e[g][i]);
        if (!ALL && p.gate_kind == kGateFull) {
          float2 w[4];
          in.get(kGate, row, stage, g, w);
#pragma unroll
          for (int i = 0; i < 4; ++i) y[g][i] = mul2(y[g][i], w[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) y[g][i] = fma2(y[g][i], r, mul2(x[i], beta));
        in.put(p.y, row, g, y[g]);
      }
    } else {
#pragma unroll
      for (int g = 0; g < NG; ++g) in.get(kX, row, stage, g, y[g]);
    }
    if (ALL || p.n != nullptr) {
      float2 s = both(0.f);
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) s = fma2(y[g][i], y[g][i], s);
      const float ry = rsqrtf(cta_sum<LANES>(s.x + s.y, red, par) * inv_d + p.eps);
      if (in.leads(row) && p.rstd_y != nullptr) p.rstd_y[row] = ry;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
#pragma unroll
        for (int i = 0; i < 4; ++i) y[g][i] = mul2(mul2(y[g][i], both(ry)), pre[g][i]);
        in.put(p.n, row, g, y[g]);
      }
    }
    stage = stage + 1 == p.depth ? 0 : stage + 1;
  }
  if constexpr (MODE != kSingle) copy_async_wait(0);
}

// part: [gridDim.x][2][d], the CTA's sums of dn yh (dpre) and of r Y hh (q; with the gate of each element)
// ALL: as in the forward, and both gradients come in and both are wanted.
template <typename T, int MODE, int NG, int LANES, bool ALL, int MAXT, int MINB>
__global__ void __launch_bounds__(MAXT, MINB) residual_norm_bwd(const __grid_constant__ NormParams p) {
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ float4 red[2 * kMaxWarps];
  const Rows<T, MODE, NG, LANES, ALL ? 1u << kX | 1u << kH | 1u << kDy | 1u << kDn : 0u> in(p, ring);
  const float inv_d = 1.f / p.d;
  const bool branch = in.has(kH), full = !ALL && p.gate_kind == kGateFull, post = p.post != nullptr;
  int par = 0, stage = 0;
  float2 e[NG][4], pre[NG][4], sum_pre[NG][4], sum_q[NG][4];
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    in.branch_weight(g, e[g]);
    in.weight(in.has(kDn) ? p.pre : nullptr, g, 0.f, pre[g]);
#pragma unroll
    for (int i = 0; i < 4; ++i) sum_pre[g][i] = sum_q[g][i] = both(0.f);
  }
  // rstd and gate of the CTA's next 32 rows, one row per lane. Loads queue up behind the copies in flight, so one for
  // each row would be late each time: 81 us against 73 us at 16384 x 2048 bf16.
  float rhs = 1.f, rys = 0.f, gates = 1.f;
  int turn = 0;
  for (int k = 0; k < p.depth - 1; ++k) in.ask(in.mine_of(in.first() + k * in.step()), k);
  for (uint32_t set = in.first(); set < p.rows; set += in.step()) {
    const uint32_t row = in.mine_of(set);
    in.ask(row + (p.depth - 1) * in.step(), stage == 0 ? p.depth - 1 : stage - 1);
    if (turn == 0) {
      const uint64_t mine = row + (uint64_t)in.lane * in.step();
      if (mine < p.rows) {
        if (post) rhs = p.rstd_h[mine];
        if (in.has(kDn)) rys = p.rstd_y[mine];
        if (p.gate_kind == kGateRow) gates = p.gate[mine];
      }
    }
    constexpr unsigned kAll = 0xffffffffu;
    const float rh = __shfl_sync(kAll, rhs, turn, LANES), ry = __shfl_sync(kAll, rys, turn, LANES),
                gate = __shfl_sync(kAll, gates, turn, LANES);
    turn = (turn + 1) & (LANES - 1);
    if constexpr (MODE != kSingle) copy_async_wait(p.depth - 1);
    float2 hh[NG][4], yh[NG][4], t[NG][4];  // t = dy + ry u, so that Y = t - ry yh mean(u yh)
    // sums of u yh, and of c = e hh with t and yh
    float2 s0 = both(0.f), s1 = both(0.f), s2 = both(0.f);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      in.get(kX, row, stage, g, yh[g]);
      in.get(kH, row, stage, g, hh[g]);
      float2 c[4], u[4];
      in.get(kDy, row, stage, g, t[g]);
      in.get(kDn, row, stage, g, u);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        hh[g][i] = mul2(hh[g][i], both(rh));
        c[i] = mul2(hh[g][i], e[g][i]);
      }
      if (full) {
        float2 w[4];
        in.get(kGate, row, stage, g, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = mul2(c[i], w[i]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        yh[g][i] = mul2(fma2(c[i], both(gate), mul2(yh[g][i], both(p.beta))), both(ry));
        sum_pre[g][i] = fma2(u[i], yh[g][i], sum_pre[g][i]);
        u[i] = mul2(u[i], pre[g][i]);
        s0 = fma2(u[i], yh[g][i], s0);
        t[g][i] = fma2(u[i], both(ry), t[g][i]);
        s1 = fma2(c[i], t[g][i], s1);
        s2 = fma2(c[i], yh[g][i], s2);
      }
    }
    const float3 s = cta_sum3<LANES>(make_float3(s0.x + s0.y, s1.x + s1.y, s2.x + s2.y), red, par);
    const float rm = ry * s.x * inv_d;
    const float cy = s.y - rm * s.z;  // sum of c Y
    if (p.gate_kind == kGateRow && p.dgate != nullptr && in.leads(row)) static_cast<float*>(p.dgate)[row] = cy;
    // without a post norm rh is 1 and dh has no mean
    const float2 minus_rm = both(-rm), minus_k = both(post ? -rh * gate * cy * inv_d : 0.f), r = both(rh * gate);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float2 o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        t[g][i] = fma2(yh[g][i], minus_rm, t[g][i]);  // Y
        o[i] = mul2(t[g][i], both(p.beta));
      }
      if (ALL || p.dx != nullptr) in.put(p.dx, row, g, o);
      if (!branch) continue;
      if (full) {
        float2 w[4];
        if (p.dgate != nullptr) {
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i] = mul2(mul2(hh[g][i], e[g][i]), t[g][i]);
          in.put(p.dgate, row, g, o);
        }
        in.get(kGate, row, stage, g, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) t[g][i] = mul2(t[g][i], w[i]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sum_q[g][i] = fma2(mul2(t[g][i], both(gate)), hh[g][i], sum_q[g][i]);
        o[i] = fma2(hh[g][i], minus_k, mul2(mul2(t[g][i], e[g][i]), r));
      }
      if (ALL || p.dh != nullptr) in.put(p.dh, row, g, o);
    }
    stage = stage + 1 == p.depth ? 0 : stage + 1;
  }
  if constexpr (MODE != kSingle) copy_async_wait(0);
  if (p.part == nullptr) return;
  if constexpr (LANES < 32) {
#pragma unroll
    for (int o = 16; o >= LANES; o >>= 1)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        for (float2* v : {&sum_pre[0][i], &sum_q[0][i]}) {
          v->x += __shfl_xor_sync(0xffffffffu, v->x, o);
          v->y += __shfl_xor_sync(0xffffffffu, v->y, o);
        }
      }
    if ((threadIdx.x & 31) >= LANES) return;
  }
  float* part = p.part + (int64_t)blockIdx.x * 2 * p.d;
#pragma unroll
  for (int g = 0; g < NG; ++g)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = in.column(g, i);
      if (c < 0 || c >= p.d) continue;
      if (p.want_dpre) part[c] = i & 1 ? sum_pre[g][i / 2].y : sum_pre[g][i / 2].x;
      if (p.want_q) part[p.d + c] = i & 1 ? sum_q[g][i / 2].y : sum_q[g][i / 2].x;
    }
}

// Sums the CTAs' parts in a fixed order, one CTA for COLS columns: dpre, or q and from it dpost = alpha g q and
// dgate = alpha post q. Bound by the latency of its loads: 8 columns to a CTA where there are few (131072 x 64 bf16
// 5.1 us, with 32 10 us; 16727 x 1003 4.6 and 5.6 us), 32 for wide rows (16384 x 2048 4.5 us, with 8 6.7 us).
constexpr int kFinishThreads = 1024;
template <int COLS>
__global__ void __launch_bounds__(kFinishThreads)
    residual_norm_finish(const float* part, int parts, int d, bool first, float alpha, const float* gate,
                         const float* post, float* dpre, float* dpost, float* dgate) {
  constexpr int kWarps = kFinishThreads / 32;
  __shared__ float sm[kWarps][COLS];
  const bool is_pre = first && blockIdx.y == 0;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * COLS + threadIdx.x % COLS;
  float t = 0.f;
  if (c < d) {
    const float* col = part + (is_pre ? 0 : d) + c;
#pragma unroll 4
    for (int b = threadIdx.x / COLS; b < parts; b += kFinishThreads / COLS) t += col[(int64_t)b * 2 * d];
  }
#pragma unroll
  for (int o = 16; o >= COLS; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  if (lane < COLS) sm[w][lane] = t;
  __syncthreads();
  if (threadIdx.x >= COLS || c >= d) return;
#pragma unroll
  for (int k = 1; k < kWarps; ++k) t += sm[k][lane];
  if (is_pre) {
    dpre[c] = t;
  } else {
    if (dpost != nullptr) dpost[c] = alpha * (gate != nullptr ? gate[c] : 1.f) * t;
    if (dgate != nullptr) dgate[c] = alpha * (post != nullptr ? post[c] : 1.f) * t;
  }
}

struct Shape {
  Mode mode;
  int threads, groups, ins, lanes;
};

constexpr int kWide = 17;  // 256-column groups of a row; more do not fit the registers of a CTA's threads otherwise

// Whether a thread of the backward for known inputs takes two groups of an aligned row. Its registers allow 8 warps on
// an SM: with a barrier for every row, 8 warps that do more each beat 16 (16384 x 2048 bf16 71.4 us against 73.5 us,
// 4096 x 4096 40.3 us against 42 us, 9362 x 1792 41.6 us against 43.2 us), but not where whole CTAs leave 2 or more of
// the 8 empty (13107 x 1280 49.5 us against 41.6 us, 7281 x 2304 56 us against 52.5 us). In 32 bits they are as fast or
// faster at every width, by up to 13 % (16256 x 1032 67 us against 78 us). The kernel for any set of inputs needs too
// many registers for it (8192 x 2048 with a gate per element 64 us against 57 us).
bool two_groups(int groups, int esize) {
  const int warps = (groups + 1) / 2;
  return groups >= 5 && (esize == 4 || 8 / warps * warps >= 7);
}

// pairs: two groups for a thread also where two_groups() says so.
Shape shape_of(const NormParams& p, int esize, bool pairs) {
  const int v = 16 / esize;
  bool ok = true;
  int ins = 0;
  for (int t = 0; t < kIns; ++t) {
    if (p.in[t] == nullptr) continue;
    ok = ok && reinterpret_cast<uintptr_t>(p.in[t]) % 16 == 0 && (p.rows == 1 || (p.ld[t] + v - p.d % v) % v == 0);
    ++ins;
  }
  for (const void* q : {p.y, p.n, p.dx, p.dh}) ok = ok && reinterpret_cast<uintptr_t>(q) % 16 == 0;
  if (p.gate_kind == kGateFull) ok = ok && reinterpret_cast<uintptr_t>(p.dgate) % 16 == 0;
  Shape s{!ok ? kSingle : p.d % v == 0 ? kAligned : kShifted, 0, 0, ins, 32};
  const int per = (p.d + (s.mode == kShifted ? v - 1 : 0) + 255) / 256;
  s.groups = per >= kWide || (pairs && s.mode == kAligned && two_groups(per, esize)) ? 2 : 1;
  s.threads = (per + s.groups - 1) / s.groups * 32;
  // a row has to fit into the ring, and into a CTA
  if (s.mode != kSingle && (ins * s.groups * s.threads * 8 * esize > kSmemBudget || s.threads > 1024)) {
    s.mode = kSingle;
    s.threads = std::min(s.threads, 1024);
  }
  // Several short rows to a warp: 131072 x 64 bf16 11.8 and 16.5 us, with one each 34 and 50 us; x 128 23.5 and 38 us,
  // with one each 34.5 and 51 us.
  if (s.mode == kAligned && p.d <= 128) s.lanes = p.d <= 64 ? 8 : 16;
  return s;
}

// f(MODE, NG, LANES, ALL, MAXT): the kernel for CTAs of up to MAXT threads, so that small ones get more registers.
// PAIRS: shape_of()'s `pairs` where `all`. Without it two groups mean 9 warps at least, and so a MAXT above 256; with it a
// thread never has one group of a row that takes 9 warps in 32 bits. Kernels that no shape asks for are not built.
template <int ESIZE, bool PAIRS, typename F>
void with_shape(const Shape& s, bool all, F&& f) {
  using std::integral_constant;
  using One = integral_constant<int, 1>;
  using Two = integral_constant<int, 2>;
  using Warp = integral_constant<int, 32>;
  auto go = [&](auto mode, auto every) {
    constexpr bool kAl = decltype(mode)::value == kAligned, kPairs = PAIRS && kAl && decltype(every)::value;
    if (s.groups == 2 && s.threads > 512) return f(mode, Two{}, Warp{}, every, integral_constant<int, 1024>{});
    if (s.groups == 2 && (!kPairs || s.threads > 256))
      return f(mode, Two{}, Warp{}, every, integral_constant<int, 512>{});
    if constexpr (kPairs) {
      if (s.groups == 2) return f(mode, Two{}, Warp{}, every, integral_constant<int, 256>{});
    }
    if constexpr (!(kPairs && ESIZE == 4)) {
      if (s.threads > 256) return f(mode, One{}, Warp{}, every, integral_constant<int, 512>{});
    }
    if constexpr (kAl) {
      if (s.lanes == 16) return f(mode, One{}, integral_constant<int, 16>{}, every, integral_constant<int, 256>{});
      if (s.lanes == 8) return f(mode, One{}, integral_constant<int, 8>{}, every, integral_constant<int, 256>{});
    }
    f(mode, One{}, Warp{}, every, integral_constant<int, 256>{});
  };
  auto with = [&](auto mode) { all ? go(mode, std::true_type{}) : go(mode, std::false_type{}); };
  if (s.mode == kAligned)
    with(integral_constant<int, kAligned>{});
  else if (s.mode == kShifted)
    with(integral_constant<int, kShifted>{});
  else
    go(integral_constant<int, kSingle>{}, std::false_type{});
}

// The grid, with rows of a CTA that lie alike where that is needed.
unsigned grid_of(int64_t wanted, const NormParams& p, const Shape& s, int esize) {
  const int per = 32 / s.lanes;  // rows at a time
  int64_t grid = std::min<int64_t>((p.rows + per - 1) / per, wanted);
  const int v = 16 / esize;
  if (s.mode == kShifted && grid < p.rows) grid = std::min<int64_t>(p.rows, std::max<int64_t>(v, grid / v * v));
  return (unsigned)grid;
}

// The ring's depth for `fit` CTAs per SM, and the CTAs that are resident with it.
int64_t plan_ring(NormParams& p, const Shape& s, int esize, int fit, int deepest) {
  p.depth = 1;
  if (s.mode != kSingle) {
    for (int t = 0, at = 0; t < kIns; ++t) {
      p.slot[t] = at;
      at += p.in[t] != nullptr ? s.groups * s.threads * 8 * esize : 0;
    }
    p.stage = s.ins * s.groups * s.threads * 8 * esize;
    p.depth = std::min(deepest, std::max(1, kSmemBudget / fit / p.stage));
    fit = std::max(1, std::min(fit, kSmemBudget / (p.stage * p.depth)));
  }
  return (int64_t)num_sms() * fit;
}

// CTAs of this size that an SM's registers (four files of 16384, a warp in one of them) hold, at most 16.
template <auto KERNEL>
int fit_of(int threads) {
  static const int warps = [] {
    cudaFuncAttributes a{};
    C10_CUDA_CHECK(cudaFuncGetAttributes(&a, KERNEL));
    return 4 * (16384 / ((a.numRegs + 7) / 8 * 8 * 32));
  }();
  return std::max(1, std::min(16, warps * 32 / threads));
}

template <typename K>
void launch_norm(K kernel, const NormParams& p, const Shape& s, unsigned grid) {
  const int smem = p.stage * p.depth;
  if (smem > 40 * 1024)  // without asking, a CTA gets 48 KB, its static part included
    C10_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBudget));
  kernel<<<grid, s.threads, smem, cur_stream()>>>(p);
  MT_LAUNCH_CHECK();
}

const void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

uint32_t ld(const at::Tensor& t) { return t.defined() && t.size(0) > 1 ? (uint32_t)t.stride(0) : 0u; }

NormParams params_of(const ResidualNormArgs& a) {
  NormParams p{};
  p.in[kX] = a.x.data_ptr();
  MT_CHECK(a.x.size(0) < (int64_t(1) << 31), "residual_norm: too many rows: ", a.x.size(0));
  p.rows = (uint32_t)a.x.size(0);
  p.d = (int)a.x.size(1);
  p.ld[kX] = ld(a.x);
  if (a.h.has_value()) {
    p.in[kH] = a.h->data_ptr();
    p.ld[kH] = ld(*a.h);
  }
  if (a.pre.has_value()) p.pre = a.pre->data_ptr<float>();
  if (a.post.has_value()) p.post = a.post->data_ptr<float>();
  if (a.gate_kind == kGateFull) {
    p.in[kGate] = a.gate->data_ptr();
    p.ld[kGate] = ld(*a.gate);
  } else if (a.gate.has_value()) {
    p.gate = a.gate->data_ptr<float>();
  }
  p.gate_kind = a.gate_kind;
  p.beta = (float)a.beta;
  p.alpha = (float)a.alpha;
  p.eps = (float)a.eps;
  return p;
}

}  // namespace

void residual_norm_fwd_launch(const ResidualNormArgs& a, const at::Tensor& y, const at::Tensor& n,
                              const at::Tensor& rstd_h, const at::Tensor& rstd_y) {
  NormParams p = params_of(a);
  p.y = const_cast<void*>(ptr(y));
  p.n = const_cast<void*>(ptr(n));
  p.rstd_h = rstd_h.defined() ? rstd_h.data_ptr<float>() : nullptr;
  p.rstd_y = rstd_y.defined() ? rstd_y.data_ptr<float>() : nullptr;
  if (p.rows == 0) return;
  dispatch_act(a.x.scalar_type(), [&](auto t) {
    using T = decltype(t);
    const Shape s = shape_of(p, sizeof(T), false);
    const bool all = p.in[kH] != nullptr && p.n != nullptr && a.gate_kind != kGateFull;
    with_shape<sizeof(T), false>(s, all, [&](auto mode, auto ng, auto lanes, auto every, auto maxt) {
      constexpr int kMaxT = decltype(maxt)::value, kMinB = kMaxT == 1024 ? 1 : 1024 / kMaxT;
      constexpr auto kernel =
          residual_norm_fwd<T, decltype(mode)::value, decltype(ng)::value, decltype(lanes)::value,
                            decltype(every)::value, kMaxT, kMinB>;
      const int64_t resident = plan_ring(p, s, sizeof(T), fit_of<kernel>(s.threads), 4);
      launch_norm(kernel, p, s, grid_of(resident, p, s, sizeof(T)));
    });
  });
}

void residual_norm_bwd_launch(const ResidualNormArgs& a, const at::Tensor& rstd_h, const at::Tensor& rstd_y,
                              const at::Tensor& dy, const at::Tensor& dn, const at::Tensor& dx, const at::Tensor& dh,
                              const at::Tensor& dgate, const at::Tensor& dpre, const at::Tensor& dpost) {
  NormParams p = params_of(a);
  p.in[kDy] = ptr(dy);
  p.ld[kDy] = ld(dy);
  p.in[kDn] = ptr(dn);
  p.ld[kDn] = ld(dn);
  p.dx = const_cast<void*>(ptr(dx));
  p.dh = const_cast<void*>(ptr(dh));
  p.dgate = const_cast<void*>(ptr(dgate));
  p.rstd_h = rstd_h.defined() ? rstd_h.data_ptr<float>() : nullptr;
  p.rstd_y = rstd_y.defined() ? rstd_y.data_ptr<float>() : nullptr;
  const bool gate_sum = dgate.defined() && a.gate_kind == kGateChannel;
  p.want_dpre = dpre.defined();
  p.want_q = dpost.defined() || gate_sum;
  if (p.rows == 0) {
    for (const at::Tensor* t : {&dpre, &dpost}) {
      if (t->defined()) t->zero_();
    }
    if (gate_sum) dgate.zero_();
    return;
  }
  dispatch_act(a.x.scalar_type(), [&](auto t) {
    using T = decltype(t);
    bool all = a.gate_kind != kGateFull;
    for (const void* q : {p.in[kH], p.in[kDy], p.in[kDn], (const void*)p.dx, (const void*)p.dh}) all = all && q != nullptr;
    const Shape s = shape_of(p, sizeof(T), all);
    with_shape<sizeof(T), true>(s, all, [&](auto mode, auto ng, auto lanes, auto every, auto maxt) {
      constexpr int kMaxT = decltype(maxt)::value, kMinB = decltype(ng)::value == 1 && kMaxT == 256 ? 2 : 1;
      constexpr auto kernel =
          residual_norm_bwd<T, decltype(mode)::value, decltype(ng)::value, decltype(lanes)::value,
                            decltype(every)::value, kMaxT, kMinB>;
      int64_t grid = plan_ring(p, s, sizeof(T), fit_of<kernel>(s.threads), 4);
      // a few rows for each CTA at least: its partial sums cost as much as two rows
      if (p.want_dpre || p.want_q) {
        const int64_t few = 4 * 32 / s.lanes;
        grid = std::min<int64_t>(grid, (p.rows + few - 1) / few);
      }
      grid = grid_of(grid, p, s, sizeof(T));
      at::Tensor part;
      if (p.want_dpre || p.want_q) {
        part = at::Tensor(at::detail::empty_cuda({grid, 2, (int64_t)p.d}, at::kFloat, a.x.device(), c10::nullopt));
        p.part = part.data_ptr<float>();
      }
      launch_norm(kernel, p, s, (unsigned)grid);
      if (p.part != nullptr) {
        auto finish = [&](auto kernel, int cols) {
          kernel<<<dim3((p.d + cols - 1) / cols, p.want_dpre + p.want_q), kFinishThreads, 0, cur_stream()>>>(
              p.part, (int)grid, p.d, p.want_dpre, p.alpha, a.gate_kind == kGateChannel ? p.gate : nullptr, p.post,
              p.want_dpre ? dpre.data_ptr<float>() : nullptr, dpost.defined() ? dpost.data_ptr<float>() : nullptr,
              gate_sum ? dgate.data_ptr<float>() : nullptr);
        };
        if (p.d <= 1024)
          finish(residual_norm_finish<8>, 8);
        else
          finish(residual_norm_finish<32>, 32);
        MT_LAUNCH_CHECK();
      }
    });
  });
}

}  // namespace mtorus

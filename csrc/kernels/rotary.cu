// Rotary positions: each pair (a, b) of a head's first rot_dim values turns by pos * w_i,
//   a' = s (a cos - b sin),  b' = s (a sin + b cos),
// the rest of the head passes through; the backward is the same with -angle.
//
// Bound by memory: every value is read once and written once, with about 3 flops each.  A thread owns one chunk of a
// head -- in the half layout VEC values of each half -- of one token and takes it through several heads, 16-byte loads
// and stores, as many tokens to a CTA as fill 256 threads.  It asks for its values first of all; while they are on their
// way the CTA computes its tokens' cosines and sines, once for all heads, into shared memory.  (Asking for the tokens'
// positions before the values makes it slower: 117 us against 105 us without given positions, 119 us against 114 us
// with them, for 32769 tokens of 40 heads x 128 bf16, where the copy's rate allows 103 us.)
//
// No table is read.  A frequency is a 64-bit fixed-point fraction of a revolution per position (cut off there); times the
// position, modulo 2^64, it is the angle without the whole revolutions, exact to |pos| 2^-64 of one and to a few 2^-53 of the
// angle from the frequency itself.  Its upper 32 bits, rounded to fp32, go on: 2^-26 of a revolution at worst, which is more
// than the former up to positions of about 2^28.  So far positions lose nothing that fp32 would keep, no longest length has
// to be set, and no 64-bit floats are needed.
#include "decoder_ops.h"
#include "vec.cuh"

namespace mtorus {

namespace {

struct Seg {
  const void* in;
  void* out;
  int64_t in_b, in_s, in_h, out_b, out_s, out_h;  // strides in values
  int heads, heads_rot;
};

struct RotParams {
  Seg seg[2];
  const uint64_t* turns;
  const void* pos;
  int64_t pos_b, pos_s, offset;
  uint32_t S, tokens;
  int pos_size;  // bytes of a position; 0: offset + index in the sequence
  int heads, half, chunks, rot_chunks, pass_vectors, head_step, tile;
  float scale, sign;
  bool copy;  // out of place: values that are not rotated are copied
};


// NV: vectors of a rotated chunk -- half a rotation apart, or (INTERLEAVED) neighbours.
template <typename T, int VEC, bool INTERLEAVED, int NV, int U>
__global__ void __launch_bounds__(VEC == 1 ? 512 : 256, VEC == 1 ? 1 : U == 2 ? 4 : 3) rotary_kernel(const __grid_constant__ RotParams p) {
  extern __shared__ float2 cs[];  // [tokens of the CTA][half]
  constexpr int NP = NV * VEC / 2;  // pairs of a chunk
  using V = Vec<T, VEC>;
  const uint32_t t0 = blockIdx.x * p.tile;
  // thread = (token of the tile * head_step + first head) * chunks + chunk
  const int row = threadIdx.x / p.chunks, c = threadIdx.x - row * p.chunks;
  const int tt = row / p.head_step, first = row - tt * p.head_step;
  const uint32_t t = t0 + tt, b = t / p.S, s = t - b * p.S;
  const bool here = tt < p.tile && t < p.tokens, rot_chunk = c < p.rot_chunks;
  const int pass_width = p.pass_vectors * VEC;
  const int at = rot_chunk ? c * (INTERLEAVED ? NV * VEC : VEC) : 2 * p.half + (c - p.rot_chunks) * pass_width;
  const int next = INTERLEAVED || !rot_chunk ? VEC : p.half;  // from a chunk's first vector to its second
  const bool two = rot_chunk ? NV == 2 : p.pass_vectors == 2;

  V x[U][2];
  auto load = [&](int h0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int hh = h0 + u * p.head_step;
      const bool second = hh >= p.seg[0].heads;
      const Seg& g = p.seg[second];
      const int h = second ? hh - p.seg[0].heads : hh;
      if (hh >= p.heads || !(p.copy || (rot_chunk && h < g.heads_rot))) continue;
      const T* in = static_cast<const T*>(g.in) + b * g.in_b + s * g.in_s + h * g.in_h + at;
      x[u][0] = load_stream(reinterpret_cast<const V*>(in));
      if (two) x[u][1] = load_stream(reinterpret_cast<const V*>(in + next));
    }
  };
  if (here) load(first);
  // The CTA's angles: thread i takes i, i + blockDim, ... of [token][pair].
  int ti = threadIdx.x / p.half, pair = threadIdx.x - ti * p.half;
  const int dt = blockDim.x / p.half, dp = blockDim.x - dt * p.half;
  for (; ti < p.tile; ti += dt, pair += dp) {
    if (pair >= p.half) {
      pair -= p.half;
      if (++ti >= p.tile) break;
    }
    const uint32_t ta = t0 + ti;
    if (ta >= p.tokens) break;
    const uint32_t ba = ta / p.S, sa = ta - ba * p.S;
    int64_t pos = p.offset + sa;
    if (p.pos_size == 8) pos = static_cast<const int64_t*>(p.pos)[ba * p.pos_b + sa * p.pos_s];
    if (p.pos_size == 4) pos = static_cast<const int32_t*>(p.pos)[ba * p.pos_b + sa * p.pos_s];
    const uint64_t turn = (uint64_t)pos * p.turns[pair];
    float sn, cn;
    sincospif((float)(int32_t)(turn >> 32) * 0x1p-31f, &sn, &cn);
    cs[ti * p.half + pair] = make_float2(cn * p.scale, sn * p.scale * p.sign);
  }
  __syncthreads();
  if (!here) return;
  float cn[NP], sn[NP];
  if (rot_chunk) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const float2 v = cs[tt * p.half + c * NP + i];
      cn[i] = v.x;
      sn[i] = v.y;
    }
  }
  for (int h0 = first; h0 < p.heads; h0 += U * p.head_step) {
    if (h0 != first) load(h0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int hh = h0 + u * p.head_step;
      const bool second = hh >= p.seg[0].heads;
      const Seg& g = p.seg[second];
      const int h = second ? hh - p.seg[0].heads : hh;
      const bool turned = rot_chunk && h < g.heads_rot;
      if (hh >= p.heads || !(p.copy || turned)) continue;
      if (turned) {
        float f[NV * VEC], r[NV * VEC];
        widen(x[u][0], f);
        if (NV == 2) widen(x[u][1], f + (NV - 1) * VEC);
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const int ia = INTERLEAVED ? 2 * i : i, ib = INTERLEAVED ? 2 * i + 1 : VEC + i;
          r[ia] = f[ia] * cn[i] - f[ib] * sn[i];
          r[ib] = f[ia] * sn[i] + f[ib] * cn[i];
        }
        x[u][0] = narrow<T, VEC>(r);
        if (NV == 2) x[u][1] = narrow<T, VEC>(r + (NV - 1) * VEC);
      }
      T* out = static_cast<T*>(g.out) + b * g.out_b + s * g.out_s + h * g.out_h + at;
      store_stream(reinterpret_cast<V*>(out), x[u][0]);
      if (two) store_stream(reinterpret_cast<V*>(out + next), x[u][1]);
    }
  }
}

// Largest number of values per vector that every pointer, stride and extent allows.
int widest_vector(const RotParams& p, int nseg, int64_t D, int esize, bool interleaved) {
  for (int v = 16 / esize; v > 1; v /= 2) {
    bool ok = D % v == 0 && (interleaved ? 2 * p.half : p.half) % v == 0;
    for (int i = 0; ok && i < nseg; ++i) {
      const Seg& g = p.seg[i];
      for (int64_t st : {g.in_b, g.in_s, g.in_h, g.out_b, g.out_s, g.out_h}) ok = ok && st % v == 0;
      ok = ok && reinterpret_cast<uintptr_t>(g.in) % (v * esize) == 0 &&
           reinterpret_cast<uintptr_t>(g.out) % (v * esize) == 0;
    }
    if (ok) return v;
  }
  return 1;
}

// With U heads in flight per thread; false, and nothing launched, where that leaves SMs without work.
template <typename T, int VEC, bool IL, int NV, int U>
bool try_launch(RotParams p, int64_t D) {
  const int rest = (int)(D - 2 * p.half) / VEC;  // vectors that pass through
  p.pass_vectors = rest % 2 == 0 ? 2 : 1;
  p.rot_chunks = 2 * p.half / (NV * VEC);
  p.chunks = p.rot_chunks + rest / p.pass_vectors;
  // threads of a token: enough to take all heads at once, in a CTA of about 256 threads
  p.head_step = std::max(1, std::min((p.heads + U - 1) / U, 256 / p.chunks));
  const int per_token = p.head_step * p.chunks;
  p.tile = std::max(1, std::min(256 / per_token, 4096 / p.half));  // up to 32 KB of cosines and sines
  const int threads = (per_token * p.tile + 31) / 32 * 32;
  const unsigned blocks = (p.tokens + p.tile - 1) / p.tile;
  if (U == 4 && blocks < 4u * num_sms()) return false;
  rotary_kernel<T, VEC, IL, NV, U><<<blocks, threads, (size_t)p.tile * p.half * sizeof(float2), cur_stream()>>>(p);
  MT_LAUNCH_CHECK();
  return true;
}

// Four heads where there are many tokens (8 x 2048 tokens of 48 heads x 128 bf16: 61 us, with two 68 us), two for few
// (500 tokens of 20 heads x 128: 3.6 us, with four 3.9 us; 8 tokens of 40 heads 2.6 us and 3.3 us).
template <typename T, int VEC, bool IL, int NV>
void launch(const RotParams& p, int64_t D) {
  if (!try_launch<T, VEC, IL, NV, 4>(p, D)) try_launch<T, VEC, IL, NV, 2>(p, D);
}

}  // namespace

void rotary_launch(const std::vector<RotarySegment>& segs, const RotaryArgs& a) {
  RotParams p{};
  const int64_t B = segs[0].in.size(0), S = segs[0].in.size(1), D = segs[0].in.size(3);
  for (size_t i = 0; i < segs.size(); ++i) {
    const at::Tensor &in = segs[i].in, &out = segs[i].out;
    // the stride of an axis of extent 1 is never used: it does not restrict the vector width either
    auto st = [](const at::Tensor& t, int64_t dim) { return t.size(dim) > 1 ? t.stride(dim) : int64_t(0); };
    p.seg[i] = Seg{in.data_ptr(),     out.data_ptr(),   st(in, 0),          st(in, 1),
                   st(in, 2),         st(out, 0),       st(out, 1),         st(out, 2),
                   (int)in.size(2),   (int)segs[i].heads_rot};
    p.heads += (int)in.size(2);
  }
  p.turns = reinterpret_cast<const uint64_t*>(a.turns.data_ptr<int64_t>());
  p.half = (int)(a.rot_dim / 2);
  MT_CHECK(B * S < (int64_t(1) << 31), "rotary: too many tokens: ", B * S);
  p.S = (uint32_t)S;
  p.tokens = (uint32_t)(B * S);
  p.offset = a.offset;
  if (a.positions.has_value()) {
    p.pos = a.positions->data_ptr();
    p.pos_size = (int)a.positions->element_size();
    p.pos_b = a.positions->stride(0);
    p.pos_s = a.positions->stride(1);
  }
  p.scale = (float)a.scale;
  p.sign = a.inverse ? -1.f : 1.f;
  p.copy = !a.in_place;
  if (p.tokens == 0 || p.heads == 0) return;
  dispatch_act(segs[0].in.scalar_type(), [&](auto t) {
    using T = decltype(t);
    const int v = widest_vector(p, (int)segs.size(), D, sizeof(T), a.interleaved);
    auto go = [&](auto il, auto nv) {
      constexpr bool IL = decltype(il)::value;
      constexpr int NV = decltype(nv)::value;
      if constexpr (sizeof(T) == 2) {
        if (v == 8) return launch<T, 8, IL, NV>(p, D);
      }
      if (v == 4) return launch<T, 4, IL, NV>(p, D);
      if (v == 2) return launch<T, 2, IL, NV>(p, D);
      launch<T, 1, IL, 2>(p, D);
    };
    using two = std::integral_constant<int, 2>;
    if (!a.interleaved)
      go(std::false_type{}, two{});
    else if (a.rot_dim % (2 * v) == 0)
      go(std::true_type{}, two{});
    else
      go(std::true_type{}, std::integral_constant<int, 1>{});
  });
}

}  // namespace mtorus

// Rotary positions: each pair (a, b) of a head's first rot_dim values turns by pos * w_i,
//   a' = s (a cos - b sin),  b' = s (a sin + b cos),
// the rest of the head passes through; the backward is the same with -angle.
//
// Bound by memory: every value is read once and written once, with about 3 flops each.  One CTA takes a few
// tokens and all their heads.  It computes the tokens' cosines and sines once, into shared memory (they are the
// same for every head), then each thread owns one chunk of a head -- in the half layout VEC values of each half
// -- and walks tokens and heads with 16-byte loads and stores.  No table is read: an angle is
// pos * (w / 2 pi) revolutions in 64 bits, of which only the fraction goes on in 32 bits, so far positions
// lose nothing and no longest length has to be set.
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
  const double* turns;
  const void* pos;
  int64_t pos_b, pos_s, offset, S, tokens;
  int pos_size;  // bytes of a position; 0: offset + index in the sequence
  int heads, half, chunks, rot_chunks, heads_per_pass, tile;
  float scale, sign;
  bool copy;  // out of place: values that are not rotated are copied
};

constexpr int kMaxThreads = 512;

template <typename T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(kMaxThreads) rotary_kernel(const __grid_constant__ RotParams p) {
  extern __shared__ float2 cs[];  // [tile][half]
  const int64_t t0 = (int64_t)blockIdx.x * p.tile;
  const int nt = (int)min((int64_t)p.tile, p.tokens - t0);
  for (int i = threadIdx.x; i < nt * p.half; i += blockDim.x) {
    const int tt = i / p.half, pair = i - tt * p.half;
    const int64_t t = t0 + tt, b = t / p.S, s = t - b * p.S;
    int64_t pos = p.offset + s;
    if (p.pos_size == 8) pos = static_cast<const int64_t*>(p.pos)[b * p.pos_b + s * p.pos_s];
    if (p.pos_size == 4) pos = static_cast<const int32_t*>(p.pos)[b * p.pos_b + s * p.pos_s];
    const double turn = (double)pos * p.turns[pair];
    float sn, cn;
    sincospif(2.f * (float)(turn - rint(turn)), &sn, &cn);
    cs[i] = make_float2(cn * p.scale, sn * p.scale * p.sign);
  }
  __syncthreads();
  const int hp = threadIdx.x / p.chunks, c = threadIdx.x - hp * p.chunks;
  if (hp >= p.heads_per_pass) return;
  // A chunk: two vectors half a rotation apart, or 1-2 vectors of neighbouring pairs.  NV vectors, NP pairs.
  constexpr int NV = INTERLEAVED ? (VEC == 1 ? 2 : 1) : 2;
  constexpr int NP = NV * VEC / 2;
  constexpr int U = INTERLEAVED ? 4 : 2;  // heads in flight per thread
  using V = Vec<T, VEC>;
  const bool rot_chunk = c < p.rot_chunks;
  const int at = rot_chunk ? (INTERLEAVED ? c * NV * VEC : c * VEC) : 2 * p.half + (c - p.rot_chunks) * VEC;
  const int next = INTERLEAVED ? VEC : p.half;  // from a chunk's first vector to its second
  for (int tt = 0; tt < nt; ++tt) {
    const int64_t t = t0 + tt, b = t / p.S, s = t - b * p.S;
    float cn[NP], sn[NP];
    if (rot_chunk) {
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const float2 v = cs[tt * p.half + c * NP + i];
        cn[i] = v.x;
        sn[i] = v.y;
      }
    }
    for (int h0 = hp; h0 < p.heads; h0 += U * p.heads_per_pass) {
      V x[U][NV];
      T* out[U];
      bool turned[U], todo[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int hh = h0 + u * p.heads_per_pass;
        const bool second = hh >= p.seg[0].heads;
        const Seg& g = p.seg[second];
        const int h = second ? hh - p.seg[0].heads : hh;
        const T* in = static_cast<const T*>(g.in) + b * g.in_b + s * g.in_s + h * g.in_h + at;
        out[u] = static_cast<T*>(g.out) + b * g.out_b + s * g.out_s + h * g.out_h + at;
        turned[u] = rot_chunk && h < g.heads_rot;
        todo[u] = hh < p.heads && (turned[u] || p.copy);
        if (todo[u]) {
          x[u][0] = load_stream(reinterpret_cast<const V*>(in));
          if (NV == 2 && rot_chunk) x[u][NV - 1] = load_stream(reinterpret_cast<const V*>(in + next));
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (!todo[u]) continue;
        if (turned[u]) {
          float f[NV * VEC], r[NV * VEC];
          widen(x[u][0], f);
          if (NV == 2) widen(x[u][NV - 1], f + (NV - 1) * VEC);
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            const int ia = INTERLEAVED ? 2 * i : i, ib = INTERLEAVED ? 2 * i + 1 : VEC + i;
            r[ia] = f[ia] * cn[i] - f[ib] * sn[i];
            r[ib] = f[ia] * sn[i] + f[ib] * cn[i];
          }
          x[u][0] = narrow<T, VEC>(r);
          if (NV == 2) x[u][NV - 1] = narrow<T, VEC>(r + (NV - 1) * VEC);
        }
        store_stream(reinterpret_cast<V*>(out[u]), x[u][0]);
        if (NV == 2 && rot_chunk) store_stream(reinterpret_cast<V*>(out[u] + next), x[u][NV - 1]);
      }
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

template <typename T, int VEC, bool IL>
void launch(RotParams p, int64_t D) {
  p.rot_chunks = IL ? 2 * p.half / (VEC == 1 ? 2 : VEC) : p.half / VEC;
  p.chunks = p.rot_chunks + (int)(D - 2 * p.half) / VEC;
  // the heads split evenly over the passes of a block of about 256 threads
  const int fit = std::max(1, 256 / p.chunks);
  const int passes = (p.heads + fit - 1) / fit;
  p.heads_per_pass = (p.heads + passes - 1) / passes;
  const int threads = (p.heads_per_pass * p.chunks + 31) / 32 * 32;
  p.tile = p.tokens >= 4 * 1024 ? 4 : 1;
  const int64_t blocks = (p.tokens + p.tile - 1) / p.tile;
  MT_CHECK(blocks < (int64_t(1) << 31), "rotary: too many tokens: ", p.tokens);
  rotary_kernel<T, VEC, IL><<<(unsigned)blocks, threads, (size_t)p.tile * p.half * sizeof(float2), cur_stream()>>>(p);
  MT_LAUNCH_CHECK();
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
  p.turns = a.turns.data_ptr<double>();
  p.half = (int)(a.rot_dim / 2);
  p.S = S;
  p.tokens = B * S;
  p.offset = a.offset;
  if (a.positions.has_value()) {
    p.pos = a.positions->data_ptr();
    p.pos_size = (int)a.positions->element_size();
    p.pos_b = a.positions->stride(0);
    p.pos_s = a.positions->stride(1);
  }
  p.scale = (float)a.scale;
  p.sign = a.inverse ? -1.f : 1.f;
  p.copy = segs[0].in.data_ptr() != segs[0].out.data_ptr();
  if (p.tokens == 0 || p.heads == 0) return;
  dispatch_act(segs[0].in.scalar_type(), [&](auto t) {
    using T = decltype(t);
    const int v = widest_vector(p, (int)segs.size(), D, sizeof(T), a.interleaved);
    auto go = [&](auto il) {
      constexpr bool IL = decltype(il)::value;
      if constexpr (sizeof(T) == 2) {
        if (v == 8) return launch<T, 8, IL>(p, D);
      }
      if (v == 4) return launch<T, 4, IL>(p, D);
      if (v == 2) return launch<T, 2, IL>(p, D);
      launch<T, 1, IL>(p, D);
    };
    if (a.interleaved)
      go(std::true_type{});
    else
      go(std::false_type{});
  });
}

}  // namespace mtorus

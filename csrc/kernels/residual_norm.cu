// Residual update of a block with its norms, in one pass each way:
//   rh = 1/sqrt(mean h^2 + eps),  b = h rh post,   y = beta x + alpha g b     (post norm, gate, scales)
//   ry = 1/sqrt(mean y^2 + eps),  n = y ry pre                               (pre norm of the next block)
// Backward, with u = dn pre, yh = y ry, hh = h rh:
//   Y = dy + ry (u - yh mean(u yh));  dx = beta Y;  dg = alpha b Y;  dpre = sum dn yh;  dpost = sum alpha g Y hh
//   dh = rh (alpha g post Y - hh mean(alpha g b Y))
// y is computed again from x and h in 32 bits (reading x instead of y costs the same bytes), so the statistics
// and the weight gradients see the value before its rounding.
//
// Bound by memory: forward 2 reads and 2 writes of [T, d], backward 4 and 2.  One CTA of d / 8 threads walks a
// strided set of rows; a thread owns the same 8 columns of every row, so the sums of weight gradients stay in its
// registers and leave once per CTA, to be added up in a fixed order by a second kernel.  The backward needs one
// row reduction, not two: mean(alpha g b Y) follows from sums of alpha g b with dy, u and yh.
#include "decoder_ops.h"
#include "vec.cuh"

namespace mtorus {

namespace {

constexpr int kMaxWarps = 32;

struct NormParams {
  const void *x, *h, *dy, *dn, *gate;
  int64_t ldx, ldh, lddy, lddn, ldg;
  const float *pre, *post;
  void *y, *n, *dx, *dh, *dgate;
  float *rstd_h, *rstd_y, *part;
  int64_t rows;
  int d, gate_kind;
  float beta, alpha, eps;
  int want_dpre, want_dpost, want_dgate;
};

// Columns of a thread's 8 values in a group of 256 columns: vectors of 16 bytes where rows are aligned
// (ALIGNED), else single values 32 apart, so that each load of the warp is contiguous.
template <typename T, bool ALIGNED>
__device__ __forceinline__ int col_of(int group, int lane, int i) {
  constexpr int VEC = 16 / sizeof(T);
  if constexpr (!ALIGNED) return group * 256 + i * 32 + lane;
  return group * 256 + (i / VEC) * (32 * VEC) + lane * VEC + i % VEC;
}

template <typename T, bool ALIGNED>
__device__ __forceinline__ void load8(const T* row, int group, int lane, int d, float* f) {
  if constexpr (ALIGNED) {
    constexpr int VEC = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 8; i += VEC) {
      const int c = col_of<T, ALIGNED>(group, lane, i);
      Vec<T, VEC> v;
      if (c < d) v = load_stream(reinterpret_cast<const Vec<T, VEC>*>(row + c));
      widen(v, f + i);
      if (c >= d) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) f[i + k] = 0.f;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = col_of<T, ALIGNED>(group, lane, i);
      f[i] = c < d ? to_f<T>(row[c]) : 0.f;
    }
  }
}

template <typename T, bool ALIGNED>
__device__ __forceinline__ void store8(T* row, int group, int lane, int d, const float* f) {
  if constexpr (ALIGNED) {
    constexpr int VEC = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 8; i += VEC) {
      const int c = col_of<T, ALIGNED>(group, lane, i);
      if (c < d) store_stream(reinterpret_cast<Vec<T, VEC>*>(row + c), narrow<T, VEC>(f + i));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = col_of<T, ALIGNED>(group, lane, i);
      if (c < d) row[c] = from_f<T>(f[i]);
    }
  }
}

// Weights are fp32 vectors of d values; missing ones read as `none`.
template <typename T, bool ALIGNED>
__device__ __forceinline__ void load_weight(const float* w, int group, int lane, int d, float none, float* f) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = col_of<T, ALIGNED>(group, lane, i);
    f[i] = w != nullptr && c < d ? w[c] : none;
  }
}

// Sums of N values over the CTA; every thread gets them.  `red` holds [2][kMaxWarps][N] floats and `par`
// alternates between its halves, so one barrier per call is enough.
template <int N>
__device__ __forceinline__ void cta_sum(float (&v)[N], float* red, int& par) {
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = warp_sum(v[k]);
  const int nw = blockDim.x >> 5;
  if (nw == 1) return;
  float* r = red + par * kMaxWarps * N;
  par ^= 1;
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int k = 0; k < N; ++k) r[(threadIdx.x >> 5) * N + k] = v[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = 0.f;
  for (int w = 0; w < nw; ++w) {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] += r[w * N + k];
  }
}

template <typename T, bool ALIGNED, int NG>
__global__ void __launch_bounds__(1024) residual_norm_fwd(const __grid_constant__ NormParams p) {
  __shared__ float red[2 * kMaxWarps];
  const int lane = threadIdx.x & 31, g0 = (threadIdx.x >> 5) * NG, d = p.d;
  const float inv_d = 1.f / d;
  int par = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    float x[NG][8], y[NG][8];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      load8<T, ALIGNED>(static_cast<const T*>(p.x) + row * p.ldx, g0 + g, lane, d, x[g]);
      if (p.h != nullptr) load8<T, ALIGNED>(static_cast<const T*>(p.h) + row * p.ldh, g0 + g, lane, d, y[g]);
    }
    if (p.h != nullptr) {
      float rh = 1.f;
      if (p.post != nullptr) {
        float s[1] = {0.f};
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
          for (int i = 0; i < 8; ++i) s[0] += y[g][i] * y[g][i];
        cta_sum<1>(s, red, par);
        rh = rsqrtf(s[0] * inv_d + p.eps);
        if (threadIdx.x == 0 && p.rstd_h != nullptr) p.rstd_h[row] = rh;
      }
      float gr = p.alpha * rh;
      if (p.gate_kind == kGateRow) gr *= static_cast<const float*>(p.gate)[row];
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float w[8];
        if (p.post != nullptr) {
          load_weight<T, ALIGNED>(p.post, g0 + g, lane, d, 0.f, w);
#pragma unroll
          for (int i = 0; i < 8; ++i) y[g][i] *= w[i];
        }
        if (p.gate_kind == kGateChannel) {
          load_weight<T, ALIGNED>(static_cast<const float*>(p.gate), g0 + g, lane, d, 0.f, w);
#pragma unroll
          for (int i = 0; i < 8; ++i) y[g][i] *= w[i];
        }
        if (p.gate_kind == kGateFull) {
          load8<T, ALIGNED>(static_cast<const T*>(p.gate) + row * p.ldg, g0 + g, lane, d, w);
#pragma unroll
          for (int i = 0; i < 8; ++i) y[g][i] *= w[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) y[g][i] = p.beta * x[g][i] + gr * y[g][i];
        if (p.y != nullptr) store8<T, ALIGNED>(static_cast<T*>(p.y) + row * d, g0 + g, lane, d, y[g]);
      }
    } else {
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int i = 0; i < 8; ++i) y[g][i] = x[g][i];
    }
    if (p.n == nullptr) continue;
    float s[1] = {0.f};
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int i = 0; i < 8; ++i) s[0] += y[g][i] * y[g][i];
    cta_sum<1>(s, red, par);
    const float ry = rsqrtf(s[0] * inv_d + p.eps);
    if (threadIdx.x == 0 && p.rstd_y != nullptr) p.rstd_y[row] = ry;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float w[8];
      load_weight<T, ALIGNED>(p.pre, g0 + g, lane, d, 0.f, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] *= y[g][i] * ry;
      store8<T, ALIGNED>(static_cast<T*>(p.n) + row * d, g0 + g, lane, d, w);
    }
  }
}

// part: [gridDim.x][3][d] sums over the CTA's rows of dpre, dpost and the per-channel dgate.
template <typename T, bool ALIGNED, int NG>
__global__ void __launch_bounds__(1024) residual_norm_bwd(const __grid_constant__ NormParams p) {
  __shared__ float red[2 * kMaxWarps * 4];
  const int lane = threadIdx.x & 31, g0 = (threadIdx.x >> 5) * NG, d = p.d;
  const float inv_d = 1.f / d;
  int par = 0;
  float sum_pre[NG][8], sum_post[NG][8], sum_gate[NG][8];
#pragma unroll
  for (int g = 0; g < NG; ++g)
#pragma unroll
    for (int i = 0; i < 8; ++i) sum_pre[g][i] = sum_post[g][i] = sum_gate[g][i] = 0.f;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    float x[NG][8], h[NG][8], dy[NG][8], dn[NG][8];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      load8<T, ALIGNED>(static_cast<const T*>(p.x) + row * p.ldx, g0 + g, lane, d, x[g]);
      if (p.h != nullptr) load8<T, ALIGNED>(static_cast<const T*>(p.h) + row * p.ldh, g0 + g, lane, d, h[g]);
      if (p.dy != nullptr) load8<T, ALIGNED>(static_cast<const T*>(p.dy) + row * p.lddy, g0 + g, lane, d, dy[g]);
      if (p.dn != nullptr) load8<T, ALIGNED>(static_cast<const T*>(p.dn) + row * p.lddn, g0 + g, lane, d, dn[g]);
    }
    const float rh = p.post != nullptr ? p.rstd_h[row] : 1.f;
    const float ry = p.dn != nullptr ? p.rstd_y[row] : 0.f;
    const float gr = p.gate_kind == kGateRow ? static_cast<const float*>(p.gate)[row] : 1.f;
    // s: sum u yh, and sums of c = alpha (g) b with dy, u and yh; a gate per row is left out of c
    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float wpre[8], wpost[8], gate[8];
      load_weight<T, ALIGNED>(p.pre, g0 + g, lane, d, 0.f, wpre);
      load_weight<T, ALIGNED>(p.post, g0 + g, lane, d, 1.f, wpost);
      if (p.gate_kind == kGateFull)
        load8<T, ALIGNED>(static_cast<const T*>(p.gate) + row * p.ldg, g0 + g, lane, d, gate);
      else
        load_weight<T, ALIGNED>(p.gate_kind == kGateChannel ? static_cast<const float*>(p.gate) : nullptr, g0 + g,
                                lane, d, 1.f, gate);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (p.dy == nullptr) dy[g][i] = 0.f;
        const float c = p.h != nullptr ? p.alpha * gate[i] * (h[g][i] * rh * wpost[i]) : 0.f;
        const float y = p.beta * x[g][i] + gr * c;
        x[g][i] = y * ry;  // yh
        const float u = p.dn != nullptr ? dn[g][i] * wpre[i] : 0.f;
        if (p.dn != nullptr) sum_pre[g][i] += dn[g][i] * x[g][i];
        dn[g][i] = u;
        s[0] += u * x[g][i];
        s[1] += c * dy[g][i];
        s[2] += c * u;
        s[3] += c * x[g][i];
      }
    }
    cta_sum<4>(s, red, par);
    const float m = s[0] * inv_d;
    const float cy = s[1] + ry * (s[2] - m * s[3]);  // sum c Y
    if (p.want_dgate && p.gate_kind == kGateRow && threadIdx.x == 0) static_cast<float*>(p.dgate)[row] = cy;
    const float k = gr * cy * inv_d;  // mean(alpha g b Y)
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float wpost[8], gate[8], o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) dy[g][i] += ry * (dn[g][i] - x[g][i] * m);  // Y
      if (p.dx != nullptr) {
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = p.beta * dy[g][i];
        store8<T, ALIGNED>(static_cast<T*>(p.dx) + row * d, g0 + g, lane, d, o);
      }
      if (p.h == nullptr) continue;
      load_weight<T, ALIGNED>(p.post, g0 + g, lane, d, 1.f, wpost);
      if (p.gate_kind == kGateFull)
        load8<T, ALIGNED>(static_cast<const T*>(p.gate) + row * p.ldg, g0 + g, lane, d, gate);
      else
        load_weight<T, ALIGNED>(p.gate_kind == kGateChannel ? static_cast<const float*>(p.gate) : nullptr, g0 + g,
                                lane, d, gr, gate);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float hh = h[g][i] * rh, ay = p.alpha * dy[g][i];
        const float db = gate[i] * ay;
        sum_post[g][i] += db * hh;
        const float dg = hh * wpost[i] * ay;
        sum_gate[g][i] += dg;
        gate[i] = dg;
        o[i] = p.post != nullptr ? rh * (db * wpost[i] - hh * k) : db;
      }
      if (p.dh != nullptr) store8<T, ALIGNED>(static_cast<T*>(p.dh) + row * d, g0 + g, lane, d, o);
      if (p.want_dgate && p.gate_kind == kGateFull)
        store8<T, ALIGNED>(static_cast<T*>(p.dgate) + row * d, g0 + g, lane, d, gate);
    }
  }
  if (p.part == nullptr) return;
  float* part = p.part + (int64_t)blockIdx.x * 3 * d;
#pragma unroll
  for (int g = 0; g < NG; ++g)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = col_of<T, ALIGNED>(g0 + g, lane, i);
      if (c >= d) continue;
      if (p.want_dpre) part[c] = sum_pre[g][i];
      if (p.want_dpost) part[d + c] = sum_post[g][i];
      if (p.want_dgate && p.gate_kind == kGateChannel) part[2 * d + c] = sum_gate[g][i];
    }
}

// Sums the CTAs' partial weight gradients in a fixed order: one CTA per 32 columns of one gradient.
__global__ void __launch_bounds__(256) residual_norm_finish(const float* part, int parts, int d, float* dpre,
                                                            float* dpost, float* dgate) {
  __shared__ float sm[8][32];
  float* out = blockIdx.y == 0 ? dpre : blockIdx.y == 1 ? dpost : dgate;
  if (out == nullptr) return;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float t = 0.f;
  if (c < d) {
    const float* col = part + (int64_t)blockIdx.y * d + c;
#pragma unroll 8
    for (int b = w; b < parts; b += 8) t += col[(int64_t)b * 3 * d];
  }
  sm[w][lane] = t;
  __syncthreads();
  if (w == 0 && c < d) {
#pragma unroll
    for (int k = 1; k < 8; ++k) t += sm[k][lane];
    out[c] = t;
  }
}

struct Shape {
  bool aligned;
  int groups, threads;
};

// Rows are read in 16-byte vectors where every tensor's rows start on 16 bytes.
Shape shape_of(const NormParams& p, int esize) {
  bool ok = p.d % (16 / esize) == 0;
  for (int64_t ld : {p.ldx, p.ldh, p.lddy, p.lddn, p.ldg}) ok = ok && ld % (16 / esize) == 0;
  for (const void* q : {p.x, p.h, p.dy, p.dn, (const void*)p.y, (const void*)p.n, (const void*)p.dx,
                        (const void*)p.dh})
    ok = ok && reinterpret_cast<uintptr_t>(q) % 16 == 0;
  if (p.gate_kind == kGateFull)
    ok = ok && reinterpret_cast<uintptr_t>(p.gate) % 16 == 0 && reinterpret_cast<uintptr_t>(p.dgate) % 16 == 0;
  const int per = (p.d + 255) / 256, groups = per > kMaxWarps ? 2 : 1;
  return Shape{ok, groups, (per + groups - 1) / groups * 32};
}

template <typename F>
void with_shape(const Shape& s, F&& f) {
  auto g = [&](auto al) {
    if (s.groups == 1)
      f(al, std::integral_constant<int, 1>{});
    else
      f(al, std::integral_constant<int, 2>{});
  };
  if (s.aligned)
    g(std::true_type{});
  else
    g(std::false_type{});
}

const void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

NormParams params_of(const ResidualNormArgs& a) {
  NormParams p{};
  p.x = a.x.data_ptr();
  p.rows = a.x.size(0);
  p.d = (int)a.x.size(1);
  auto ld = [](const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : int64_t(0); };
  p.ldx = ld(a.x);
  if (a.h.has_value()) {
    p.h = a.h->data_ptr();
    p.ldh = ld(*a.h);
  }
  if (a.pre.has_value()) p.pre = a.pre->data_ptr<float>();
  if (a.post.has_value()) p.post = a.post->data_ptr<float>();
  if (a.gate.has_value()) {
    p.gate = a.gate->data_ptr();
    if (a.gate_kind == kGateFull) p.ldg = ld(*a.gate);
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
    const Shape s = shape_of(p, sizeof(T));
    with_shape(s, [&](auto al, auto ng) {
      const int64_t resident = (int64_t)num_sms() * std::max(1, 2048 / s.threads);
      const unsigned grid = (unsigned)std::min<int64_t>(p.rows, resident);
      residual_norm_fwd<T, decltype(al)::value, decltype(ng)::value><<<grid, s.threads, 0, cur_stream()>>>(p);
      MT_LAUNCH_CHECK();
    });
  });
}

void residual_norm_bwd_launch(const ResidualNormArgs& a, const at::Tensor& rstd_h, const at::Tensor& rstd_y,
                              const at::Tensor& dy, const at::Tensor& dn, const at::Tensor& dx, const at::Tensor& dh,
                              const at::Tensor& dgate, const at::Tensor& dpre, const at::Tensor& dpost) {
  NormParams p = params_of(a);
  auto ld = [](const at::Tensor& t) { return t.defined() && t.size(0) > 1 ? t.stride(0) : int64_t(0); };
  p.dy = ptr(dy);
  p.lddy = ld(dy);
  p.dn = ptr(dn);
  p.lddn = ld(dn);
  p.dx = const_cast<void*>(ptr(dx));
  p.dh = const_cast<void*>(ptr(dh));
  p.dgate = const_cast<void*>(ptr(dgate));
  p.rstd_h = rstd_h.defined() ? rstd_h.data_ptr<float>() : nullptr;
  p.rstd_y = rstd_y.defined() ? rstd_y.data_ptr<float>() : nullptr;
  p.want_dpre = dpre.defined();
  p.want_dpost = dpost.defined();
  p.want_dgate = dgate.defined();
  const bool gate_sum = dgate.defined() && a.gate_kind == kGateChannel;
  const bool sums = dpre.defined() || dpost.defined() || gate_sum;
  if (p.rows == 0) {
    for (const at::Tensor* t : {&dpre, &dpost}) {
      if (t->defined()) t->zero_();
    }
    if (gate_sum) dgate.zero_();
    return;
  }
  dispatch_act(a.x.scalar_type(), [&](auto t) {
    using T = decltype(t);
    const Shape s = shape_of(p, sizeof(T));
    with_shape(s, [&](auto al, auto ng) {
      const int64_t resident = (int64_t)num_sms() * std::max(1, 1024 / s.threads);
      const unsigned grid = (unsigned)std::min<int64_t>(p.rows, resident);
      at::Tensor part;
      if (sums) {
        part = at::empty({(int64_t)grid, 3, (int64_t)p.d}, a.x.options().dtype(at::kFloat));
        p.part = part.data_ptr<float>();
      }
      residual_norm_bwd<T, decltype(al)::value, decltype(ng)::value><<<grid, s.threads, 0, cur_stream()>>>(p);
      MT_LAUNCH_CHECK();
      if (sums) {
        residual_norm_finish<<<dim3((p.d + 31) / 32, 3), 256, 0, cur_stream()>>>(
            p.part, (int)grid, p.d, dpre.defined() ? dpre.data_ptr<float>() : nullptr,
            dpost.defined() ? dpost.data_ptr<float>() : nullptr, gate_sum ? dgate.data_ptr<float>() : nullptr);
        MT_LAUNCH_CHECK();
      }
    });
  });
}

}  // namespace mtorus

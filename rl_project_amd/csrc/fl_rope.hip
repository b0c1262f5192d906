// Norms of queries and keys for each head, and their rotation by position.
//
//   y   = x r w,  r = 1 / sqrt(sum x^2 / D + eps)
//   out = R y:    (y_i, y_j) -> (y_i c - y_j s, y_i s + y_j c) for each pair,
//         c = gain cos a, s = gain sin a, a = position inv_freq
// and the gradients for an upstream g:
//   u  = R^T g    (the same with -s)
//   dw = sum over tokens and heads of u x r
//   dx = r (u w - x r^2 mean(u w x))
//
// HBM bounds both passes: every value is read once and written once.  A thread
// holds N pairs of a row (16 bytes of each half), L threads a row, and a
// work-group takes TK tokens: their angles' sines and cosines once, into LDS, for
// all heads; then the rows, 256 / L at a time.  The angle is reduced to a fraction
// of a turn in float64, so that a far position keeps its digits (a float32 product
// is off by 0.03 at 2^20 radians).
//
// 8192 tokens of 32 + 8 heads of 128, bf16: the pass 94 us (4.5 TB/s; 81 at a copy's rate),
// its kernels one by one forward 34 us, backward 58, reduction 6; 64 tokens: 5.4 us, one
// row's latency.
#include <algorithm>
#include <type_traits>

#include "fl_device.h"
#include "fl_kernels.h"

namespace fl {

namespace {

constexpr int RP_NT = 256;
constexpr int RP_MAX_PARTS = 1024;   // work-groups of the backward pass: partial sums of the weights' gradients

// The turns of a work-group's tokens: cs[tk][p] = gain (cos, sin) of pair p, (1, 0)
// from the first pair that is not rotated on.
__device__ __forceinline__ void rp_turns(const fl_rope_args& a, int64_t t0, int tk, int P, float2* cs) {
  const int R2 = static_cast<int>(a.rotated / 2);
  for (int i = threadIdx.x; i < tk * P; i += RP_NT) {
    const int t = i / P, p = i % P;
    float2 v = make_float2(1.0f, 0.0f);
    if (p < R2) {
      const int64_t pos = (a.flags & FL_ROPE_POSITIONS32) ? static_cast<const int32_t*>(a.positions)[t0 + t]
                                                          : static_cast<const int64_t*>(a.positions)[t0 + t];
      const double turns = static_cast<double>(pos) * a.inv_freq[p] * 0.15915494309189535;   // (1 / 2 pi)
      float s, c;
      sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &s, &c);
      v = make_float2(a.gain * c, a.gain * s);
    }
    cs[i] = v;
  }
}

// Where N pairs from pair p on lie in a row: VEC takes them as whole chunks.
struct RpRow {
  int P, R2, T2;      // pairs, rotated pairs, pairs behind them
  bool inter;
  __device__ __forceinline__ int first(int p) const { return inter ? 2 * p : p < R2 ? p : R2 + p; }
  __device__ __forceinline__ int second(int p) const { return inter ? 2 * p + 1 : p < R2 ? p + R2 : R2 + T2 + p; }
};

// The two chunks of N pairs from pair p on, as they lie.
template <class D>
__device__ __forceinline__ void rp_raw(const void* row, const RpRow& R, int p, uint4 (&q)[2]) {
  constexpr int ESZ = D::id == FL_DTYPE_F32 ? 4 : 2;
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  const char* c = static_cast<const char*>(row) + ESZ * R.first(p);
  const u32x4 a = *reinterpret_cast<const u32x4*>(c);
  const u32x4 b = *reinterpret_cast<const u32x4*>(R.inter ? c + 16 : static_cast<const char*>(row) + ESZ * R.second(p));
  q[0] = make_uint4(a[0], a[1], a[2], a[3]);
  q[1] = make_uint4(b[0], b[1], b[2], b[3]);
}
template <class D, int N>
__device__ __forceinline__ void rp_pairs(const uint4 (&q)[2], const RpRow& R, float (&x)[N], float (&y)[N]) {
  using C = RowChunk<D>;
  static_assert(C::N == N, "a chunk holds N values");
  float u[N], v[N];
  C::unpack(q[0], u);
  C::unpack(q[1], v);
  if (R.inter) {
#pragma unroll
    for (int e = 0; e < N / 2; ++e) {
      x[e] = u[2 * e], y[e] = u[2 * e + 1];
      x[e + N / 2] = v[2 * e], y[e + N / 2] = v[2 * e + 1];
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = u[e], y[e] = v[e];
  }
}

template <class D, bool VEC, int N>
__device__ __forceinline__ void rp_load(const void* row, const RpRow& R, int p, float (&x)[N], float (&y)[N]) {
  if (p >= R.P) {
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = y[e] = 0.0f;
  } else if constexpr (VEC) {
    uint4 q[2];
    rp_raw<D>(row, R, p, q);
    rp_pairs<D>(q, R, x, y);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      x[e] = y[e] = 0.0f;
      if (p + e < R.P) {
        if constexpr (D::id == FL_DTYPE_F32) {
          x[e] = static_cast<const float*>(row)[R.first(p + e)];
          y[e] = static_cast<const float*>(row)[R.second(p + e)];
        } else {
          x[e] = D::to_f32(static_cast<const uint16_t*>(row)[R.first(p + e)]);
          y[e] = D::to_f32(static_cast<const uint16_t*>(row)[R.second(p + e)]);
        }
      }
    }
  }
}

template <class D, int N>
__device__ __forceinline__ uint4 rp_pack(const float (&x)[N]) {
  if constexpr (D::id == FL_DTYPE_F32)
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  else
    return make_uint4(D::from_f32(x[0]) | (D::from_f32(x[1]) << 16), D::from_f32(x[2]) | (D::from_f32(x[3]) << 16),
                      D::from_f32(x[4]) | (D::from_f32(x[5]) << 16), D::from_f32(x[6]) | (D::from_f32(x[7]) << 16));
}

template <class D, bool VEC, int N>
__device__ __forceinline__ void rp_store(void* row, const RpRow& R, int p, const float (&x)[N], const float (&y)[N]) {
  if (p >= R.P) return;
  if constexpr (VEC) {
    constexpr int ESZ = D::id == FL_DTYPE_F32 ? 4 : 2;
    float u[N], v[N];
    if (R.inter) {
#pragma unroll
      for (int e = 0; e < N / 2; ++e) {
        u[2 * e] = x[e], u[2 * e + 1] = y[e];
        v[2 * e] = x[e + N / 2], v[2 * e + 1] = y[e + N / 2];
      }
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) u[e] = x[e], v[e] = y[e];
    }
    char* c = static_cast<char*>(row) + ESZ * R.first(p);
    *reinterpret_cast<uint4*>(c) = rp_pack<D>(u);
    *reinterpret_cast<uint4*>(R.inter ? c + 16 : static_cast<char*>(row) + ESZ * R.second(p)) = rp_pack<D>(v);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (p + e < R.P) {
        if constexpr (D::id == FL_DTYPE_F32) {
          static_cast<float*>(row)[R.first(p + e)] = x[e];
          static_cast<float*>(row)[R.second(p + e)] = y[e];
        } else {
          static_cast<uint16_t*>(row)[R.first(p + e)] = static_cast<uint16_t>(D::from_f32(x[e]));
          static_cast<uint16_t*>(row)[R.second(p + e)] = static_cast<uint16_t>(D::from_f32(y[e]));
        }
      }
  }
}

template <int N>
__device__ __forceinline__ float rp_sum(float v, int L) {
#pragma unroll 1
  for (int m = 1; m < L; m <<= 1) v += shfl_xor(v, m);
  return v;
}

template <class D>
__device__ __forceinline__ char* rp_at(const void* p, int64_t i) {
  return static_cast<char*>(const_cast<void*>(p)) + i * (D::id == FL_DTYPE_F32 ? 4 : 2);
}

// The weights of a thread's pairs (1 without), which need no alignment.
template <class W, int N>
__device__ __forceinline__ void rp_weights(const void* w, const RpRow& R, int p, float (&x)[N], float (&y)[N]) {
  if (w != nullptr) rp_load<W, false>(w, R, p, x, y);
  else
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = y[e] = 1.0f;
}

// The other value's share of a rotated value: none in channels behind the rotated ones,
// which are no pair, so that infinity and NaN stay in theirs (0 times them is NaN; -0
// leaves every value as it is).  (TAIL: there are such channels; a test of it in the
// loop cost the training step of 8192 tokens 2.4 us of 94.)
template <bool TAIL>
__device__ __forceinline__ float rp_share(const RpRow& R, int p, float v) {
  return TAIL && p >= R.R2 ? -0.0f : v;
}

__device__ __forceinline__ RpRow rp_row(const fl_rope_args& a) {
  const int P = static_cast<int>(a.dim / 2), R2 = static_cast<int>(a.rotated / 2);
  return RpRow{P, R2, P - R2, (a.flags & FL_ROPE_INTERLEAVED) != 0};
}

}  // namespace

template <class D, class W, bool VEC, bool TAIL>
__global__ __launch_bounds__(RP_NT) void k_rope(const fl_rope_args a, int L, int TK) {
  constexpr int N = RowChunk<D>::N;
  __shared__ float2 cs[1024], ws[2][FL_ROPE_MAX_DIM / 2];   // the turns; the pairs' weights (queries', keys')
  const RpRow R = rp_row(a);
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * TK;
  const int tk = static_cast<int>(min(static_cast<int64_t>(TK), a.tokens - t0));
  const int p = (threadIdx.x & (L - 1)) * N, g = threadIdx.x / L, GR = RP_NT / L;
  const int H = static_cast<int>(a.heads), K = static_cast<int>(a.kv_heads), nq = tk * H, n = nq + tk * K;
  // row i of the tokens': the queries' first
  struct Row {
    const void* x;
    void* out;
    int t;
  };
  const auto row = [&](int i) {
    const bool key = i >= nq;
    const int j = key ? i - nq : i, heads = key ? K : H, t = j / heads, h = j - t * heads;
    const int64_t to = ((t0 + t) * heads + h) * a.dim;
    return key ? Row{rp_at<D>(a.k, (t0 + t) * a.k_ld + h * a.k_hs), rp_at<D>(a.out_k, to), t}
               : Row{rp_at<D>(a.q, (t0 + t) * a.q_ld + h * a.q_hs), rp_at<D>(a.out_q, to), t};
  };
  // the first row is on its way while the angles are taken, and each next one while
  // one is worked on
  uint4 raw[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  Row at = {};
  const auto fetch = [&](int i) {
    at = row(i);
    if (VEC && p < R.P) rp_raw<D>(at.x, R, p, raw);
  };
  if (g < n) fetch(g);
  if (a.norm)
    for (int i = threadIdx.x; i < 2 * R.P; i += RP_NT) {
      const int key = i >= R.P, pair = i - key * R.P;
      float w0[1], w1[1];
      rp_weights<W>(key ? a.k_weight : a.q_weight, R, pair, w0, w1);
      ws[key][pair] = make_float2(w0[0], w1[0]);
    }
  rp_turns(a, t0, tk, R.P, cs);
  __syncthreads();
  const float inv = 1.0f / static_cast<float>(a.dim);
  for (int i = g; i < n; i += GR) {
    float x0[N], x1[N];
    if constexpr (VEC) rp_pairs<D>(raw, R, x0, x1);
    else rp_load<D, false>(at.x, R, p, x0, x1);
    const Row now = at;
    if (i + GR < n) fetch(i + GR);
    if (a.norm) {
      float s = 0.0f;
#pragma unroll
      for (int e = 0; e < N; ++e) s = fmaf(x0[e], x0[e], fmaf(x1[e], x1[e], s));
      const float r = 1.0f / sqrtf(fmaf(rp_sum<N>(s, L), inv, a.eps));
      const float2* w = ws[i >= nq];
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float2 y = w[min(p + e, R.P - 1)];
        x0[e] *= r * y.x, x1[e] *= r * y.y;
      }
    }
    float y0[N], y1[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float2 c = cs[now.t * R.P + min(p + e, R.P - 1)];
      // (the same fused products in every variant: a row's results do not depend on how
      // it was read)
      y0[e] = fmaf(x0[e], c.x, rp_share<TAIL>(R, p + e, -(x1[e] * c.y)));
      y1[e] = fmaf(rp_share<TAIL>(R, p + e, x0[e]), c.y, x1[e] * c.x);   // (c.y is 0 there)
    }
    rp_store<D, VEC>(now.out, R, p, y0, y1);
  }
}

// One side a work-group (blockIdx.y 0: queries, 1: keys): the sums of one weight's
// gradient in registers (both sides at once: 125 us for the training step of 8192
// tokens, so 102).
template <class D, class W, bool VEC, bool TAIL>
__global__ __launch_bounds__(RP_NT, 4) void k_rope_grad(const fl_rope_grad_args b, int L, int TK) {
  constexpr int N = RowChunk<D>::N;
  const fl_rope_args& a = b.fwd;
  __shared__ float2 cs[1024];
  __shared__ float sum[RP_NT / WAVE][FL_ROPE_MAX_DIM];
  const bool key = blockIdx.y != 0;
  const int heads = static_cast<int>(key ? a.kv_heads : a.heads);
  if (heads == 0 && (key ? b.out_dwk : b.out_dwq) == nullptr) return;   // (a weight without heads has gradient 0)
  const void* x = key ? a.k : a.q;
  const void* grad = key ? b.grad_k : b.grad_q;
  const int64_t ld = key ? a.k_ld : a.q_ld, hs = key ? a.k_hs : a.q_hs;
  void* out = key ? a.out_k : a.out_q;
  const RpRow R = rp_row(a);
  const int p = (threadIdx.x & (L - 1)) * N, g = threadIdx.x / L, GR = RP_NT / L;
  const float inv = 1.0f / static_cast<float>(a.dim);
  float w0[N], w1[N], d0[N], d1[N];
  rp_weights<W>(a.norm ? (key ? a.k_weight : a.q_weight) : nullptr, R, p, w0, w1);
#pragma unroll
  for (int e = 0; e < N; ++e) d0[e] = d1[e] = 0.0f;
  for (int64_t t0 = static_cast<int64_t>(blockIdx.x) * TK; t0 < a.tokens; t0 += static_cast<int64_t>(gridDim.x) * TK) {
    const int tk = static_cast<int>(min(static_cast<int64_t>(TK), a.tokens - t0));
    __syncthreads();   // (the last tokens' angles have been read)
    rp_turns(a, t0, tk, R.P, cs);
    __syncthreads();
    for (int i = g; i < tk * heads; i += GR) {
      const int t = i / heads, h = i - t * heads;
      const int64_t at = ((t0 + t) * heads + h) * a.dim;
      float x0[N], x1[N], g0[N], g1[N], u0[N], u1[N];
      const char* xr = rp_at<D>(x, (t0 + t) * ld + h * hs);
      if constexpr (VEC) {   // (both rows on their way before either is unpacked)
        uint4 qg[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)}, qx[2] = {qg[0], qg[0]};
        if (p < R.P) {
          if (grad != nullptr) rp_raw<D>(rp_at<D>(grad, at), R, p, qg);
          if (a.norm) rp_raw<D>(xr, R, p, qx);
        }
        rp_pairs<D>(qg, R, g0, g1);
        rp_pairs<D>(qx, R, x0, x1);
      } else {
        if (grad != nullptr) rp_load<D, false>(rp_at<D>(grad, at), R, p, g0, g1);
        else
#pragma unroll
          for (int e = 0; e < N; ++e) g0[e] = g1[e] = 0.0f;
        if (a.norm) rp_load<D, false>(xr, R, p, x0, x1);
      }
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float2 c = cs[t * R.P + min(p + e, R.P - 1)];
        u0[e] = fmaf(g0[e], c.x, rp_share<TAIL>(R, p + e, g1[e] * c.y));
        u1[e] = fmaf(g1[e], c.x, rp_share<TAIL>(R, p + e, -(g0[e] * c.y)));
      }
      if (a.norm) {
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < N; ++e) s = fmaf(x0[e], x0[e], fmaf(x1[e], x1[e], s));
        const float r = 1.0f / sqrtf(fmaf(rp_sum<N>(s, L), inv, a.eps));
        float dot = 0.0f;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          x0[e] *= r, x1[e] *= r;
          d0[e] = fmaf(u0[e], x0[e], d0[e]);
          d1[e] = fmaf(u1[e], x1[e], d1[e]);
          u0[e] *= w0[e], u1[e] *= w1[e];
          dot = fmaf(u0[e], x0[e], fmaf(u1[e], x1[e], dot));
        }
        dot = rp_sum<N>(dot, L) * inv;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          u0[e] = r * fmaf(-x0[e], dot, u0[e]);
          u1[e] = r * fmaf(-x1[e], dot, u1[e]);
        }
      }
      if (out != nullptr) rp_store<D, VEC>(rp_at<D>(out, at), R, p, u0, u1);
    }
  }
  if ((key ? b.out_dwk : b.out_dwq) == nullptr) return;
  // the row groups' sums: over a wave's by exchange, then over the waves
  float* part = static_cast<float*>(b.workspace) + (static_cast<int64_t>(blockIdx.x) * 2 + blockIdx.y) * a.dim;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    for (int m = L; m < WAVE; m <<= 1) {
      d0[e] += shfl_xor(d0[e], m);
      d1[e] += shfl_xor(d1[e], m);
    }
    if ((threadIdx.x & (WAVE - 1)) < L && p + e < R.P) {
      sum[threadIdx.x / WAVE][R.first(p + e)] = d0[e];
      sum[threadIdx.x / WAVE][R.second(p + e)] = d1[e];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.dim; i += RP_NT) part[i] = (sum[0][i] + sum[1][i]) + (sum[2][i] + sum[3][i]);
}

// The partial sums added: one work-group per 64 columns of dwq (blockIdx.y 0) or
// dwk (1), a wave per 16th of the parts, in float64.
constexpr int RP_RW = 16;
template <class W>
__global__ __launch_bounds__(RP_RW * WAVE) void k_rope_reduce(const fl_rope_grad_args b, int parts) {
  __shared__ double s[RP_RW][WAVE];
  const int n = static_cast<int>(b.fwd.dim), lane = threadIdx.x & (WAVE - 1), w = threadIdx.x / WAVE;
  const int i = blockIdx.x * WAVE + lane;
  void* out = blockIdx.y == 0 ? b.out_dwq : b.out_dwk;
  if (out == nullptr) return;
  double v = 0.0;
  if (i < n) {
    const float* p = static_cast<const float*>(b.workspace) + static_cast<int64_t>(blockIdx.y) * n + i;
#pragma unroll 8
    for (int q = w; q < parts; q += RP_RW) v += static_cast<double>(p[static_cast<int64_t>(q) * 2 * n]);
  }
  s[w][lane] = v;
  __syncthreads();
  if (w != 0 || i >= n) return;
#pragma unroll
  for (int q = 1; q < RP_RW; ++q) v += s[q][lane];
  if constexpr (W::id == FL_DTYPE_F32) static_cast<float*>(out)[i] = static_cast<float>(v);
  else static_cast<uint16_t*>(out)[i] = static_cast<uint16_t>(W::from_f32(static_cast<float>(v)));
}

namespace {

template <class F>
void rp_types(int dtype, int wdtype, F&& f) {
  if (dtype == FL_DTYPE_F32) f(F32{}, F32{});
  else if (dtype == FL_DTYPE_BF16 && wdtype == FL_DTYPE_F32) f(BF16{}, F32{});
  else if (dtype == FL_DTYPE_BF16) f(BF16{}, BF16{});
  else if (wdtype == FL_DTYPE_F32) f(F16{}, F32{});
  else f(F16{}, F16{});
}

// Whole 16-byte chunks: rows that start and pairs that lie on them.
bool rp_vector(const fl_rope_args& a, int N, std::initializer_list<const void*> more) {
  const int64_t R2 = a.rotated / 2, T2 = (a.dim - a.rotated) / 2;
  if (a.flags & FL_ROPE_INTERLEAVED ? a.dim % (2 * N) != 0 : R2 % N != 0 || T2 % N != 0) return false;
  uintptr_t bits = 0;
  const uintptr_t esz = a.dtype == FL_DTYPE_F32 ? 4 : 2;
  if (a.q) bits |= reinterpret_cast<uintptr_t>(a.q) | static_cast<uintptr_t>(a.q_ld) * esz | static_cast<uintptr_t>(a.q_hs) * esz;
  if (a.k) bits |= reinterpret_cast<uintptr_t>(a.k) | static_cast<uintptr_t>(a.k_ld) * esz | static_cast<uintptr_t>(a.k_hs) * esz;
  bits |= reinterpret_cast<uintptr_t>(a.out_q) | reinterpret_cast<uintptr_t>(a.out_k);
  for (const void* p : more) bits |= reinterpret_cast<uintptr_t>(p);
  return bits % 16 == 0;
}

// Threads of a row: a power of two that holds its pairs.
int rp_lanes(int64_t dim, int N) {
  int L = 1;
  while (L * N < dim / 2) L *= 2;
  return L;
}
// Tokens of a work-group: 4 share one round of sines and cosines where that still
// leaves four work-groups for every CU (8192 tokens: 34 us against 39 with one; 512: 10
// against 6.5).
int rp_tokens(int64_t tokens) { return tokens >= 4096 ? 4 : 1; }

}  // namespace

int64_t rope_grad_parts(int64_t tokens) {
  const int TK = rp_tokens(tokens);
  return std::min<int64_t>((tokens + TK - 1) / TK, RP_MAX_PARTS);
}

hipError_t launch_rope(const fl_rope_args& a, hipStream_t s) {
  rp_types(a.dtype, a.wdtype, [&](auto d, auto w) {
    using D = decltype(d);
    constexpr int N = RowChunk<D>::N;
    const int L = rp_lanes(a.dim, N), TK = rp_tokens(a.tokens);
    const dim3 grid(static_cast<unsigned>((a.tokens + TK - 1) / TK));
    using W = decltype(w);
    const auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(RP_NT), 0, s, a, L, TK); };
    if (rp_vector(a, N, {})) a.rotated < a.dim ? run(k_rope<D, W, true, true>) : run(k_rope<D, W, true, false>);
    else a.rotated < a.dim ? run(k_rope<D, W, false, true>) : run(k_rope<D, W, false, false>);
  });
  return hipGetLastError();
}

hipError_t launch_rope_grad(const fl_rope_grad_args& b, hipStream_t s) {
  const fl_rope_args& a = b.fwd;
  rp_types(a.dtype, a.wdtype, [&](auto d, auto w) {
    using D = decltype(d);
    using W = decltype(w);
    constexpr int N = RowChunk<D>::N;
    const int L = rp_lanes(a.dim, N), TK = rp_tokens(a.tokens);
    const int parts = static_cast<int>(rope_grad_parts(a.tokens));
    if (parts > 0) {
      const auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(parts, 2), dim3(RP_NT), 0, s, b, L, TK); };
      if (rp_vector(a, N, {b.grad_q, b.grad_k})) a.rotated < a.dim ? run(k_rope_grad<D, W, true, true>) : run(k_rope_grad<D, W, true, false>);
      else a.rotated < a.dim ? run(k_rope_grad<D, W, false, true>) : run(k_rope_grad<D, W, false, false>);
    }
    if (b.out_dwq || b.out_dwk)
      hipLaunchKernelGGL(k_rope_reduce<W>, dim3(static_cast<unsigned>((a.dim + WAVE - 1) / WAVE), 2), dim3(RP_RW * WAVE), 0, s, b,
                         parts);
  });
  return hipGetLastError();
}

}  // namespace fl

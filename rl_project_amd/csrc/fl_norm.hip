// Layer norm over the last dimension, forward and backward.
//
//   y  = (x - mean) rstd w + b,   mean = sum x / D,
//        rstd = 1 / sqrt(sum (x - mean)^2 / D + eps)
//   dx = rstd (g - mean(g) - xh mean(g xh)),  g = dy w,  xh = (x - mean) rstd
//   dw = sum over rows of dy xh,   db = sum over rows of dy
//
// A row lives in the registers of G threads (64, 256 or 1024 by its length, U
// chunks of 16 bytes each), so that HBM, which bounds both passes, is read
// once: mean, then the squares about it, then the result.  Statistics and sums
// in float32; one rounding to the type of x (dw, db: of the weight) at the end.
#include <algorithm>
#include <type_traits>

#include "fl_device.h"
#include "fl_kernels.h"

namespace fl {

namespace {

constexpr int LN_NT = 256;    // forward threads (G = 1024: 1024)
constexpr int LN_BT = 512;    // backward threads (G = 1024: 1024)
constexpr int LN_MAX_PARTS = 256;   // work-groups of the backward pass: partial sums of dw and db

// 16 bytes (N values) of a row at element i, as floats; the last value of an
// odd 16-bit row by itself (the range check goes by dwords).  Past the row: 0.
template <class D>
__device__ __forceinline__ void ln_load(__amdgpu_buffer_rsrc_t r, int i, int n, float (&x)[RowChunk<D>::N]) {
  using C = RowChunk<D>;
  constexpr int ESZ = D::id == FL_DTYPE_F32 ? 4 : 2;
  C::unpack(buf_load16(r, static_cast<uint32_t>(ESZ * i), 0u), x);
  if (D::id != FL_DTYPE_F32 && (n & 1) && i < n && n - i < C::N) {
#pragma unroll
    for (int e = 0; e < C::N; e += 2)
      if (i + e == n - 1) x[e] = C::elem(r, n - 1);
  }
}
// N values of a weight row of another chunk size (float32 beside 16-bit x).
template <class W, int N>
__device__ __forceinline__ void ln_load_w(__amdgpu_buffer_rsrc_t r, int i, int n, float (&x)[N]) {
  constexpr int M = RowChunk<W>::N;
  static_assert(N % M == 0, "whole chunks");
#pragma unroll
  for (int c = 0; c < N / M; ++c) {
    float t[M];
    ln_load<W>(r, i + c * M, n, t);
#pragma unroll
    for (int e = 0; e < M; ++e) x[c * M + e] = t[e];
  }
}
template <class D>
__device__ __forceinline__ void ln_store(__amdgpu_buffer_rsrc_t r, int i, int n, const float (&x)[RowChunk<D>::N]) {
  constexpr int N = RowChunk<D>::N;
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  if (n - i >= N) {
    u32x4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (D::id == FL_DTYPE_F32) o[j] = __float_as_uint(x[j]);
      else o[j] = D::from_f32(x[2 * j]) | (D::from_f32(x[2 * j + 1]) << 16);
    }
    __builtin_amdgcn_raw_buffer_store_b128(o, r, (D::id == FL_DTYPE_F32 ? 4 : 2) * i, 0, 0);
  } else {   // the row's last chunk, value by value
#pragma unroll
    for (int e = 0; e < N; ++e) {
      if (i + e >= n) break;
      if constexpr (D::id == FL_DTYPE_F32)
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(x[e]), r, 4 * (i + e), 0, 0);
      else
        __builtin_amdgcn_raw_buffer_store_b16(static_cast<short>(D::from_f32(x[e])), r, 2 * (i + e), 0, 0);
    }
  }
}

template <class D>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t ln_row(const void* p, int64_t r, int64_t ld, int n) {
  constexpr int64_t ESZ = D::id == FL_DTYPE_F32 ? 4 : 2;
  return row_rsrc(static_cast<const char*>(p) + r * ld * ESZ, static_cast<uint32_t>(n * ESZ));
}

// Sum over the G threads of a row; `red` holds two turns of one float per wave
// of the work-group, so that one barrier per sum is enough.
template <int G>
__device__ __forceinline__ float ln_sum(float v, float* red, int& turn) {
  v = wave_reduce(v, OpAdd());
  if constexpr (G > WAVE) {
    constexpr int GW = G / WAVE;
    const int nw = blockDim.x / WAVE, w = threadIdx.x / WAVE;
    float* t = red + turn * nw;
    if ((threadIdx.x & (WAVE - 1)) == 0) t[w] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < GW; ++i) v += t[w / GW * GW + i];
    turn ^= 1;
  }
  return v;
}

}  // namespace

// Every work-group takes rows p, p + grid, ... of its G-thread groups (all
// groups of a work-group step together: those past the last row do the work
// of none).
template <class D, class W, int G, int U>
__global__ __launch_bounds__(G == 1024 ? 1024 : LN_NT) void k_norm(const fl_norm_args a) {
  constexpr int N = RowChunk<D>::N;
  constexpr int NT_ = G == 1024 ? 1024 : LN_NT, GR = NT_ / G;
  __shared__ float red[2 * NT_ / WAVE];
  const int n = static_cast<int>(a.dim), g = threadIdx.x / G, t = threadIdx.x % G;
  const float inv = 1.0f / static_cast<float>(n);
  float w[U][N], b[U][N];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = N * (t + G * u);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      w[u][e] = 1.0f;
      b[u][e] = 0.0f;
    }
    if (a.weight) ln_load_w<W>(ln_row<W>(a.weight, 0, 0, n), i, n, w[u]);
    if (a.bias) ln_load_w<W>(ln_row<W>(a.bias, 0, 0, n), i, n, b[u]);
  }
  int turn = 0;
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * GR; r0 < a.rows; r0 += static_cast<int64_t>(gridDim.x) * GR) {
    const int64_t r = r0 + g;
    const bool on = r < a.rows;
    const __amdgpu_buffer_rsrc_t rx = ln_row<D>(a.x, on ? r : 0, a.ld, on ? n : 0);
    float x[U][N], s = 0.0f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      ln_load<D>(rx, N * (t + G * u), on ? n : 0, x[u]);
#pragma unroll
      for (int e = 0; e < N; ++e) s += x[u][e];
    }
    const float mean = ln_sum<G>(s, red, turn) * inv;
    float v = 0.0f;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        x[u][e] -= mean;
        const float c = N * (t + G * u) + e < n ? x[u][e] : 0.0f;
        v = fmaf(c, c, v);
      }
    const float rstd = 1.0f / sqrtf(fmaf(ln_sum<G>(v, red, turn), inv, a.eps));
    if (!on) continue;
    if (t == 0) {
      if (a.out_mean) a.out_mean[r] = mean;
      if (a.out_rstd) a.out_rstd[r] = rstd;
    }
    const __amdgpu_buffer_rsrc_t ry = ln_row<D>(a.out, r, a.out_ld, n);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = N * (t + G * u);
      if (i >= n) continue;
      float y[N];
#pragma unroll
      for (int e = 0; e < N; ++e) y[e] = fmaf(x[u][e] * rstd, w[u][e], b[u][e]);
      ln_store<D>(ry, i, n, y);
    }
  }
}

// Backward.  A work-group's groups keep dw and db of the rows they take in
// registers; at the end the groups' sums are added in LDS, in order, and stored
// as one partial row of each (WG: they are asked for).
template <class D, class W, int G, int U, bool WG>
__global__ __launch_bounds__(G == 1024 ? 1024 : LN_BT) void k_norm_grad(const fl_norm_grad_args a, float* part) {
  constexpr int N = RowChunk<D>::N;
  constexpr int NT_ = G == 1024 ? 1024 : LN_BT, GR = NT_ / G;
  __shared__ float red[2 * NT_ / WAVE], red2[2 * NT_ / WAVE];
  const int n = static_cast<int>(a.dim), g = threadIdx.x / G, t = threadIdx.x % G;
  const float inv = 1.0f / static_cast<float>(n);
  float dw[U][N], db[U][N];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int e = 0; e < N; ++e) dw[u][e] = db[u][e] = 0.0f;
  int turn = 0, turn2 = 0;
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * GR; r0 < a.rows; r0 += static_cast<int64_t>(gridDim.x) * GR) {
    const int64_t r = r0 + g;
    const bool on = r < a.rows;
    const int m = on ? n : 0;
    const __amdgpu_buffer_rsrc_t rx = ln_row<D>(a.x, on ? r : 0, a.ld, m);
    const __amdgpu_buffer_rsrc_t rd = ln_row<D>(a.grad, on ? r : 0, a.grad_ld, m);
    const float mean = on ? a.mean[r] : 0.0f, rstd = on ? a.rstd[r] : 0.0f;
    float x[U][N], d[U][N], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      ln_load<D>(rx, N * (t + G * u), m, x[u]);
      ln_load<D>(rd, N * (t + G * u), m, d[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = N * (t + G * u);
      float w[N];
#pragma unroll
      for (int e = 0; e < N; ++e) w[e] = 1.0f;
      if (a.weight) ln_load_w<W>(ln_row<W>(a.weight, 0, 0, n), i, n, w);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        // (past the row dy is 0, and x - mean is not used)
        const float xh = i + e < m ? (x[u][e] - mean) * rstd : 0.0f;
        if (WG) {
          dw[u][e] = fmaf(d[u][e], xh, dw[u][e]);
          db[u][e] += d[u][e];
        }
        x[u][e] = xh;
        d[u][e] *= w[e];
        s1 += d[u][e];
        s2 = fmaf(d[u][e], xh, s2);
      }
    }
    if (a.out_dx == nullptr) continue;
    const float c1 = ln_sum<G>(s1, red, turn) * inv, c2 = ln_sum<G>(s2, red2, turn2) * inv;
    if (!on) continue;
    const __amdgpu_buffer_rsrc_t ro = ln_row<D>(a.out_dx, r, a.out_ld, n);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = N * (t + G * u);
      if (i >= n) continue;
      float o[N];
#pragma unroll
      for (int e = 0; e < N; ++e) o[e] = rstd * (d[u][e] - c1 - x[u][e] * c2);
      ln_store<D>(ro, i, n, o);
    }
  }
  if constexpr (WG) {
    float* pw = part + static_cast<int64_t>(blockIdx.x) * 2 * n;
    if constexpr (GR == 1) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const int i = N * (t + G * u) + e;
          if (i < n) {
            pw[i] = dw[u][e];
            pw[n + i] = db[u][e];
          }
        }
    } else {
      // [U][N][G]: a wave's accesses side by side
      __shared__ float sum[2 * U * N * G];
#pragma unroll 1
      for (int q = 0; q < GR; ++q) {
        if (g == q) {
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < N; ++e) {
              float* p = sum + (u * N + e) * G + t;
              p[0] = q == 0 ? dw[u][e] : p[0] + dw[u][e];
              p[U * N * G] = q == 0 ? db[u][e] : p[U * N * G] + db[u][e];
            }
        }
        __syncthreads();
      }
      for (int i = threadIdx.x; i < n; i += NT_) {
        const int c = i / N;   // chunk: thread c % G, turn c / G
        const float* p = sum + (c / G * N + i % N) * G + c % G;
        pw[i] = p[0];
        pw[n + i] = p[U * N * G];
      }
    }
  }
}

// The partial rows added: one work-group per 64 columns of dw (blockIdx.y 0) or
// db (1), a wave per 16th of the rows, in float64.
constexpr int LN_RW = 16;
template <class W>
__global__ __launch_bounds__(LN_RW * WAVE) void k_norm_reduce(const fl_norm_grad_args a, const float* part, int parts) {
  __shared__ double s[LN_RW][WAVE];
  const int n = static_cast<int>(a.dim), lane = threadIdx.x & (WAVE - 1), w = threadIdx.x / WAVE;
  const int i = blockIdx.x * WAVE + lane;
  void* out = blockIdx.y == 0 ? a.out_dweight : a.out_dbias;
  if (out == nullptr) return;
  double v = 0.0;
  if (i < n) {
    const float* p = part + static_cast<int64_t>(blockIdx.y) * n + i;
#pragma unroll 4
    for (int q = w; q < parts; q += LN_RW) v += static_cast<double>(p[static_cast<int64_t>(q) * 2 * n]);
  }
  s[w][lane] = v;
  __syncthreads();
  if (w != 0 || i >= n) return;
#pragma unroll
  for (int q = 1; q < LN_RW; ++q) v += s[q][lane];
  if constexpr (W::id == FL_DTYPE_F32) static_cast<float*>(out)[i] = static_cast<float>(v);
  else static_cast<uint16_t*>(out)[i] = static_cast<uint16_t>(W::from_f32(static_cast<float>(v)));
}

namespace {

// f(G, U): the threads and chunks that hold a row of n values of N per chunk
template <int N, class F>
void ln_shape(int64_t n, F&& f) {
  using std::integral_constant;
  if (n <= 64 * N) f(integral_constant<int, 64>{}, integral_constant<int, 1>{});
  else if (n <= 64 * N * 2) f(integral_constant<int, 64>{}, integral_constant<int, 2>{});
  else if (n <= 64 * N * 4) f(integral_constant<int, 64>{}, integral_constant<int, 4>{});
  else if (n <= 256 * N * 2) f(integral_constant<int, 256>{}, integral_constant<int, 2>{});
  else if (n <= 256 * N * 4) f(integral_constant<int, 256>{}, integral_constant<int, 4>{});
  else if (N == 8 || n <= 1024 * N * 2) f(integral_constant<int, 1024>{}, integral_constant<int, 2>{});
  else f(integral_constant<int, 1024>{}, integral_constant<int, N == 8 ? 2 : 4>{});
}
static_assert(FL_NORM_MAX_DIM <= 1024 * 8 * 2 && FL_NORM_MAX_DIM <= 1024 * 4 * 4, "the longest row fits");

template <class F>
void ln_types(int dtype, int wdtype, F&& f) {
  if (dtype == FL_DTYPE_F32) f(F32{}, F32{});
  else if (dtype == FL_DTYPE_BF16 && wdtype == FL_DTYPE_F32) f(BF16{}, F32{});
  else if (dtype == FL_DTYPE_BF16) f(BF16{}, BF16{});
  else if (wdtype == FL_DTYPE_F32) f(F16{}, F32{});
  else f(F16{}, F16{});
}

// Work-groups of the backward pass: a CU's worth of rows each at most
int ln_parts(int64_t rows, int64_t dim, int dtype) {
  const int N = dtype == FL_DTYPE_F32 ? 4 : 8;
  const int64_t gr = dim <= 64 * N * 4 ? LN_BT / 64 : dim <= 256 * N * 4 ? LN_BT / 256 : 1;
  return static_cast<int>(std::min<int64_t>((rows + gr - 1) / gr, LN_MAX_PARTS));
}

}  // namespace

size_t norm_grad_workspace_bytes(int64_t rows, int64_t dim, int dtype) {
  return static_cast<size_t>(ln_parts(rows, dim, dtype)) * 2 * static_cast<size_t>(dim) * sizeof(float);
}

hipError_t launch_norm(const fl_norm_args& a, hipStream_t s) {
  ln_types(a.dtype, a.wdtype, [&](auto d, auto w) {
    using D = decltype(d);
    ln_shape<RowChunk<D>::N>(a.dim, [&](auto g, auto u) {
      constexpr int G = decltype(g)::value, NT_ = G == 1024 ? 1024 : LN_NT, GR = NT_ / G;
      // (2048 threads per CU; more rows loop, with the weights in registers)
      const unsigned grid = static_cast<unsigned>(std::min<int64_t>((a.rows + GR - 1) / GR, 256 * 2048 / NT_));
      hipLaunchKernelGGL((k_norm<D, decltype(w), G, decltype(u)::value>), dim3(grid), dim3(NT_), 0, s, a);
    });
  });
  return hipGetLastError();
}

hipError_t launch_norm_grad(const fl_norm_grad_args& a, hipStream_t s) {
  const bool wg = a.out_dweight != nullptr || a.out_dbias != nullptr;
  const int parts = ln_parts(a.rows, a.dim, a.dtype);
  float* part = static_cast<float*>(a.workspace);
  ln_types(a.dtype, a.wdtype, [&](auto d, auto w) {
    using D = decltype(d);
    using W = decltype(w);
    if (parts > 0 && (wg || a.out_dx != nullptr))
      ln_shape<RowChunk<D>::N>(a.dim, [&](auto g, auto u) {
        constexpr int G = decltype(g)::value, NT_ = G == 1024 ? 1024 : LN_BT;
        if (wg) hipLaunchKernelGGL((k_norm_grad<D, W, G, decltype(u)::value, true>), dim3(parts), dim3(NT_), 0, s, a, part);
        else hipLaunchKernelGGL((k_norm_grad<D, W, G, decltype(u)::value, false>), dim3(parts), dim3(NT_), 0, s, a, part);
      });
    if (wg)
      hipLaunchKernelGGL(k_norm_reduce<W>, dim3(static_cast<unsigned>((a.dim + WAVE - 1) / WAVE), 2), dim3(LN_RW * WAVE), 0, s,
                         a, part, parts);
  });
  return hipGetLastError();
}

}  // namespace fl

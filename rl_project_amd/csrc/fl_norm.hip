// Layer norm over the last dimension, forward and backward.
//
//   y  = (x - mean) rstd w + b,   mean = sum x / D,
//        rstd = 1 / sqrt(sum (x - mean)^2 / D + eps)
//   dx = rstd (g - mean(g) - xh mean(g xh)),  g = dy w,  xh = (x - mean) rstd
//   dw = sum over rows of dy xh,   db = sum over rows of dy
//
// A row lives in the registers of G threads (64 to 1024 by its length, U chunks
// of 16 bytes each), so that HBM, which bounds both passes, is read once: mean,
// then the squares about it, then the result; the next row's values are on
// their way meanwhile (the sums' barriers and the loads took turns before:
// backward of bf16 4096x4096 32.5 us, 22.6 so).  Statistics and sums in
// float32; one rounding to the type of x (dw, db: of the weight) at the end.
// bf16 4096x4096: forward 15.0 to 16.5 us (4.5 to 4.1 TB/s of 67 MB), backward 22.6
// to 23.9 us (4.5 to 4.2 TB/s of 101 MB) and 3.9 us for the partial sums; 64x4096:
// 3.9 to 4.3 us, a launch's length.
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
__device__ __forceinline__ uint4 ln_raw(__amdgpu_buffer_rsrc_t r, int i) {
  return buf_load16(r, static_cast<uint32_t>(D::id == FL_DTYPE_F32 ? 4 * i : 2 * i), 0u);
}
template <class D>
__device__ __forceinline__ void ln_unpack(uint4 q, __amdgpu_buffer_rsrc_t r, int i, int n, float (&x)[RowChunk<D>::N]) {
  using C = RowChunk<D>;
  C::unpack(q, x);
  if (D::id != FL_DTYPE_F32 && (n & 1) && i < n && n - i < C::N) {
    const float last = C::elem(r, n - 1);
#pragma unroll
    for (int e = 0; e < C::N; e += 2) x[e] = i + e == n - 1 ? last : x[e];
  }
}
template <class D>
__device__ __forceinline__ void ln_load(__amdgpu_buffer_rsrc_t r, int i, int n, float (&x)[RowChunk<D>::N]) {
  ln_unpack<D>(ln_raw<D>(r, i), r, i, n, x);
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

// M sums over the G threads of a row; `red` holds two turns of M floats per wave
// of the work-group, so that one barrier per call is enough.
template <int G, int M>
__device__ __forceinline__ void ln_sum(float (&v)[M], float* red, int& turn) {
#pragma unroll
  for (int k = 0; k < M; ++k) v[k] = wave_reduce(v[k], OpAdd());
  if constexpr (G > WAVE) {
    constexpr int GW = G / WAVE;
    const int nw = blockDim.x / WAVE, w = threadIdx.x / WAVE;
    float* t = red + turn * M * nw;
    if ((threadIdx.x & (WAVE - 1)) == 0)
#pragma unroll
      for (int k = 0; k < M; ++k) t[M * w + k] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < M; ++k) {
      v[k] = 0.0f;
#pragma unroll
      for (int i = 0; i < GW; ++i) v[k] += t[M * (w / GW * GW + i) + k];
    }
    turn ^= 1;
  }
}

}  // namespace

// Every work-group takes rows p, p + grid, ... of its G-thread groups (all
// groups of a work-group step together: those past the last row do the work
// of none).
template <class D, class W, int G, int U>
__global__ __launch_bounds__(G > LN_NT ? G : LN_NT) void k_norm(const fl_norm_args a) {
  constexpr int N = RowChunk<D>::N;
  constexpr int NT_ = G > LN_NT ? G : LN_NT, GR = NT_ / G;
  __shared__ float red[2 * NT_ / WAVE];
  const int n = static_cast<int>(a.dim), g = __builtin_amdgcn_readfirstlane(threadIdx.x / G), t = threadIdx.x % G;
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
  const int64_t step = static_cast<int64_t>(gridDim.x) * GR;
  int64_t r0 = static_cast<int64_t>(blockIdx.x) * GR;
  uint4 q[U];
  __amdgpu_buffer_rsrc_t rx;
  auto fetch = [&]() {   // row r0 + g, nothing past the last
    const bool on = r0 + g < a.rows;
    rx = ln_row<D>(a.x, on ? r0 + g : 0, a.ld, on ? n : 0);
#pragma unroll
    for (int u = 0; u < U; ++u) q[u] = ln_raw<D>(rx, N * (t + G * u));
  };
  fetch();
  int turn = 0;
  while (r0 < a.rows) {
    const int64_t r = r0 + g;
    const bool on = r < a.rows;
    float x[U][N], s[1] = {0.0f};
#pragma unroll
    for (int u = 0; u < U; ++u) {
      ln_unpack<D>(q[u], rx, N * (t + G * u), on ? n : 0, x[u]);
#pragma unroll
      for (int e = 0; e < N; ++e) s[0] += x[u][e];
    }
    r0 += step;
    if (r0 < a.rows) fetch();   // (the next row is on its way while this one is worked on)
    ln_sum<G>(s, red, turn);
    const float mean = s[0] * inv;
    float v[1] = {0.0f};
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int left = n - N * (t + G * u);
#pragma unroll
      for (int e = 0; e < N; ++e) x[u][e] -= mean;
      if (left >= N) {
#pragma unroll
        for (int e = 0; e < N; ++e) v[0] = fmaf(x[u][e], x[u][e], v[0]);
      } else {   // (the row's last values; one comparison a chunk where it has them all)
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (e < left) v[0] = fmaf(x[u][e], x[u][e], v[0]);
      }
    }
    ln_sum<G>(v, red, turn);
    const float rstd = 1.0f / sqrtf(fmaf(v[0], inv, a.eps));
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
template <class D, class W, int G, int U, bool WG, int NT_>
__global__ __launch_bounds__(NT_) void k_norm_grad(const fl_norm_grad_args a, float* part) {
  constexpr int N = RowChunk<D>::N;
  constexpr int GR = NT_ / G;
  __shared__ float red[4 * NT_ / WAVE];
  const int n = static_cast<int>(a.dim), g = __builtin_amdgcn_readfirstlane(threadIdx.x / G), t = threadIdx.x % G;
  const float inv = 1.0f / static_cast<float>(n);
  // The weights, and the next row, have a place in the registers, but not of 16
  // values by 1024 threads: they are read when they are needed.
  constexpr bool KEEP = NT_ * U * N <= 8192;
  float dw[U][N], db[U][N], wk[KEEP ? U : 1][N];
  const __amdgpu_buffer_rsrc_t rw = ln_row<W>(a.weight, 0, 0, a.weight ? n : 0);
  auto weights = [&](int u, float (&w)[N]) {
#pragma unroll
    for (int e = 0; e < N; ++e) w[e] = 1.0f;
    if (a.weight) ln_load_w<W>(rw, N * (t + G * u), n, w);
  };
#pragma unroll
  for (int u = 0; u < U; ++u) {
#pragma unroll
    for (int e = 0; e < N; ++e) dw[u][e] = db[u][e] = 0.0f;
    if constexpr (KEEP) weights(u, wk[u]);
  }
  const int64_t step = static_cast<int64_t>(gridDim.x) * GR;
  int64_t r0 = static_cast<int64_t>(blockIdx.x) * GR;
  uint4 qx[U], qd[U];
  __amdgpu_buffer_rsrc_t rx, rd;
  float mean, rstd;
  auto fetch = [&]() {   // row r0 + g, nothing past the last
    const bool on = r0 + g < a.rows;
    const int64_t r = on ? r0 + g : 0;
    rx = ln_row<D>(a.x, r, a.ld, on ? n : 0);
    rd = ln_row<D>(a.grad, r, a.grad_ld, on ? n : 0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      qx[u] = ln_raw<D>(rx, N * (t + G * u));
      qd[u] = ln_raw<D>(rd, N * (t + G * u));
    }
    mean = on ? a.mean[r] : 0.0f;
    rstd = on ? a.rstd[r] : 0.0f;
  };
  if (KEEP) fetch();
  int turn = 0;
  while (r0 < a.rows) {
    if (!KEEP) fetch();
    const int64_t r = r0 + g;
    const bool on = r < a.rows;
    const int m = on ? n : 0;
    const float rs = rstd;
    float x[U][N], d[U][N], s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = N * (t + G * u);
      ln_unpack<D>(qx[u], rx, i, m, x[u]);
      ln_unpack<D>(qd[u], rd, i, m, d[u]);
      if constexpr (!KEEP) weights(u, wk[0]);
      const float (&w)[N] = wk[KEEP ? u : 0];
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float xh = (x[u][e] - mean) * rs;   // (past the row dy is 0, and what it is multiplied with no matter)
        if (WG) {
          dw[u][e] = fmaf(d[u][e], xh, dw[u][e]);
          db[u][e] += d[u][e];
        }
        x[u][e] = xh;
        d[u][e] *= w[e];
        s[0] += d[u][e];
        s[1] = fmaf(d[u][e], xh, s[1]);
      }
    }
    r0 += step;
    if (KEEP && r0 < a.rows) fetch();   // (the next row is on its way while this one is worked on)
    if (a.out_dx == nullptr) continue;
    ln_sum<G>(s, red, turn);
    const float c1 = s[0] * inv, c2 = s[1] * inv;
    if (!on) continue;
    const __amdgpu_buffer_rsrc_t ro = ln_row<D>(a.out_dx, r, a.out_ld, n);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = N * (t + G * u);
      if (i >= n) continue;
      float o[N];
#pragma unroll
      for (int e = 0; e < N; ++e) o[e] = rs * (d[u][e] - c1 - x[u][e] * c2);
      ln_store<D>(ro, i, n, o);
    }
  }
  if constexpr (WG) {
    float* pw = part + static_cast<int64_t>(blockIdx.x) * 2 * n;
    if constexpr (GR == 1) {
      const __amdgpu_buffer_rsrc_t r1 = ln_row<F32>(pw, 0, 0, n), r2 = ln_row<F32>(pw, 1, n, n);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int c = 0; c < N; c += 4) {
          const int i = N * (t + G * u) + c;
          if (i >= n) continue;
          ln_store<F32>(r1, i, n, reinterpret_cast<const float(&)[4]>(dw[u][c]));
          ln_store<F32>(r2, i, n, reinterpret_cast<const float(&)[4]>(db[u][c]));
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

// f(G, U): the threads and chunks that hold a row of n values of N per chunk: a
// wave up to 1024, then 8 values a thread (the backward pass, which holds five
// arrays of them: 4096x2048 35.0 us with 32, 18.1 so) or 16 (WIDE: fewer waves
// that meet), and 16 past 8192.
template <int N, bool WIDE, class F>
void ln_shape(int64_t n, F&& f) {
  using std::integral_constant;
  constexpr int U8 = 8 / N;
  if (n <= 64 * N) f(integral_constant<int, 64>{}, integral_constant<int, 1>{});
  else if (n <= 64 * 16) f(integral_constant<int, 64>{}, integral_constant<int, 2 * U8>{});
  else if (n <= 256 * 8) f(integral_constant<int, 256>{}, integral_constant<int, U8>{});
  else if (WIDE && n <= 256 * 16) f(integral_constant<int, 256>{}, integral_constant<int, 2 * U8>{});
  else if (!WIDE && n <= 512 * 8) f(integral_constant<int, 512>{}, integral_constant<int, U8>{});
  else if (n <= 1024 * 8) f(integral_constant<int, 1024>{}, integral_constant<int, U8>{});
  else f(integral_constant<int, 1024>{}, integral_constant<int, 2 * U8>{});
}
static_assert(FL_NORM_MAX_DIM <= 1024 * 16, "the longest row fits");

template <class F>
void ln_types(int dtype, int wdtype, F&& f) {
  if (dtype == FL_DTYPE_F32) f(F32{}, F32{});
  else if (dtype == FL_DTYPE_BF16 && wdtype == FL_DTYPE_F32) f(BF16{}, F32{});
  else if (dtype == FL_DTYPE_BF16) f(BF16{}, BF16{});
  else if (wdtype == FL_DTYPE_F32) f(F16{}, F32{});
  else f(F16{}, F16{});
}

// Work-groups of the backward pass, each with partial sums to add at the end: one
// per CU at most.  Of 1024 threads where the registers allow it and 512 leave
// rows for a second turn (bf16 4096x4096: 22.6 us, 24.9 of 512).
constexpr int ln_threads(int G, int U, int N, bool many) { return G == 1024 || (many && U * N <= 8) ? 1024 : LN_BT; }
int ln_parts(int64_t rows, int threads, int G) {
  const int64_t gr = threads / G;
  return static_cast<int>(std::min<int64_t>((rows + gr - 1) / gr, LN_MAX_PARTS));
}
bool ln_many(int64_t rows, int G) { return rows > static_cast<int64_t>(LN_MAX_PARTS) * (LN_BT / std::min(G, LN_BT)); }

}  // namespace

size_t norm_grad_workspace_bytes(int64_t rows, int64_t dim, int dtype) {
  int parts = 0;
  const auto count = [&](auto g, auto u, int N) {
    constexpr int G = decltype(g)::value;
    parts = ln_parts(rows, ln_threads(G, decltype(u)::value, N, ln_many(rows, G)), G);
  };
  if (dtype == FL_DTYPE_F32) ln_shape<4, false>(dim, [&](auto g, auto u) { count(g, u, 4); });
  else ln_shape<8, false>(dim, [&](auto g, auto u) { count(g, u, 8); });
  return static_cast<size_t>(parts) * 2 * static_cast<size_t>(dim) * sizeof(float);
}

hipError_t launch_norm(const fl_norm_args& a, hipStream_t s) {
  ln_types(a.dtype, a.wdtype, [&](auto d, auto w) {
    using D = decltype(d);
    constexpr int N = RowChunk<D>::N;
    const auto run = [&](auto g, auto u) {
      constexpr int G = decltype(g)::value, NT_ = G > LN_NT ? G : LN_NT, GR = NT_ / G;
      // (2048 threads per CU; more rows loop, with the weights in registers)
      const unsigned grid = static_cast<unsigned>(std::min<int64_t>((a.rows + GR - 1) / GR, 256 * 2048 / NT_));
      hipLaunchKernelGGL((k_norm<D, decltype(w), G, decltype(u)::value>), dim3(grid), dim3(NT_), 0, s, a);
    };
    // (16 values a thread, 8: bf16 4096x4096 15.0, 16.9 us; 64x4096 3.8, 3.6 us.  Not
    // chosen by the number of rows: a row's result is a function of the row alone.)
    ln_shape<N, true>(a.dim, run);
  });
  return hipGetLastError();
}

hipError_t launch_norm_grad(const fl_norm_grad_args& a, hipStream_t s) {
  const bool wg = a.out_dweight != nullptr || a.out_dbias != nullptr;
  float* part = static_cast<float*>(a.workspace);
  ln_types(a.dtype, a.wdtype, [&](auto d, auto w) {
    using D = decltype(d);
    using W = decltype(w);
    constexpr int N = RowChunk<D>::N;
    int parts = 0;
    ln_shape<N, false>(a.dim, [&](auto g, auto u) {
      constexpr int G = decltype(g)::value, U = decltype(u)::value;
      const auto run = [&](auto nt) {
        constexpr int NT_ = decltype(nt)::value;
        parts = ln_parts(a.rows, NT_, G);
        if (parts == 0) return;
        if (wg) hipLaunchKernelGGL((k_norm_grad<D, W, G, U, true, NT_>), dim3(parts), dim3(NT_), 0, s, a, part);
        else hipLaunchKernelGGL((k_norm_grad<D, W, G, U, false, NT_>), dim3(parts), dim3(NT_), 0, s, a, part);
      };
      if (ln_many(a.rows, G)) run(std::integral_constant<int, ln_threads(G, U, N, true)>{});
      else run(std::integral_constant<int, ln_threads(G, U, N, false)>{});
    });
    if (wg)
      hipLaunchKernelGGL(k_norm_reduce<W>, dim3(static_cast<unsigned>((a.dim + WAVE - 1) / WAVE), 2), dim3(LN_RW * WAVE), 0, s,
                         a, part, parts);
  });
  return hipGetLastError();
}

}  // namespace fl

// New keys and values into a paged cache, and back.
//
// A work-group takes 16 neighbouring slots of one page, aligned, and one head: 16
// threads a token, 8 values each.  Keys go as they lie; values go through LDS to
// where a channel's 16 tokens lie side by side (32 bytes, 16 in 8 bits), stored
// whole where the call has all 16 and value by value where not (a decode step's
// one).  In 8 bits: the row's largest finite magnitude over its 16 threads, and
// from its bits the least power of two that takes it to 448; the product with it
// is exact, so that the e4m3 rounding is the only one.
#include <algorithm>

#include "fl_paged.h"
#include "fl_kernels.h"

namespace fl {

namespace {

constexpr int KV_NT = 256;
constexpr int KV_MAX_C = FL_CACHE_MAX_DIM / 8 / 16;   // chunks of a thread

// The scale's exponent for a row whose largest finite magnitude is m.
__device__ __forceinline__ int kv_exponent(float m) {
  if (m == 0.0f) return 0;
  int e;
  const float f = frexpf(m, &e);   // m = f 2^e, f in [0.5, 1); 448 = 0.875 2^9
  return min(max(e - 9 + (f > 0.875f ? 1 : 0), -96), 120);
}

__device__ __forceinline__ float kv_finite(float x) { return fabsf(x) <= 0x1.fffffep127f ? fabsf(x) : 0.0f; }

// e4m3 of 8 values (a NaN's code for those that are not finite: the format has no
// infinity)
__device__ __forceinline__ uint2 kv_e4m3(const float (&x)[8]) {
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = fabsf(x[i]) <= 448.0f ? x[i] : __builtin_nanf("");
  uint2 o;
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  o.x = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false);
  o.y = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], w, true);
  return o;
}

// 8 values of a row as floats (VEC: the row's chunks are 16-byte aligned)
template <class D, bool VEC>
__device__ __forceinline__ void kv_load(const void* row, int i, float (&x)[8]) {
  if constexpr (D::id == FL_DTYPE_F32) {
    const float* p = static_cast<const float*>(row) + i;
    if constexpr (VEC) {
      const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
      x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = p[e];
    }
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(row) + i;
    if constexpr (VEC) RowChunk<D>::unpack(*reinterpret_cast<const uint4*>(p), x);
    else
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = D::to_f32(p[e]);
  }
}
template <class D, bool VEC>
__device__ __forceinline__ void kv_store(void* row, int i, const float (&x)[8]) {
  if constexpr (D::id == FL_DTYPE_F32) {
    float* p = static_cast<float*>(row) + i;
    if constexpr (VEC) {
      *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
      *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) p[e] = x[e];
    }
  } else {
    uint16_t* p = static_cast<uint16_t*>(row) + i;
    uint32_t h[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = D::from_f32(x[e]);
    if constexpr (VEC)
      *reinterpret_cast<uint4*>(p) = make_uint4(h[0] | (h[1] << 16), h[2] | (h[3] << 16), h[4] | (h[5] << 16), h[6] | (h[7] << 16));
    else
#pragma unroll
      for (int e = 0; e < 8; ++e) p[e] = static_cast<uint16_t>(h[e]);
  }
}

}  // namespace

// E: the cache's dtype, D: the rows'.
template <class D, bool E8, bool VEC>
__global__ __launch_bounds__(KV_NT) void k_cache_write(const fl_cache_args a, int each) {
  const int Hk = static_cast<int>(a.cache.heads), h = blockIdx.x % Hk;
  __shared__ __attribute__((aligned(16))) uint16_t tv[FL_CACHE_MAX_DIM * KV_T];
  KvTile T;
  if (!kv_tile(a.rows, a.cache, paged_seq(a.rows, blockIdx.x / Hk, 1, KV_T, 2, each), T) || T.page < 0) return;
  const int t = threadIdx.x / 16, c0 = threadIdx.x % 16, dim = static_cast<int>(a.cache.dim);
  const int64_t ph = static_cast<int64_t>(T.page) * a.cache.heads + h, S = a.cache.page_size;
  const bool on = t >= T.t0 && t < T.t1;
  float k[KV_MAX_C][8], v[KV_MAX_C][8], mk = 0.0f, mv = 0.0f;
#pragma unroll
  for (int c = 0; c < KV_MAX_C; ++c) {
    const int i = 8 * (c0 + 16 * c);
    if (!on || i >= dim) {
#pragma unroll
      for (int e = 0; e < 8; ++e) k[c][e] = v[c][e] = 0.0f;
      continue;
    }
    constexpr int ESZ = D::id == FL_DTYPE_F32 ? 4 : 2;
    kv_load<D, VEC>(static_cast<const char*>(a.k) + ((T.row0 + t) * a.k_ld + h * a.k_hs) * ESZ, i, k[c]);
    kv_load<D, VEC>(static_cast<const char*>(a.v) + ((T.row0 + t) * a.v_ld + h * a.v_hs) * ESZ, i, v[c]);
    if constexpr (E8)
#pragma unroll
      for (int e = 0; e < 8; ++e) mk = fmaxf(mk, kv_finite(k[c][e])), mv = fmaxf(mv, kv_finite(v[c][e]));
  }
  int ek = 0, ev = 0;
  if constexpr (E8) {
#pragma unroll
    for (int m = 1; m < 16; m <<= 1) mk = fmaxf(mk, shfl_xor(mk, m)), mv = fmaxf(mv, shfl_xor(mv, m));
    ek = kv_exponent(mk), ev = kv_exponent(mv);
    if (on && c0 == 0) {
      a.cache.k_scale[ph * S + T.slot + t] = static_cast<uint8_t>(ek + 127);
      a.cache.v_scale[ph * S + T.slot + t] = static_cast<uint8_t>(ev + 127);
    }
  }
  uint8_t* tb = reinterpret_cast<uint8_t*>(tv);
#pragma unroll
  for (int c = 0; c < KV_MAX_C; ++c) {
    const int i = 8 * (c0 + 16 * c);
    if (!on || i >= dim) continue;
    const int64_t at = (ph * S + T.slot + t) * dim + i;
    if constexpr (E8) {
      // (a power of two, and its own in two steps below 2^-126: exact)
#pragma unroll
      for (int e = 0; e < 8; ++e) k[c][e] = ldexpf(k[c][e], -ek), v[c][e] = ldexpf(v[c][e], -ev);
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.cache.k) + at) = kv_e4m3(k[c]);
      const uint2 q = kv_e4m3(v[c]);
#pragma unroll
      for (int e = 0; e < 8; ++e) tb[(i + e) * KV_T + t] = static_cast<uint8_t>((e < 4 ? q.x : q.y) >> (8 * (e & 3)));
    } else {
      kv_store<D, true>(static_cast<uint16_t*>(a.cache.k) + at, 0, k[c]);
#pragma unroll
      for (int e = 0; e < 8; ++e) tv[(i + e) * KV_T + t] = static_cast<uint16_t>(D::from_f32(v[c][e]));
    }
  }
  __syncthreads();
  const int n = T.t1 - T.t0;
  const int64_t base = ph * dim * S + T.slot;
  if (n == KV_T) {
    constexpr int Q = E8 ? 1 : 2;   // 16-byte pieces of a channel's 16 tokens
    for (int i = threadIdx.x; i < Q * dim; i += KV_NT) {
      const int64_t at = base + static_cast<int64_t>(i / Q) * S;
      const uint4 q = reinterpret_cast<const uint4*>(tv)[i];
      if constexpr (E8) *reinterpret_cast<uint4*>(static_cast<uint8_t*>(a.cache.v) + at) = q;
      else reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.cache.v) + at)[i % Q] = q;
    }
  } else {
    for (int i = threadIdx.x; i < n * dim; i += KV_NT) {
      const int d = i / n, u = T.t0 + i % n;
      const int64_t at = base + static_cast<int64_t>(d) * S + u;
      if constexpr (E8) static_cast<uint8_t*>(a.cache.v)[at] = tb[d * KV_T + u];
      else static_cast<uint16_t*>(a.cache.v)[at] = tv[d * KV_T + u];
    }
  }
}

// O: the dtype of the rows written; C: a 16-bit cache's own (E8: none).
template <class O, class C, bool E8, bool VEC>
__global__ __launch_bounds__(KV_NT) void k_cache_read(const fl_cache_args a, int each) {
  const int Hk = static_cast<int>(a.cache.heads), h = blockIdx.x % Hk;
  __shared__ __attribute__((aligned(16))) uint16_t tv[FL_CACHE_MAX_DIM * KV_T];
  constexpr int ESZ = O::id == FL_DTYPE_F32 ? 4 : 2;
  const int t = threadIdx.x / 16, c0 = threadIdx.x % 16, dim = static_cast<int>(a.cache.dim);
  auto put = [&](int64_t row, int i, const float(&k)[8], const float(&v)[8]) {
    kv_store<O, VEC>(static_cast<char*>(a.k) + (row * a.k_ld + h * a.k_hs) * ESZ, i, k);
    kv_store<O, VEC>(static_cast<char*>(a.v) + (row * a.v_ld + h * a.v_hs) * ESZ, i, v);
  };
  const PagedSeq s = paged_seq(a.rows, blockIdx.x / Hk, 1, KV_T, 2, each);
  if (s.tile == 0 && s.pos < 0) {   // the tokens that do not exist
    const float zero[8] = {};
    const int64_t none = min(static_cast<int64_t>(s.n), -s.pos);
    for (int64_t u = t; u < none; u += KV_T)
      for (int i = 8 * c0; i < dim; i += 128) put(s.row + u, i, zero, zero);
  }
  KvTile T;
  if (!kv_tile(a.rows, a.cache, s, T)) return;
  const int64_t ph = static_cast<int64_t>(max(T.page, 0)) * a.cache.heads + h, S = a.cache.page_size;
  const bool on = t >= T.t0 && t < T.t1;
  if (T.page >= 0) {
    constexpr int Q = E8 ? 1 : 2;
    const int64_t base = ph * dim * S + T.slot;
    for (int i = threadIdx.x; i < Q * dim; i += KV_NT) {
      const int64_t at = base + static_cast<int64_t>(i / Q) * S;
      if constexpr (E8) reinterpret_cast<uint4*>(tv)[i] = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.cache.v) + at);
      else reinterpret_cast<uint4*>(tv)[i] = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.cache.v) + at)[i % Q];
    }
  }
  __syncthreads();
  if (!on) return;
  const uint8_t* tb = reinterpret_cast<const uint8_t*>(tv);
  int ek = 0, ev = 0;
  if constexpr (E8) {
    ek = a.cache.k_scale[ph * S + T.slot + t] - 127;
    ev = a.cache.v_scale[ph * S + T.slot + t] - 127;
  }
  for (int i = 8 * c0; i < dim; i += 128) {
    float k[8], v[8];
    if (T.page < 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) k[e] = v[e] = __builtin_nanf("");
    } else if constexpr (E8) {
      const uint2 q = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.cache.k) + (ph * S + T.slot + t) * dim + i);
      typedef float f32x2 __attribute__((ext_vector_type(2)));
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const int u = static_cast<int>(w == 0 ? q.x : q.y);
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(u, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(u, true);
        k[4 * w] = ldexpf(lo[0], ek), k[4 * w + 1] = ldexpf(lo[1], ek);
        k[4 * w + 2] = ldexpf(hi[0], ek), k[4 * w + 3] = ldexpf(hi[1], ek);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = ldexpf(__builtin_amdgcn_cvt_f32_fp8(tb[(i + e) * KV_T + t], 0), ev);
    } else {
      kv_load<C, true>(static_cast<const uint16_t*>(a.cache.k) + (ph * S + T.slot + t) * dim, i, k);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = C::to_f32(tv[(i + e) * KV_T + t]);
    }
    put(T.row0 + t, i, k, v);
  }
}

namespace {

template <class F>
void kv_types(int dtype, F&& f) {
  if (dtype == FL_DTYPE_F32) f(F32{});
  else if (dtype == FL_DTYPE_BF16) f(BF16{});
  else f(F16{});
}

bool kv_vector(const fl_cache_args& a) {
  const uintptr_t esz = a.dtype == FL_DTYPE_F32 ? 4 : 2;
  const uintptr_t strides = static_cast<uintptr_t>(a.k_ld) | static_cast<uintptr_t>(a.k_hs) | static_cast<uintptr_t>(a.v_ld) |
                            static_cast<uintptr_t>(a.v_hs);
  return ((reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) | strides * esz) & 15u) == 0;
}

}  // namespace

int64_t cache_blocks(const fl_cache_args& a) {
  int each = 0;
  return a.rows.seqs == 0 || a.rows.tokens == 0 ? 0 : kv_tiles(a.rows, &each) * a.cache.heads;
}

hipError_t launch_cache_write(const fl_cache_args& a, hipStream_t s) {
  int each = 0;
  const dim3 grid(static_cast<unsigned>(kv_tiles(a.rows, &each) * a.cache.heads));
  const bool vec = kv_vector(a);
  kv_types(a.dtype, [&](auto d) {
    using D = decltype(d);
    const auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(KV_NT), 0, s, a, each); };
    if (a.cache.dtype == FL_DTYPE_E4M3) vec ? run(k_cache_write<D, true, true>) : run(k_cache_write<D, true, false>);
    else if constexpr (D::id != FL_DTYPE_F32) vec ? run(k_cache_write<D, false, true>) : run(k_cache_write<D, false, false>);
  });
  return hipGetLastError();
}

hipError_t launch_cache_read(const fl_cache_args& a, hipStream_t s) {
  int each = 0;
  const dim3 grid(static_cast<unsigned>(kv_tiles(a.rows, &each) * a.cache.heads));
  const bool vec = kv_vector(a);
  kv_types(a.dtype, [&](auto d) {
    using O = decltype(d);
    const auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(KV_NT), 0, s, a, each); };
    if (a.cache.dtype == FL_DTYPE_E4M3) vec ? run(k_cache_read<O, BF16, true, true>) : run(k_cache_read<O, BF16, true, false>);
    else if (a.cache.dtype == FL_DTYPE_BF16) vec ? run(k_cache_read<O, BF16, false, true>) : run(k_cache_read<O, BF16, false, false>);
    else vec ? run(k_cache_read<O, F16, false, true>) : run(k_cache_read<O, F16, false, false>);
  });
  return hipGetLastError();
}

}  // namespace fl

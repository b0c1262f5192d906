// New keys and values into a paged cache, and back.
//
// A work-group takes 16 neighbouring slots of one page, aligned, and one head: 16
// threads a token, 8 values each.  Keys go as they lie; values go through LDS to
// where a channel's 16 tokens lie side by side (32 bytes, 16 in 8 bits), stored
// whole where the call has all 16 and value by value where not (a decode step's
// one).  In 8 bits: the row's largest finite magnitude over its 16 threads, and
// from its bits the least power of two that takes it to 448; the product with it
// is exact, so that the e4m3 rounding is the only one.
//
// The waves' instructions bound it, then HBM: 7240 tokens of 8 heads of 128, bf16 to 8
// bits, 44.5 MB each way: write 13.6 to 14.2 us, read 13.4 to 13.9 (3.3 TB/s; with values through LDS by
// the byte and float compares 17.9 and 16.2; 4 heads a work-group were 22).  A decode
// step's 64 tokens: 4.4 and 3.6 us, one launch's latency.
#include <algorithm>

#include "fl_paged.h"
#include "fl_kernels.h"

namespace fl {

namespace {

constexpr int KV_NT = 256;
constexpr int KV_MAX_C = FL_CACHE_MAX_DIM / 8 / 16;   // chunks of a thread

// The scale's exponent for a row whose largest finite magnitude has the bits m: the
// least e with m <= 448 2^e, 448 = 1.75 2^8.
__device__ __forceinline__ int kv_exponent(uint32_t m) {
  const int e = static_cast<int>((m + 0x1FFFFFu) >> 23) - 135;   // (a fraction above .75 carries)
  return m == 0 ? 0 : min(max(e, -96), 120);
}

// The largest over a row's 16 lanes.
template <int CTRL>
__device__ __forceinline__ uint32_t kv_dpp_max(uint32_t v) {
  return max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xF, 0xF, true)));
}
__device__ __forceinline__ uint32_t kv_row_max(uint32_t v) {
  // lanes 1 and 2 apart, then the half row's and the row's mirror images
  return kv_dpp_max<0x140>(kv_dpp_max<0x141>(kv_dpp_max<0x4E>(kv_dpp_max<0xB1>(v))));
}
constexpr uint32_t KV_INF = 0x7F800000u;

// e4m3 of 8 values of at most 448 (or NaN)
__device__ __forceinline__ uint2 kv_e4m3(const float (&x)[8]) {
  uint2 o;
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
  o.x = __builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], w, true);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(x[4], x[5], 0, false);
  o.y = __builtin_amdgcn_cvt_pk_fp8_f32(x[6], x[7], w, true);
  return o;
}

// Two values in 16 bits.
template <class D>
__device__ __forceinline__ uint32_t kv_pack(float lo, float hi) {
  if constexpr (D::id == FL_DTYPE_BF16) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){lo, hi}, bf16x2));
  } else return D::from_f32(lo) | (D::from_f32(hi) << 16);
}

// 8 values of a 16-bit row as they are (VEC: the row's chunks are 16-byte aligned)
template <bool VEC>
__device__ __forceinline__ uint4 kv_raw(const void* row, int i) {
  const uint16_t* p = static_cast<const uint16_t*>(row) + i;
  if constexpr (VEC) return *reinterpret_cast<const uint4*>(p);
  else return make_uint4(p[0] | (p[1] << 16), p[2] | (p[3] << 16), p[4] | (p[5] << 16), p[6] | (p[7] << 16));
}
template <bool VEC>
__device__ __forceinline__ void kv_store_raw(void* row, int i, uint4 q) {
  uint16_t* p = static_cast<uint16_t*>(row) + i;
  if constexpr (VEC) *reinterpret_cast<uint4*>(p) = q;
  else {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = static_cast<uint16_t>(e & 1 ? w[e / 2] >> 16 : w[e / 2]);
  }
}

// ... and of any row as floats
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
  } else RowChunk<D>::unpack(kv_raw<VEC>(row, i), x);
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
  } else
    kv_store_raw<VEC>(row, i, make_uint4(kv_pack<D>(x[0], x[1]), kv_pack<D>(x[2], x[3]), kv_pack<D>(x[4], x[5]), kv_pack<D>(x[6], x[7])));
}

// 8 e4m3 values times 2^e
__device__ __forceinline__ void kv_floats(uint2 q, int e, float (&x)[8]) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const int u = static_cast<int>(w == 0 ? q.x : q.y);
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(u, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(u, true);
    x[4 * w] = ldexpf(lo[0], e), x[4 * w + 1] = ldexpf(lo[1], e);
    x[4 * w + 2] = ldexpf(hi[0], e), x[4 * w + 3] = ldexpf(hi[1], e);
  }
}

// Values change between a lane's 8 channels of one token and 4 tokens of its 2
// channels within a wave (whose four rows of 16 lanes are 4 tokens), so that LDS is
// read and written by the dword: lanes 32 apart exchange dwords, then lanes 16 apart.
// Both ways are their own inverse.
__device__ __forceinline__ void kv_swap32(uint32_t& a, uint32_t& b) {   // a's upper lanes with b's lower ones
  const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = r[0], b = r[1];
}
__device__ __forceinline__ void kv_swap16(uint32_t& a, uint32_t& b) {   // a's odd rows of lanes with b's even ones
  const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
  a = r[0], b = r[1];
}
// bytes of a (0 to 3) and b (4 to 7), the selector's lowest first
template <uint32_t SEL>
__device__ __forceinline__ uint32_t kv_perm(uint32_t a, uint32_t b) {
  return __builtin_amdgcn_perm(b, a, SEL);
}

// Where the 16-byte piece p of a tile's values (a channel's 16 tokens in 8 bits, 8 of
// them in 16) lies in LDS: the lanes of an access, 8 channels apart, in different banks.
template <bool E8>
__device__ __forceinline__ int kv_piece(int p) {
  return p ^ ((p >> 4) & (E8 ? 7 : 3));
}

// The values of channels i to i + 7 of token t to LDS, and back (all lanes of a wave).
__device__ __forceinline__ void kv_put8(uint16_t* tv, int i, int t, bool on, uint2 q) {
  kv_swap32(q.x, q.y);
  uint32_t a = kv_perm<0x05010400>(q.x, q.y), b = kv_perm<0x07030602>(q.x, q.y);
  kv_swap16(a, b);
  const int ch = i + 2 * (t & 3);
  uint32_t* const to = reinterpret_cast<uint32_t*>(tv) + (t >> 2);
  if (on) to[4 * kv_piece<true>(ch)] = kv_perm<0x05010400>(a, b), to[4 * kv_piece<true>(ch + 1)] = kv_perm<0x07030602>(a, b);
}
__device__ __forceinline__ uint2 kv_get8(const uint16_t* tv, int i, int t, bool on) {
  const int ch = i + 2 * (t & 3);
  const uint32_t* const from = reinterpret_cast<const uint32_t*>(tv) + (t >> 2);
  uint32_t x = 0, y = 0;
  if (on) x = from[4 * kv_piece<true>(ch)], y = from[4 * kv_piece<true>(ch + 1)];
  uint32_t a = kv_perm<0x06040200>(x, y), b = kv_perm<0x07050301>(x, y);
  kv_swap16(a, b);
  uint2 q = make_uint2(kv_perm<0x06040200>(a, b), kv_perm<0x07050301>(a, b));
  kv_swap32(q.x, q.y);
  return q;
}
__device__ __forceinline__ void kv_put16(uint16_t* tv, int i, int t, bool on, uint32_t (&q)[4]) {
  kv_swap32(q[0], q[2]), kv_swap32(q[1], q[3]);
  kv_swap16(q[0], q[1]), kv_swap16(q[2], q[3]);
  const int ch = i + 2 * (t & 3), half = t >> 3;
  uint2* const to = reinterpret_cast<uint2*>(tv) + ((t >> 2) & 1);
  if (on) {
    to[2 * kv_piece<false>(2 * ch + half)] = make_uint2(kv_perm<0x05040100>(q[0], q[1]), kv_perm<0x05040100>(q[2], q[3]));
    to[2 * kv_piece<false>(2 * ch + 2 + half)] = make_uint2(kv_perm<0x07060302>(q[0], q[1]), kv_perm<0x07060302>(q[2], q[3]));
  }
}
__device__ __forceinline__ void kv_get16(const uint16_t* tv, int i, int t, bool on, uint32_t (&q)[4]) {
  const int ch = i + 2 * (t & 3), half = t >> 3;
  const uint2* const from = reinterpret_cast<const uint2*>(tv) + ((t >> 2) & 1);
  uint2 x = make_uint2(0, 0), y = x;
  if (on) x = from[2 * kv_piece<false>(2 * ch + half)], y = from[2 * kv_piece<false>(2 * ch + 2 + half)];
  q[0] = kv_perm<0x05040100>(x.x, y.x), q[1] = kv_perm<0x07060302>(x.x, y.x);
  q[2] = kv_perm<0x05040100>(x.y, y.y), q[3] = kv_perm<0x07060302>(x.y, y.y);
  kv_swap16(q[0], q[1]), kv_swap16(q[2], q[3]);
  kv_swap32(q[0], q[2]), kv_swap32(q[1], q[3]);
}

}  // namespace

// E: the cache's dtype, D: the rows'.
template <class D, bool E8, bool VEC>
__global__ __launch_bounds__(KV_NT) void k_cache_write(const fl_cache_args a, int each) {
  const int Hk = static_cast<int>(a.cache.heads), h = blockIdx.x % Hk;
  __shared__ __attribute__((aligned(16))) uint16_t tv[FL_CACHE_MAX_DIM * KV_T];
  KvTile T;
  if (!kv_tile(a.rows, a.cache, paged_seq(a.rows, blockIdx.x / Hk, 1, KV_T, 2, each), T)) return;
  const int t = threadIdx.x / 16, c0 = threadIdx.x % 16, dim = static_cast<int>(a.cache.dim);
  const int64_t ph = static_cast<int64_t>(T.page) * a.cache.heads + h, S = a.cache.page_size;
  const bool on = t >= T.t0 && t < T.t1;
  constexpr int ESZ = D::id == FL_DTYPE_F32 ? 4 : 2;
  const char* kp = static_cast<const char*>(a.k) + ((T.row0 + t) * a.k_ld + h * a.k_hs) * ESZ;
  const char* vp = static_cast<const char*>(a.v) + ((T.row0 + t) * a.v_ld + h * a.v_hs) * ESZ;
  const int64_t to = (ph * S + T.slot + t) * dim;
  if constexpr (E8) {
    float k[KV_MAX_C][8], v[KV_MAX_C][8];
    uint32_t mk = 0, mv = 0;
#pragma unroll
    for (int c = 0; c < KV_MAX_C; ++c) {
      if (128 * c >= dim) break;   // (the same for all: no instructions for channels that are not there)
      const int i = 8 * (c0 + 16 * c);
#pragma unroll
      for (int e = 0; e < 8; ++e) k[c][e] = v[c][e] = 0.0f;
      if (on && i < dim) kv_load<D, VEC>(kp, i, k[c]), kv_load<D, VEC>(vp, i, v[c]);
    }
    // (the page last: the rows are on their way before the table's entry is there)
    asm volatile("" ::: "memory");
    if (T.page < 0) return;
#pragma unroll
    for (int c = 0; c < KV_MAX_C; ++c) {
      if (128 * c >= dim) break;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        mk = max(mk, __float_as_uint(k[c][e]) & 0x7FFFFFFFu), mv = max(mv, __float_as_uint(v[c][e]) & 0x7FFFFFFFu);
    }
    if (__any(max(mk, mv) >= KV_INF)) {   // infinities are NaN, and neither counts
      mk = mv = 0;
      const auto finite = [](float& x, uint32_t& m) {
        const uint32_t u = __float_as_uint(x) & 0x7FFFFFFFu;
        if (u >= KV_INF) x = __builtin_nanf("");
        else m = max(m, u);
      };
#pragma unroll
      for (int c = 0; c < KV_MAX_C; ++c) {
        if (128 * c >= dim) break;
#pragma unroll
        for (int e = 0; e < 8; ++e) finite(k[c][e], mk), finite(v[c][e], mv);
      }
    }
    const int ek = kv_exponent(kv_row_max(mk)), ev = kv_exponent(kv_row_max(mv));
    if (on && c0 == 0) {
      a.cache.k_scale[ph * S + T.slot + t] = static_cast<uint8_t>(ek + 127);
      a.cache.v_scale[ph * S + T.slot + t] = static_cast<uint8_t>(ev + 127);
    }
#pragma unroll
    for (int c = 0; c < KV_MAX_C; ++c) {
      if (128 * c >= dim) break;
      const int i = 8 * (c0 + 16 * c);
#pragma unroll
      for (int e = 0; e < 8; ++e) k[c][e] = ldexpf(k[c][e], -ek), v[c][e] = ldexpf(v[c][e], -ev);
      if (on && i < dim) *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.cache.k) + to + i) = kv_e4m3(k[c]);
      kv_put8(tv, i, t, i < dim, kv_e4m3(v[c]));
    }
  } else {
    uint4 k[KV_MAX_C], v[KV_MAX_C];
#pragma unroll
    for (int c = 0; c < KV_MAX_C; ++c) {
      if (128 * c >= dim) break;
      const int i = 8 * (c0 + 16 * c);
      k[c] = v[c] = make_uint4(0, 0, 0, 0);
      if (on && i < dim) k[c] = kv_raw<VEC>(kp, i), v[c] = kv_raw<VEC>(vp, i);
    }
    asm volatile("" ::: "memory");
    if (T.page < 0) return;
#pragma unroll
    for (int c = 0; c < KV_MAX_C; ++c) {
      if (128 * c >= dim) break;
      const int i = 8 * (c0 + 16 * c);
      if (on && i < dim) kv_store_raw<true>(static_cast<uint16_t*>(a.cache.k) + to, i, k[c]);
      uint32_t q[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
      kv_put16(tv, i, t, i < dim, q);
    }
  }
  __syncthreads();
  const int n = T.t1 - T.t0;
  const int64_t base = ph * dim * S + T.slot;
  if (n == KV_T) {
    constexpr int Q = E8 ? 1 : 2;   // 16-byte pieces of a channel's 16 tokens
    for (int i = threadIdx.x; i < Q * dim; i += KV_NT) {
      const int64_t at = base + static_cast<int64_t>(i / Q) * S;
      const uint4 q = reinterpret_cast<const uint4*>(tv)[kv_piece<E8>(i)];
      if constexpr (E8) *reinterpret_cast<uint4*>(static_cast<uint8_t*>(a.cache.v) + at) = q;
      else reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.cache.v) + at)[i % Q] = q;
    }
  } else {
    for (int i = threadIdx.x; i < n * dim; i += KV_NT) {
      const int d = i / n, u = T.t0 + i % n;
      const int64_t at = base + static_cast<int64_t>(d) * S + u;
      if constexpr (E8) static_cast<uint8_t*>(a.cache.v)[at] = reinterpret_cast<const uint8_t*>(tv)[16 * kv_piece<true>(d) + u];
      else static_cast<uint16_t*>(a.cache.v)[at] = tv[8 * kv_piece<false>(2 * d + (u >> 3)) + (u & 7)];
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
  // the keys are on their way beside the values
  uint4 kq[KV_MAX_C];
  int ek = 0, ev = 0;
#pragma unroll
  for (int c = 0; c < KV_MAX_C; ++c) {
    if (128 * c >= dim) break;
    const int i = 8 * (c0 + 16 * c);
    kq[c] = make_uint4(0, 0, 0, 0);
    if (!on || i >= dim) continue;
    const int64_t at = (ph * S + T.slot + t) * dim + i;
    if constexpr (E8) {
      const uint2 q = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.cache.k) + at);
      kq[c].x = q.x, kq[c].y = q.y;
    } else kq[c] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.cache.k) + at);
  }
  if (E8 && on) {
    ek = a.cache.k_scale[ph * S + T.slot + t] - 127;
    ev = a.cache.v_scale[ph * S + T.slot + t] - 127;
  }
  if (T.page >= 0) {
    constexpr int Q = E8 ? 1 : 2;
    const int64_t base = ph * dim * S + T.slot;
    for (int i = threadIdx.x; i < Q * dim; i += KV_NT) {
      const int64_t at = base + static_cast<int64_t>(i / Q) * S;
      uint4& to = reinterpret_cast<uint4*>(tv)[kv_piece<E8>(i)];
      if constexpr (E8) to = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.cache.v) + at);
      else to = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.cache.v) + at)[i % Q];
    }
  }
  __syncthreads();
#pragma unroll
  for (int c = 0; c < KV_MAX_C; ++c) {
    if (128 * c >= dim) break;
    const int i = 8 * (c0 + 16 * c);
    float k[8], v[8];
    if constexpr (E8) {
      kv_floats(make_uint2(kq[c].x, kq[c].y), ek, k);
      kv_floats(kv_get8(tv, i, t, i < dim), ev, v);
    } else {
      RowChunk<C>::unpack(kq[c], k);
      uint32_t q[4];
      kv_get16(tv, i, t, i < dim, q);
      if (O::id == C::id && T.page >= 0) {
        if (on && i < dim) {
          kv_store_raw<VEC>(static_cast<char*>(a.k) + ((T.row0 + t) * a.k_ld + h * a.k_hs) * ESZ, i, kq[c]);
          kv_store_raw<VEC>(static_cast<char*>(a.v) + ((T.row0 + t) * a.v_ld + h * a.v_hs) * ESZ, i, make_uint4(q[0], q[1], q[2], q[3]));
        }
        continue;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = C::to_f32(e & 1 ? q[e / 2] >> 16 : q[e / 2] & 0xFFFFu);
    }
    if (T.page < 0)
#pragma unroll
      for (int e = 0; e < 8; ++e) k[e] = v[e] = __builtin_nanf("");
    if (on && i < dim) put(T.row0 + t, i, k, v);
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

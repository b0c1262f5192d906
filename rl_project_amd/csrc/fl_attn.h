// What the attention kernels share: types of the matrix instructions' operands, the
// keys that a tile of queries sees, how they are split, and the partial results.
#pragma once

#include <type_traits>

#include "fl_kernels.h"
#include "fl_paged.h"

namespace fl {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// 16 bytes by value (an assignment between uint4 lvalues is a memory copy to the
// compiler, which can leave an array of them in scratch memory).
__device__ __forceinline__ uint4 ld16(const void* p) {
  const u32x4 x = *static_cast<const u32x4*>(p);
  return make_uint4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ void st16(void* p, uint4 x) { *static_cast<u32x4*>(p) = (u32x4){x.x, x.y, x.z, x.w}; }

// 16-bit operands: 8 values of a lane as a uint4.
//
// With an 8-bit cache the weights of the second product carry their values' scales,
// 2^(s - m) 2^e.  bfloat16 has the range for any, half precision has not, and no maximum
// brings those that count near 1: a token whose values are all 0 may have any scale.
// So over 8 bits the second product is in bfloat16 (which holds e4m3 as well), of float16
// queries with the weights as two bfloat16, the second what the first leaves: 15 bits.
struct OpBF16 {
  using D = BF16;
  typedef __bf16 x8 __attribute__((ext_vector_type(8)));
  typedef __bf16 x2 __attribute__((ext_vector_type(2)));
  static constexpr uint32_t EXP = 0x7F80u, ONE = 0x0080u;   // the exponent's bits and its lowest
  __device__ static __forceinline__ f32x4 mfma16(uint4 a, uint4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  __device__ static __forceinline__ f32x16 mfma32(uint4 a, uint4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  __device__ static __forceinline__ uint32_t pack(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){lo, hi}, x2));
  }
  // 4 e4m3 values, times a power of two, as two dwords: exact (both types hold every
  // e4m3 value, bfloat16 also times any scale of a cache)
  static constexpr bool SCALES = true;
  __device__ static __forceinline__ uint2 widen(uint32_t q, float f = 1.0f) {
    return make_uint2(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q, f, false)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q, f, true)));
  }
};
struct OpF16 {
  using D = F16;
  typedef _Float16 x8 __attribute__((ext_vector_type(8)));
  typedef _Float16 x2 __attribute__((ext_vector_type(2)));
  static constexpr uint32_t EXP = 0x7C00u, ONE = 0x0400u;
  __device__ static __forceinline__ f32x4 mfma16(uint4 a, uint4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  __device__ static __forceinline__ f32x16 mfma32(uint4 a, uint4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  __device__ static __forceinline__ uint32_t pack(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){lo, hi}, x2));
  }
  static constexpr bool SCALES = false;   // (of scales below 2^-14 half precision loses bits, of some above 2^7 all)
  __device__ static __forceinline__ uint2 widen(uint32_t q, float f = 1.0f) {
    return make_uint2(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(q, f, false)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(q, f, true)));
  }
};

// The second product's type, and whether its weights are two for their type's sake.
template <class Op, bool E8>
using OpValues = std::conditional_t<E8, OpBF16, Op>;
template <class Op, bool E8>
constexpr bool TWO_WEIGHTS = E8 && !std::is_same_v<Op, OpBF16>;
// A weight as two bfloat16: its first 8 bits as they are, and the rest, rounded: 15 bits.
// The rest has 2^-22 of the weight added and so is above 0, like the first: times a value
// that is infinite both are, and not NaN.
__device__ __forceinline__ uint32_t weights_first(float lo, float hi) {
  return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302);
}
__device__ __forceinline__ uint32_t weights_rest(float lo, float hi) {
  const auto rest = [](float x) { return fmaf(x, 1.0f + 0x1p-22f, -__uint_as_float(__float_as_uint(x) & 0xFFFF0000u)); };
  return OpBF16::pack(rest(lo), rest(hi));
}

// The bits of 0x8000 where a 16-bit value of a dword is NaN or infinite.
template <class Op>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  return ((w & (Op::EXP * 0x10001u)) + Op::ONE * 0x10001u) & 0x80008000u;
}
template <class Op>
__device__ __forceinline__ uint32_t not_finite(uint4 q) {
  return not_finite<Op>(q.x) | not_finite<Op>(q.y) | not_finite<Op>(q.z) | not_finite<Op>(q.w);
}
// ... and the dword with 0 for those.
template <class Op>
__device__ __forceinline__ uint32_t finite_or_0(uint32_t w) {
  const uint32_t bad = not_finite<Op>(w);
  return w & ~((bad >> 15) * 0xFFFFu);
}
template <class Op>
__device__ __forceinline__ uint4 finite_or_0(uint4 q) {
  return make_uint4(finite_or_0<Op>(q.x), finite_or_0<Op>(q.y), finite_or_0<Op>(q.z), finite_or_0<Op>(q.w));
}

// 1 / l for a row's sum l, which is 0 where the row sees nothing (its position is below 0;
// the result is 0 then) or where every score that it sees is -infinity (0 / 0).
__device__ __forceinline__ float attn_inverse(float l, bool sees) {
  return l == 0.0f ? (sees ? __builtin_nanf("") : 0.0f) : 1.0f / l;
}

constexpr float AT_LAZY = 8.0f;     // how far, in powers of two, scores may pass the maximum in use

// A lane's 16 scores' soft-cap, in powers of two afterwards: cap tanh(z) log2(e), z = s scale / cap.
//
// Caps up to 64: 1 - 2 / (e^2z + 1), off by 10 2^-24 cap whatever the score, that is by
// 4e-5 in a score and in its weight, which is rounded to 2^-9 or 2^-11 of itself after.
// Above, that error would grow with the cap (a score of 0.3 is off by a thousandth at a
// cap of 1e4, and gone at 1e8), so there
//   |z| < 0.625: tanh z = z + z^3 p(z^2), the samplers' polynomial, on the score itself,
//     x + x z^2 p: as near to a score far below the cap as without one
//   above: 1 - 2 / (e^2|z| + 1), off by 5 2^-24 of 0.55 and more: 2^-20 of the score
// with the second left out where no lane of the wave needs it.  (4096 tokens of 8192,
// scores of 2: 552 us in the first form, 612 with the polynomial, 829 with both.)
constexpr float AT_SMALL_CAP = 64.0f;
struct AttnCap {
  float to_z, to2, cap2;   // of s q k: scale / cap, scale log2(e), cap log2(e)
  bool small;
};
__device__ __forceinline__ AttnCap attn_cap_of(float scale, float cap) {
  const float LOG2E = 1.4426950408889634f;
  return {cap > 0.0f ? scale / cap : 0.0f, scale * LOG2E, fminf(cap * LOG2E, 3.4028235e38f), cap <= AT_SMALL_CAP};
}
template <class X>
__device__ __forceinline__ void attn_cap(X& s, const AttnCap& c) {
  if (c.small) {
    const float to_e = c.to_z * 2.8853900817779268f;   // 2 log2(e)
#pragma unroll
    for (int e = 0; e < 16; ++e)
      s[e] = c.cap2 - 2.0f * c.cap2 * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(s[e] * to_e) + 1.0f);
    return;
  }
  float top = 0.0f;
#pragma unroll
  for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(s[e]));
  const auto near = [&](float x) {
    const float z = x * c.to_z, y = x * c.to2, t = z * z;
    float p = fmaf(t, TANH_P[5], TANH_P[4]);
#pragma unroll
    for (int i = 3; i >= 0; --i) p = fmaf(t, p, TANH_P[i]);
    return fmaf(y * t, p, y);
  };
  if (!__any(top * fabsf(c.to_z) >= 0.625f)) {
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] = near(s[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float z = s[e] * c.to_z, r = __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(fabsf(z) * 2.8853900817779268f) + 1.0f);
      s[e] = fabsf(z) < 0.625f ? near(s[e]) : copysignf(c.cap2 * fmaf(-2.0f, r, 1.0f), z);   // (a NaN stays NaN)
    }
  }
}

// The kernel for many rows: its tiles, and the rows of a sequence (tokens by heads of a
// group) up to which fl_attn.hip's is taken: 32 sequences of up to 4096, 40 and 64 rows, that
// one 148 and 155 us and this one 127 and 128 in 16 bits, but 100 and 106 against 114 in
// 8, which the other widens for four waves at once; with 80 rows 138 against 120.
constexpr int ATTN_WIDE_QT = 1, ATTN_WIDE_ROWS = 128 * ATTN_WIDE_QT;
constexpr int ATTN_FEW_ROWS = 32, ATTN_FEW_ROWS8 = 64;
hipError_t launch_attn_wide(const fl_attn_args& a, const AttnPlan& p, hipStream_t s);

}  // namespace fl

// Attention of a sequence's newest tokens over its pages, for few rows of queries
// (a row: one token's one head of a cached head's group): decode and verify steps.
//
//   s_t = scale q . k_t,  m = max s,  l = sum 2^(s_t - m),  out = sum 2^(s_t - m) v_t / l
//
// (scores in powers of two: scale log2(e) is one factor.)  One pass over the keys;
// HBM bounds it: each cached value is read once for all rows of the group.  A wave
// takes 16 (or 32) rows and 64 keys a step, four waves of a work-group different
// steps, work-groups different parts of a long sequence.
//
// Both products are transposed, so that everything stays in the wave's registers:
//   S^T = K Q^T   a lane gets 16 keys' scores of one row (its column, lane % 16)
//   O^T += V^T P^T   and so holds, of that row, the weights that the second product
//                 takes from it as they are
// with keys assigned to the first product's rows such that a lane's keys lie side by
// side: it then reads the values' 8 (16 in 8 bits) tokens of a channel in one load,
// as the cache has them.  No key, value or weight passes through LDS.  The maximum
// follows lazily: sums are rescaled when a score passes it by 2^8, not each time.
#include <algorithm>

#include "fl_attn.h"

namespace fl {

namespace {

constexpr int AR_NT = 256, AR_NW = AR_NT / WAVE;

// The cache's elements: how a lane (column c = lane % 16, quarter g = lane / 16)
// reads 64 keys.  Key of row m = 4 g' + i of score tile j: KEY(g', j) + i.
template <class Op_>
struct Cache16 {
  using Op = Op_;
  using Pv = Op_;
  static constexpr bool E8 = false;
  static constexpr int ESZ = 2;
  static constexpr int SUBS = 2;   // pages that a lane looks up for a step
  __device__ static __forceinline__ int key(int g, int j) { return (j >> 1) * 32 + g * 8 + (j & 1) * 4; }
  __device__ static __forceinline__ int chan(int g, int ks) { return ks * 32 + g * 8; }
};
template <class Op_>
struct Cache8 {
  using Op = Op_;
  // The second product's weights carry the values' scales, 2^-96 to 2^120: bfloat16
  // whatever the queries have (its 8 bits are twice what the values hold).
  using Pv = OpBF16;
  static constexpr bool E8 = true;
  static constexpr int ESZ = 1;
  static constexpr int SUBS = 1;
  __device__ static __forceinline__ int key(int g, int j) { return g * 16 + j * 4; }
  __device__ static __forceinline__ int chan(int g, int ks) { return (ks >> 1) * 64 + g * 16 + (ks & 1) * 8; }
};

__device__ __forceinline__ uint4 ar_load16(const char* p) { return *reinterpret_cast<const uint4*>(p); }
// (a row of 8-bit keys may start at any multiple of 8 bytes)
__device__ __forceinline__ uint4 ar_load16_8(const char* p) {
  const uint2 a = *reinterpret_cast<const uint2*>(p), b = *reinterpret_cast<const uint2*>(p + 8);
  return make_uint4(a.x, a.y, b.x, b.y);
}

}  // namespace

// C: the cache's elements, DT: channels (a multiple of 64, dim or more), FULL: dim ==
// DT, CT: tiles of 16 rows.
template <class C, int DT, bool FULL, int CT>
__global__ __launch_bounds__(AR_NT, 2) void k_attn_rows(const fl_attn_args a, const AttnPlan p) {
  using Op = typename C::Op;
  using Pv = typename C::Pv;
  constexpr int KS = DT / 32;   // steps of the first product
  constexpr int DM = DT / 16;   // tiles of channels of the second
  constexpr int TR = 16 * CT;
  // the waves' results side by side; before that, weights where values are not finite
  constexpr int OS = DT + 4;
  __shared__ __attribute__((aligned(16))) float so[AR_NW][16][OS];
  __shared__ float sm[AR_NW][TR], sl[AR_NW][TR];

  const int lane = threadIdx.x & (WAVE - 1), w = threadIdx.x / WAVE, c = lane & 15, g = lane >> 4;
  const int Hk = static_cast<int>(a.cache.heads), dim = static_cast<int>(a.cache.dim);
  const int h = blockIdx.x % Hk, rest = blockIdx.x / Hk, split = rest % p.splits;
  const PagedSeq s = paged_seq(a.rows, rest / p.splits, p.group, TR, 1, p.each);
  const int rows = s.n * p.group;
  if (rows < p.min_rows || rows > p.max_rows || s.tile >= (rows + TR - 1) / TR) return;
  const AttnSpan v = attn_span(a, p, s, s.tile);
  if (split >= v.splits) return;
  // (at most 2^25 steps by 64 parts)
  const int b0 = static_cast<uint32_t>(v.blocks) * split / static_cast<uint32_t>(v.splits);
  const int b1 = static_cast<uint32_t>(v.blocks) * (split + 1) / static_cast<uint32_t>(v.splits);

  // this lane's rows: their queries, and the keys they see: t <= at && (t >= from || t < sinks)
  uint4 q[CT][KS];
  int64_t at[CT], from[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int r = s.tile * TR + 16 * ct + c, i = r / p.group;
    const bool on = r < rows;
    at[ct] = on ? s.pos + i : -1;
    from[ct] = a.window > 0 ? at[ct] - a.window + 1 : 0;
    const char* row = static_cast<const char*>(a.q) +
                      2 * ((s.row + i) * a.q_ld + (h * p.group + (r - i * p.group)) * a.q_hs);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int d = C::chan(g, ks);
      q[ct][ks] = on && d < dim ? ar_load16(row + 2 * d) : make_uint4(0, 0, 0, 0);
    }
  }

  f32x4 o[CT][DM];
  float m[CT], l[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    m[ct] = -INFINITY;
    l[ct] = 0.0f;
#pragma unroll
    for (int i = 0; i < DM; ++i) o[ct][i] = (f32x4){0, 0, 0, 0};
  }
  const float LOG2E = 1.4426950408889634f;
  const float to2 = a.scale * LOG2E, cap2 = a.softcap * LOG2E, to_z = a.softcap > 0 ? 2.0f * LOG2E * a.scale / a.softcap : 0.0f;
  const int64_t S = a.cache.page_size;
  const char* K = static_cast<const char*>(a.cache.k);
  const char* V = static_cast<const char*>(a.cache.v);

  // the pages of a step that this lane reads keys (row c of a tile) and values from
  int pk[C::SUBS], pv[C::SUBS];
  auto pages = [&](int i) {
    const int64_t t0 = v.key(i);
#pragma unroll
    for (int u = 0; u < C::SUBS; ++u) {
      pk[u] = paged_page(a.rows, a.cache, s.b, t0 + C::key(c >> 2, 2 * u));
      pv[u] = paged_page(a.rows, a.cache, s.b, t0 + C::key(g, 2 * u));
    }
  };
  if (b0 + w < b1) pages(b0 + w);
  for (int i = b0 + w; i < b1; i += AR_NW) {
    const int64_t t0 = v.key(i);
    // ------------------------------------------------ S^T = K Q^T
    const char* kp[C::SUBS];
    int64_t vp[C::SUBS];
    bool bad[C::SUBS];
    uint4 ek, ev;
#pragma unroll
    for (int u = 0; u < C::SUBS; ++u) {
      const int64_t tk = t0 + C::key(c >> 2, 2 * u), tv = t0 + C::key(g, 2 * u);
      bad[u] = pv[u] < 0;
      const int64_t hk = static_cast<int64_t>(max(pk[u], 0)) * Hk + h, hv = static_cast<int64_t>(max(pv[u], 0)) * Hk + h;
      kp[u] = K + C::ESZ * ((hk * S + (tk & (S - 1)) + (c & 3)) * dim);
      vp[u] = C::ESZ * (hv * dim * S + (tv & (S - 1)));
      if constexpr (C::E8) {   // the scales of this lane's 16 keys
        ek = ar_load16(reinterpret_cast<const char*>(a.cache.k_scale) + hv * S + (tv & (S - 1)));
        ev = ar_load16(reinterpret_cast<const char*>(a.cache.v_scale) + hv * S + (tv & (S - 1)));
      }
    }
    bool some_bad = bad[0];
    if constexpr (C::SUBS == 2) some_bad |= bad[1];
    if (i + AR_NW < b1) pages(i + AR_NW);
    f32x4 st[CT][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const char* kr = kp[C::SUBS == 2 ? j >> 1 : 0] + C::ESZ * static_cast<int64_t>(dim) * (C::SUBS == 2 ? (j & 1) * 4 : j * 4);
      uint4 kf[KS];
      if constexpr (C::E8) {
#pragma unroll
        for (int ks = 0; ks < KS; ks += 2) {
          const int d = C::chan(g, ks);
          uint4 x = make_uint4(0, 0, 0, 0);
          if constexpr (FULL) x = ar_load16(kr + d);
          else if (d + 16 <= dim) x = ar_load16_8(kr + d);
          else if (d < dim) {
            const uint2 y = *reinterpret_cast<const uint2*>(kr + d);
            x.x = y.x, x.y = y.y;
          }
          const uint2 y0 = Op::widen(x.x), y1 = Op::widen(x.y), y2 = Op::widen(x.z), y3 = Op::widen(x.w);
          kf[ks] = make_uint4(y0.x, y0.y, y1.x, y1.y);
          kf[ks + 1] = make_uint4(y2.x, y2.y, y3.x, y3.y);
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const int d = C::chan(g, ks);
          kf[ks] = FULL || d < dim ? ar_load16(kr + 2 * d) : make_uint4(0, 0, 0, 0);
        }
      }
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        st[ct][j] = (f32x4){0, 0, 0, 0};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) st[ct][j] = Op::mfma16(kf[ks], q[ct][ks], st[ct][j]);
      }
    }
    // the values, on their way during the softmax (V^T: channel 16 dm + c, this lane's keys)
    uint4 vr[DM][C::SUBS];
#pragma unroll
    for (int dm = 0; dm < DM; ++dm)
#pragma unroll
      for (int u = 0; u < C::SUBS; ++u)
        vr[dm][u] = FULL || 16 * dm + c < dim ? ar_load16(V + vp[u] + C::ESZ * S * (16 * dm + c)) : make_uint4(0, 0, 0, 0);

    // ------------------------------------------------ the weights
    const bool masked = !attn_whole(a, v, t0) || __any(some_bad);
    uint4 pf[CT][2];
    float pw[CT][16];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      float x[16];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float y = st[ct][j][e];
          if constexpr (C::E8) y *= scale_of((j == 0 ? ek.x : j == 1 ? ek.y : j == 2 ? ek.z : ek.w) >> (8 * e) & 255u);
          x[4 * j + e] = y;
        }
      if (a.softcap > 0.0f) {
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = attn_cap(x[e], to_z, cap2);
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] *= to2;
      }
      if (masked) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int64_t t = t0 + C::key(g, j) + e;
            const bool seen = t <= at[ct] && (t >= from[ct] || t < a.sinks);
            const bool no_page = bad[C::SUBS == 2 ? j >> 1 : 0];
            x[4 * j + e] = !seen ? -INFINITY : no_page ? __builtin_nanf("") : x[4 * j + e];
          }
      }
      float top = x[0];
#pragma unroll
      for (int e = 1; e < 16; ++e) top = fmaxf(top, x[e]);
      if (__any(top > m[ct] + AT_LAZY)) {   // (m = -inf at first)
        top = fmaxf(top, shfl_xor(top, 16));
        top = fmaxf(top, shfl_xor(top, 32));
        const float to = fmaxf(m[ct], top);
        const float f = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[ct] - to);
        m[ct] = to;
        l[ct] *= f;
#pragma unroll
        for (int dm = 0; dm < DM; ++dm) o[ct][dm] *= f;
      }
      const float mm = m[ct] == -INFINITY ? 0.0f : m[ct];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        x[e] = __builtin_amdgcn_exp2f(x[e] - mm);
        l[ct] += x[e];
      }
      if constexpr (C::E8) {
        // the values' scales go to the weights
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float sv = scale_of((j == 0 ? ev.x : j == 1 ? ev.y : j == 2 ? ev.z : ev.w) >> (8 * e) & 255u);
            // (a masked slot may hold no scale)
            x[4 * j + e] = x[4 * j + e] == 0.0f ? 0.0f : x[4 * j + e] * sv;
          }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
        pf[ct][u] = make_uint4(Pv::pack(x[8 * u], x[8 * u + 1]), Pv::pack(x[8 * u + 2], x[8 * u + 3]),
                               Pv::pack(x[8 * u + 4], x[8 * u + 5]), Pv::pack(x[8 * u + 6], x[8 * u + 7]));
#pragma unroll
      for (int e = 0; e < 16; ++e) pw[ct][e] = x[e];
    }

    // ------------------------------------------------ O^T += V^T P^T
    // A value that is not finite would reach the rows that do not see its key (0 times
    // it is NaN): in a step with masks such values are taken out of the product, and
    // added to the rows that see them.
    bool odd = false;
    if (masked) {
      uint32_t any = 0;
#pragma unroll
      for (int dm = 0; dm < DM; ++dm)
#pragma unroll
        for (int u = 0; u < C::SUBS; ++u) {
          if constexpr (C::E8) {
            const uint4 y = vr[dm][u];
            any |= ((y.x & 0x7f7f7f7fu) + 0x01010101u) | ((y.y & 0x7f7f7f7fu) + 0x01010101u) |
                   ((y.z & 0x7f7f7f7fu) + 0x01010101u) | ((y.w & 0x7f7f7f7fu) + 0x01010101u);
            any &= 0x80808080u;
          } else any |= not_finite<Pv>(vr[dm][u]);
        }
      odd = __any(any != 0);
    }
#pragma unroll
    for (int dm = 0; dm < DM; ++dm) {
      uint4 vf[2];
      if constexpr (C::E8) {
        const uint4 x = vr[dm][0];
        const uint2 y0 = Pv::widen(x.x), y1 = Pv::widen(x.y), y2 = Pv::widen(x.z), y3 = Pv::widen(x.w);
        vf[0] = make_uint4(y0.x, y0.y, y1.x, y1.y);
        vf[1] = make_uint4(y2.x, y2.y, y3.x, y3.y);
      } else {
        vf[0] = vr[dm][0];
        vf[1] = vr[dm][C::SUBS - 1];
      }
      if (odd) vf[0] = finite_or_0<Pv>(vf[0]), vf[1] = finite_or_0<Pv>(vf[1]);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        o[ct][dm] = Pv::mfma16(vf[0], pf[ct][0], o[ct][dm]);
        o[ct][dm] = Pv::mfma16(vf[1], pf[ct][1], o[ct][dm]);
      }
    }
    if (odd) {
      float* wl = &so[w][0][0];   // [64 keys][16 rows]
      static_assert(64 * 16 <= 16 * OS, "a wave's weights fit");
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int k = C::key(g, j) + e;
            const int64_t t = t0 + k;
            const bool seen = t <= at[ct] && (t >= from[ct] || t < a.sinks);
            wl[k * 16 + c] = seen ? pw[ct][4 * j + e] : -1.0f;
          }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll 1
        for (int k = 0; k < AT_BLK; ++k) {
          const float x = wl[k * 16 + c];
          const int page = paged_page(a.rows, a.cache, s.b, t0 + k);
          if (!(x >= 0.0f) || page < 0) continue;   // (a NaN weight is in the sums already)
          const char* col = V + C::ESZ * ((static_cast<int64_t>(page) * Hk + h) * dim * S + ((t0 + k) & (S - 1)));
#pragma unroll
          for (int dm = 0; dm < DM; ++dm)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int d = 16 * dm + 4 * g + e;
              if (!FULL && d >= dim) continue;
              float y;
              if constexpr (C::E8) y = __builtin_amdgcn_cvt_f32_fp8(static_cast<uint8_t>(col[S * d]), 0);
              else y = Op::D::to_f32(*reinterpret_cast<const uint16_t*>(col + 2 * S * d));
              if (!(fabsf(y) < INFINITY)) o[ct][dm][e] += x * y;
            }
        }
        __builtin_amdgcn_wave_barrier();
      }
    }
  }

  // ------------------------------------------------ the waves together
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    l[ct] += shfl_xor(l[ct], 16);
    l[ct] += shfl_xor(l[ct], 32);
    if (g == 0) sm[w][16 * ct + c] = m[ct], sl[w][16 * ct + c] = l[ct];
  }
  __syncthreads();
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int col = 16 * ct + c;
    const float top = fmaxf(fmaxf(sm[0][col], sm[1][col]), fmaxf(sm[2][col], sm[3][col]));
    const float f = m[ct] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[ct] - top);
#pragma unroll
    for (int dm = 0; dm < DM; ++dm) *reinterpret_cast<f32x4*>(&so[w][c][16 * dm + 4 * g]) = o[ct][dm] * f;
    __syncthreads();
    // 16 threads a row, 4 channels each
    const int rr = threadIdx.x / 16, k = threadIdx.x % 16;
    const int r = s.tile * TR + 16 * ct + rr;
    if (r < rows) {
      float mm = -INFINITY, ll = 0.0f;
#pragma unroll
      for (int x = 0; x < AR_NW; ++x) mm = fmaxf(mm, sm[x][16 * ct + rr]);
#pragma unroll
      for (int x = 0; x < AR_NW; ++x) {
        const float y = sm[x][16 * ct + rr], z = sl[x][16 * ct + rr];
        ll += y == -INFINITY ? z : z * __builtin_amdgcn_exp2f(y - mm);   // (z is 0 then, or NaN)
      }
      const int i = r / p.group;
      if (s.pos + i >= a.rows.table_width * S) ll = __builtin_nanf("");
      const int64_t head = h * p.group + (r - i * p.group), row = (s.row + i) * a.q_heads + head;
      const float inv = v.splits > 1 ? 1.0f : ll == 0.0f ? 0.0f : 1.0f / ll;
#pragma unroll
      for (int d = 4 * k; d < DT; d += 64) {
        if (d >= dim) break;
        f32x4 y = *reinterpret_cast<const f32x4*>(&so[0][rr][d]);
#pragma unroll
        for (int x = 1; x < AR_NW; ++x) y += *reinterpret_cast<const f32x4*>(&so[x][rr][d]);
        if (v.splits > 1) *reinterpret_cast<f32x4*>(p.part + (row * p.splits + split) * dim + d) = y;
        else {
          y *= inv;
          *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + (s.row + i) * a.out_ld + head * a.out_hs + d) =
              make_uint2(Op::pack(y[0], y[1]), Op::pack(y[2], y[3]));
        }
      }
      if (k == 0) {
        if (v.splits > 1) *reinterpret_cast<float2*>(p.stat + 2 * (row * p.splits + split)) = make_float2(mm, ll);
        else if (a.out_lse) a.out_lse[row] = ll == 0.0f ? -INFINITY : (mm == -INFINITY ? ll : (mm + log2f(ll)) * 0.6931471805599453f);
      }
    }
    __syncthreads();
  }
}

// The parts of rows whose keys were split: a wave a row.
template <class Op>
__global__ __launch_bounds__(AR_NT) void k_attn_join(const fl_attn_args a, const AttnPlan p) {
  const int lane = threadIdx.x & (WAVE - 1), Hk = static_cast<int>(a.cache.heads), dim = static_cast<int>(a.cache.dim);
  // a work-group takes 4 rows of one tile and cached head
  const int per = (p.tr + 3) / 4;
  const int h = blockIdx.x % Hk, rest = blockIdx.x / Hk;
  const PagedSeq s = paged_seq(a.rows, rest / per, p.group, p.tr, 1, p.each);
  const int rows = s.n * p.group, k4 = 4 * (rest % per) + threadIdx.x / WAVE;
  if (rows < p.min_rows || rows > p.max_rows || k4 >= p.tr || s.tile >= (rows + p.tr - 1) / p.tr) return;
  const int r = s.tile * p.tr + k4;
  if (r >= rows) return;
  const AttnSpan v = attn_span(a, p, s, s.tile);
  if (v.splits <= 1) return;
  const int i = r / p.group;
  const int64_t head = h * p.group + (r - i * p.group), row = (s.row + i) * a.q_heads + head;
  static_assert(AT_MAX_SPLITS <= WAVE, "a lane for every part");
  float2 st = make_float2(-INFINITY, 0.0f);
  if (lane < v.splits) st = *reinterpret_cast<const float2*>(p.stat + 2 * (row * p.splits + lane));
  const float m = wave_reduce(st.x, OpMax());
  const float f = st.x == -INFINITY ? (st.y == 0.0f ? 0.0f : 1.0f) : __builtin_amdgcn_exp2f(st.x - m);
  const float l = wave_reduce(st.y * f, OpAdd());
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  if (lane == 0 && a.out_lse) a.out_lse[row] = l == 0.0f ? -INFINITY : (m == -INFINITY ? l : (m + log2f(l)) * 0.6931471805599453f);
  f32x4 y = {0, 0, 0, 0};
  const float* part = p.part + row * p.splits * dim + 4 * lane;
#pragma unroll 4
  for (int k = 0; k < v.splits; ++k) {
    const float x = __shfl(f, k, WAVE);
    if (4 * lane < dim && x != 0.0f) y += x * *reinterpret_cast<const f32x4*>(part + static_cast<int64_t>(k) * dim);
  }
  if (4 * lane < dim) {
    y *= inv;
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + (s.row + i) * a.out_ld + head * a.out_hs + 4 * lane) =
        make_uint2(Op::pack(y[0], y[1]), Op::pack(y[2], y[3]));
  }
}

namespace {

template <class C, int DT, bool FULL>
void ar_launch(const fl_attn_args& a, const AttnPlan& p, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(p.tiles * p.splits * a.cache.heads));
  if (p.tr == 16) hipLaunchKernelGGL((k_attn_rows<C, DT, FULL, 1>), grid, dim3(AR_NT), 0, s, a, p);
  else hipLaunchKernelGGL((k_attn_rows<C, DT, FULL, 2>), grid, dim3(AR_NT), 0, s, a, p);
}
template <class C>
void ar_dims(const fl_attn_args& a, const AttnPlan& p, hipStream_t s) {
  switch (a.cache.dim) {
    case 64: return ar_launch<C, 64, true>(a, p, s);
    case 128: return ar_launch<C, 128, true>(a, p, s);
    case 256: return ar_launch<C, 256, true>(a, p, s);
  }
  if (a.cache.dim < 64) ar_launch<C, 64, false>(a, p, s);
  else if (a.cache.dim < 128) ar_launch<C, 128, false>(a, p, s);
  else ar_launch<C, 256, false>(a, p, s);
}

int64_t attn_groups(const fl_attn_args& a) { return a.q_heads / a.cache.heads; }

// The plan of a launch with tiles of tr rows.
AttnPlan attn_plan(const fl_attn_args& a, int tr) {
  AttnPlan p = {};
  p.group = static_cast<int>(attn_groups(a));
  p.tr = tr;
  p.min_rows = 0;
  p.max_rows = 0x7fffffff;
  p.each = static_cast<int>((a.rows.tokens / a.rows.seqs * p.group + tr - 1) / tr);
  p.tiles = paged_tiles(a.rows, p.group, tr, 1, p.each);
  // Splits: enough for 4 work-groups on every CU, none shorter than 4 steps of 64
  // keys of the longest sequence the table (or the window) allows.
  int64_t keys = a.rows.table_width * a.cache.page_size;
  if (a.window > 0 && a.window <= keys) keys = std::min(keys, a.window + tr / p.group + std::min(a.sinks, keys) + 3 * AT_BLK);
  const int64_t blocks = (keys + AT_BLK - 1) / AT_BLK, groups = std::max<int64_t>(p.tiles * a.cache.heads, 1);
  const int64_t want = (1024 + groups - 1) / groups, most = (blocks + AT_MIN_BLKS - 1) / AT_MIN_BLKS;
  p.splits = static_cast<int>(std::max<int64_t>(1, std::min({want, most, static_cast<int64_t>(AT_MAX_SPLITS)})));
  return p;
}

int attn_tile_rows(const fl_attn_args& a) {
  return a.rows.tokens * attn_groups(a) <= 16 * a.rows.seqs ? 16 : 32;
}

size_t attn_part_bytes(const fl_attn_args& a, const AttnPlan& p) {
  return p.splits > 1 ? static_cast<size_t>(a.rows.tokens) * a.q_heads * p.splits * (a.cache.dim + 2) * sizeof(float) : 0;
}

}  // namespace

size_t attn_workspace_bytes(const fl_attn_args& a) {
  if (a.rows.tokens == 0 || a.rows.seqs == 0) return 0;
  return attn_part_bytes(a, attn_plan(a, attn_tile_rows(a)));
}

int64_t attn_blocks(const fl_attn_args& a) {
  if (a.rows.tokens == 0 || a.rows.seqs == 0) return 0;
  const AttnPlan p = attn_plan(a, attn_tile_rows(a));
  return p.tiles * a.cache.heads * std::max<int64_t>(p.splits, (p.tr + 3) / 4);
}

hipError_t launch_attn(const fl_attn_args& args, hipStream_t s) {
  fl_attn_args a = args;
  // (positions are below 2^31: a longer window is none)
  a.window = a.window > 0x7fffffff ? 0 : a.window;
  a.sinks = std::min<int64_t>(a.sinks, 0x7fffffff);
  AttnPlan p = attn_plan(a, attn_tile_rows(a));
  p.part = static_cast<float*>(a.workspace);
  p.stat = p.part ? p.part + a.rows.tokens * a.q_heads * p.splits * a.cache.dim : nullptr;
  const bool bf = a.dtype == FL_DTYPE_BF16;
  if (a.cache.dtype == FL_DTYPE_E4M3) bf ? ar_dims<Cache8<OpBF16>>(a, p, s) : ar_dims<Cache8<OpF16>>(a, p, s);
  else bf ? ar_dims<Cache16<OpBF16>>(a, p, s) : ar_dims<Cache16<OpF16>>(a, p, s);
  if (p.splits > 1) {
    const dim3 grid(static_cast<unsigned>(p.tiles * ((p.tr + 3) / 4) * a.cache.heads));
    if (bf) hipLaunchKernelGGL(k_attn_join<OpBF16>, grid, dim3(AR_NT), 0, s, a, p);
    else hipLaunchKernelGGL(k_attn_join<OpF16>, grid, dim3(AR_NT), 0, s, a, p);
  }
  return hipGetLastError();
}

}  // namespace fl

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
//
// 64 sequences of 1024 to 8192 tokens, 32 heads over 8, dim 128, bf16: 244 us, 5.0 TB/s of
// the cache (values after their step's keys: 531; all of a step under way at once, 267;
// joins by work-groups, 243).  4 of up to 131072 in 8 bits: 127 us, 5.1 TB/s.  Where little
// is read, two launches bound it: 16 windows of 1024, 24 us (18.5 + 4.8 for the join).
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
  static constexpr bool E8 = false;
  static constexpr int ESZ = 2;
  static constexpr int SUBS = 2;   // pages that a lane looks up for a step
  __device__ static __forceinline__ int key(int g, int j) { return (j >> 1) * 32 + g * 8 + (j & 1) * 4; }
  __device__ static __forceinline__ int chan(int g, int ks) { return ks * 32 + g * 8; }
};
template <class Op_>
struct Cache8 {
  using Op = Op_;
  static constexpr bool E8 = true;
  static constexpr int ESZ = 1;
  static constexpr int SUBS = 1;
  __device__ static __forceinline__ int key(int g, int j) { return g * 16 + j * 4; }
  __device__ static __forceinline__ int chan(int g, int ks) { return (ks >> 1) * 64 + g * 16 + (ks & 1) * 8; }
};

// A row of 8-bit keys may start at any multiple of 8 bytes.
__device__ __forceinline__ uint4 ar_load16_8(const char* p) {
  const uint2 a = *reinterpret_cast<const uint2*>(p), b = *reinterpret_cast<const uint2*>(p + 8);
  return make_uint4(a.x, a.y, b.x, b.y);
}

}  // namespace

// C: the cache's elements, DT: channels (a multiple of 64, dim or more), FULL: dim ==
// DT, CT: tiles of 16 rows.
template <class C, int DT, bool FULL, int CT>
__global__ __launch_bounds__(AR_NT, DT * CT > 256 ? 1 : 2) void k_attn_rows(const fl_attn_args a, const AttnPlan p) {
  using Op = typename C::Op;
  using VOp = OpValues<Op, C::E8>;
  // bfloat16's weights as two, too: the float32 product's result but for the last
  // rounding (distance from 64 bits 1.66e-3, 2.0e-3 to 2.3e-3 with one).  Memory hides the
  // second product (64 x 8192 242 us either way, 4 x 131072 in 8 bits 126); above 128
  // channels registers do not hold it (dim 256 508 against 535 us), nor do the matrix
  // cores of fl_attn_wide.hip hide it (435 against 591).
  constexpr bool TWO = TWO_WEIGHTS<Op, C::E8> || (std::is_same_v<VOp, OpBF16> && DT <= 128);
  constexpr int KS = DT / 32;   // steps of the first product
  constexpr int DM = DT / 16;   // tiles of channels of the second
  // a step's keys on their way beside all its values, by their bytes (of queries and
  // accumulators above 128 channels in 8 bits some 110 registers go to scratch); else the
  // tiles of values that are loaded ahead of their step's softmax
  constexpr bool ALL = DT * CT * C::ESZ <= 256;
  constexpr int VPRE = ALL || DM * C::SUBS * CT <= 16 ? DM : DM / 2;
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

  // this lane's rows: their queries, and the keys they see
  uint4 q[CT][KS];
  AttnSeen see[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int r = s.tile * TR + 16 * ct + c, i = r / p.group;
    const bool on = r < rows;
    see[ct] = attn_seen(a, on ? s.pos + i : -1);
    const char* row = static_cast<const char*>(a.q) +
                      2 * ((s.row + i) * a.q_ld + (h * p.group + (r - i * p.group)) * a.q_hs);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int d = C::chan(g, ks);
      q[ct][ks] = on && d < dim ? ld16(row + 2 * d) : make_uint4(0, 0, 0, 0);
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
  const AttnCap cap = attn_cap_of(a.scale, a.softcap);
  const int64_t S = a.cache.page_size;
  const char* K = static_cast<const char*>(a.cache.k);
  const char* V = static_cast<const char*>(a.cache.v);

  // the pages of a step that this lane reads keys (row c of a tile) and values from
  int pk[C::SUBS], pv[C::SUBS];
  auto pages = [&](int i) {
    const int t0 = v.key(i);
#pragma unroll
    for (int u = 0; u < C::SUBS; ++u) {
      pk[u] = paged_page(a.rows, a.cache, s.b, t0 + C::key(c >> 2, 2 * u));
      pv[u] = paged_page(a.rows, a.cache, s.b, t0 + C::key(g, 2 * u));
    }
  };
  if (b0 + w < b1) pages(b0 + w);
  for (int i = b0 + w; i < b1; i += AR_NW) {
    const int t0 = v.key(i);
    // ------------------------------------------------ S^T = K Q^T
    const char* kp[C::SUBS];
    int64_t vp[C::SUBS];
    bool bad[C::SUBS];
    uint4 ek, ev;
#pragma unroll
    for (int u = 0; u < C::SUBS; ++u) {
      const int tk = t0 + C::key(c >> 2, 2 * u), tv = t0 + C::key(g, 2 * u);
      bad[u] = pv[u] < 0;
      const int64_t hk = static_cast<int64_t>(max(pk[u], 0)) * Hk + h, hv = static_cast<int64_t>(max(pv[u], 0)) * Hk + h;
      kp[u] = K + C::ESZ * ((hk * S + (tk & (S - 1)) + (c & 3)) * dim);
      vp[u] = C::ESZ * (hv * dim * S + (tv & (S - 1)));
      if constexpr (C::E8) {   // the scales of this lane's 16 keys
        ek = ld16(reinterpret_cast<const char*>(a.cache.k_scale) + hv * S + (tv & (S - 1)));
        ev = ld16(reinterpret_cast<const char*>(a.cache.v_scale) + hv * S + (tv & (S - 1)));
      }
    }
    bool some_bad = bad[0];
    if constexpr (C::SUBS == 2) some_bad |= bad[1];
    if (i + AR_NW < b1) pages(i + AR_NW);
    f32x4 st[CT][4];
    constexpr int KR = C::E8 ? KS / 2 : KS;   // loads of a tile's key
    const auto keys = [&](int j, uint4(&x)[KR]) {
      const char* kr = kp[C::SUBS == 2 ? j >> 1 : 0] + C::ESZ * static_cast<int64_t>(dim) * (C::SUBS == 2 ? (j & 1) * 4 : j * 4);
#pragma unroll
      for (int n = 0; n < KR; ++n) {
        const int d = C::chan(g, C::E8 ? 2 * n : n);
        if constexpr (FULL) x[n] = ld16(kr + C::ESZ * d);
        else if constexpr (C::E8) {
          x[n] = make_uint4(0, 0, 0, 0);
          if (d + 16 <= dim) x[n] = ar_load16_8(kr + d);
          else if (d < dim) {
            const uint2 y = *reinterpret_cast<const uint2*>(kr + d);
            x[n] = make_uint4(y.x, y.y, 0, 0);
          }
        } else x[n] = d < dim ? ld16(kr + 2 * d) : make_uint4(0, 0, 0, 0);
      }
    };
    const auto scores = [&](int j, const uint4(&x)[KR]) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) st[ct][j] = (f32x4){0, 0, 0, 0};
#pragma unroll
      for (int n = 0; n < KR; ++n) {
        if constexpr (C::E8) {
          const uint2 y0 = Op::widen(x[n].x), y1 = Op::widen(x[n].y), y2 = Op::widen(x[n].z), y3 = Op::widen(x[n].w);
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) {
            st[ct][j] = Op::mfma16(make_uint4(y0.x, y0.y, y1.x, y1.y), q[ct][2 * n], st[ct][j]);
            st[ct][j] = Op::mfma16(make_uint4(y2.x, y2.y, y3.x, y3.y), q[ct][2 * n + 1], st[ct][j]);
          }
        } else
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) st[ct][j] = Op::mfma16(x[n], q[ct][n], st[ct][j]);
      }
    };
    // the values (V^T: channel 16 dm + c, this lane's keys)
    uint4 vr[DM][C::SUBS];
    const char* vs[C::SUBS];
#pragma unroll
    for (int u = 0; u < C::SUBS; ++u) vs[u] = V + vp[u] + C::ESZ * S * c;
    const auto values = [&](int dm) {
#pragma unroll
      for (int u = 0; u < C::SUBS; ++u) {
        vr[dm][u] = FULL || 16 * dm + c < dim ? ld16(vs[u]) : make_uint4(0, 0, 0, 0);
        vs[u] += C::ESZ * S * 16;
        asm("" : "+v"(vs[u]));   // (one address that moves, not one for every tile)
      }
    };
    if constexpr (ALL) {   // all of a step on its way at once
      uint4 x[4][KR];
#pragma unroll
      for (int j = 0; j < 4; ++j) keys(j, x[j]);
#pragma unroll
      for (int dm = 0; dm < DM; ++dm) values(dm);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < 4; ++j) scores(j, x[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint4 x[KR];
        keys(j, x);
        scores(j, x);
        // (a tile's keys, no more, where their registers are many)
        if (DT * CT > 256) __builtin_amdgcn_sched_barrier(0);
      }
      // (the values' registers are the keys')
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int dm = 0; dm < VPRE; ++dm) values(dm);
    }

    // ------------------------------------------------ the weights
    const bool masked = !v.whole(t0) || __any(some_bad);
    uint4 pf[CT][2], pr[TWO ? CT : 1][2];
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
      if (a.softcap > 0.0f) attn_cap(x, cap);
      else {
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] *= cap.to2;
      }
      if (masked) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int t = t0 + C::key(g, j) + e;
            const bool seen = (t <= see[ct].last) & ((t >= see[ct].from) | (t < v.sinks));
            const float y = bad[C::SUBS == 2 ? j >> 1 : 0] ? __builtin_nanf("") : x[4 * j + e];
            x[4 * j + e] = seen ? y : -INFINITY;
          }
      }
      float top = -INFINITY;
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, x[e]);
      if (__any(top > m[ct] + AT_LAZY)) {   // (m = -inf at first)
        top = fmaxf(top, shfl_xor(top, 16));
        top = fmaxf(top, shfl_xor(top, 32));
        const float to = top > m[ct] + AT_LAZY ? top : m[ct];   // (each row by its own scores)
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
          for (int e = 0; e < 4; ++e)
            x[4 * j + e] *= scale_of((j == 0 ? ev.x : j == 1 ? ev.y : j == 2 ? ev.z : ev.w) >> (8 * e) & 255u);
      }
      const auto packed = [&](auto f, int u) {
        return make_uint4(f(x[8 * u], x[8 * u + 1]), f(x[8 * u + 2], x[8 * u + 3]), f(x[8 * u + 4], x[8 * u + 5]), f(x[8 * u + 6], x[8 * u + 7]));
      };
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if constexpr (TWO) {
          pf[ct][u] = packed(weights_first, u);
          pr[ct][u] = packed(weights_rest, u);
        } else pf[ct][u] = packed(VOp::pack, u);
      }
    }

    // ------------------------------------------------ O^T += V^T P^T
    // A value that is not finite would reach the rows that do not see its key (0 times
    // it is NaN): in a step with masks such values are taken out of the product, and
    // added to the rows that see them.
    uint32_t odd = 0;
#pragma unroll
    for (int dm = 0; dm < DM; ++dm) {
      if (dm + VPRE < DM) values(dm + VPRE);
      uint4 vf[2];
      if constexpr (C::E8) {
        const uint4 x = vr[dm][0];
        const uint2 y0 = VOp::widen(x.x), y1 = VOp::widen(x.y), y2 = VOp::widen(x.z), y3 = VOp::widen(x.w);
        vf[0] = make_uint4(y0.x, y0.y, y1.x, y1.y);
        vf[1] = make_uint4(y2.x, y2.y, y3.x, y3.y);
      } else {
        vf[0] = vr[dm][0];
        vf[1] = vr[dm][C::SUBS - 1];
      }
      if (masked) {
        odd |= not_finite<VOp>(vf[0]) | not_finite<VOp>(vf[1]);
        vf[0] = finite_or_0<VOp>(vf[0]), vf[1] = finite_or_0<VOp>(vf[1]);
      }
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        o[ct][dm] = VOp::mfma16(vf[0], pf[ct][0], o[ct][dm]);
        o[ct][dm] = VOp::mfma16(vf[1], pf[ct][1], o[ct][dm]);
        if constexpr (TWO) {
          o[ct][dm] = VOp::mfma16(vf[0], pr[ct][0], o[ct][dm]);
          o[ct][dm] = VOp::mfma16(vf[1], pr[ct][1], o[ct][dm]);
        }
      }
    }
    if (masked && __any(odd != 0)) {
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
            const int t = t0 + k;
            const bool seen = (t <= see[ct].last) & ((t >= see[ct].from) | (t < v.sinks));
            const uint4 y = pf[ct][j >> 1];
            const uint32_t x = j & 1 ? (e < 2 ? y.z : y.w) : (e < 2 ? y.x : y.y);
            wl[k * 16 + c] = seen ? VOp::D::to_f32((e & 1 ? x >> 16 : x) & 0xFFFFu) : -1.0f;
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
          const char* src = col + C::ESZ * (4 * g * S);
#pragma unroll
          for (int dm = 0; dm < DM; ++dm)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              // (one load at a time: this path is rare, the registers are the kernel's)
              asm volatile("" : "+v"(src) : : "memory");
              if (FULL || 16 * dm + 4 * g + e < dim) {
                float y;
                if constexpr (C::E8) y = __builtin_amdgcn_cvt_f32_fp8(static_cast<uint8_t>(*src), 0);
                else y = Op::D::to_f32(*reinterpret_cast<const uint16_t*>(src));
                if (!(fabsf(y) < INFINITY)) o[ct][dm][e] += x * y;
              }
              src += C::ESZ * S * (e == 3 ? 13 : 1);
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
      const int64_t place = attn_place(p, s.b, Hk, h, r, row) * p.splits + split;
      const float inv = v.splits > 1 ? 1.0f : attn_inverse(ll, s.pos + i >= 0);
#pragma unroll
      for (int d = 4 * k; d < DT; d += 64) {
        if (d >= dim) break;
        f32x4 y = *reinterpret_cast<const f32x4*>(&so[0][rr][d]);
#pragma unroll
        for (int x = 1; x < AR_NW; ++x) y += *reinterpret_cast<const f32x4*>(&so[x][rr][d]);
        if (v.splits > 1) *reinterpret_cast<f32x4*>(p.part + place * dim + d) = y;
        else {
          y *= inv;
          *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + (s.row + i) * a.out_ld + head * a.out_hs + d) =
              make_uint2(Op::pack(y[0], y[1]), Op::pack(y[2], y[3]));
        }
      }
      if (k == 0) {
        if (v.splits > 1) *reinterpret_cast<float2*>(p.stat + 2 * place) = make_float2(mm, ll);
        else if (a.out_lse) a.out_lse[row] = ll == 0.0f ? -INFINITY : (mm == -INFINITY ? ll : (mm + log2f(ll)) * 0.6931471805599453f);
      }
    }
    __syncthreads();
  }
}

// The parts of rows whose keys were split.  A work-group looks at `rb` places (a thread
// each), and joins those that have parts: `tpr` threads a part (4 channels each), its
// groups different parts.  few and many: the plans of sequences of few rows and of many;
// the first `by_row` places are the call's rows, the others few's slots.
constexpr int AJ_ROWS = 64;
template <class Op>
__global__ __launch_bounds__(AR_NT) void k_attn_join(const fl_attn_args a, const AttnPlan few, const AttnPlan many, int64_t by_row,
                                                     int tpr, int rb) {
  __shared__ f32x4 sy[AR_NT];
  __shared__ int parts[AJ_ROWS], rows[AJ_ROWS];   // (parts: negative those of `few`; rows: ~ of tokens that do not exist)
  const int lane = threadIdx.x & (WAVE - 1), dim = static_cast<int>(a.cache.dim), heads = static_cast<int>(a.q_heads);
  const int seqs = static_cast<int>(a.rows.seqs);
  const int64_t place0 = static_cast<int64_t>(blockIdx.x) * rb;
  if (threadIdx.x < rb) {
    const int64_t x = place0 + threadIdx.x;
    int splits = 0;
    int64_t row = x;
    if (x < by_row) {
      const int n = static_cast<int>(row / heads), head = static_cast<int>(row - static_cast<int64_t>(n) * heads);
      const PagedSeq s = paged_rows(a.rows, a.rows.starts == nullptr ? n / (static_cast<int>(a.rows.tokens) / seqs)
                                                                     : paged_find(seqs, n, [&](int m) { return a.rows.starts[m]; }));
      const int i = n - static_cast<int>(s.row);
      if (i >= 0 && i < s.n) {   // (else a row behind the last sequence)
        const bool is_few = s.n * few.group <= few.max_rows;
        const AttnPlan& p = is_few ? few : many;
        if (p.slots == 0) splits = attn_span(a, p, s, (i * p.group + head % p.group) / p.tr).splits;
        if (is_few) splits = -splits;
        if (s.pos + i < 0) row = ~row;
      }
    } else if (few.slots > 0) {
      const int64_t bh = (x - by_row) / few.slots;
      const int r = static_cast<int>((x - by_row) % few.slots), h = static_cast<int>(bh % a.cache.heads);
      if (bh < seqs * a.cache.heads) {
        const PagedSeq s = paged_rows(a.rows, static_cast<int>(bh / a.cache.heads));
        if (r < s.n * few.group && s.n * few.group <= few.max_rows) splits = -attn_span(a, few, s, r / few.tr).splits;
        row = (s.row + r / few.group) * heads + h * few.group + r % few.group;
        if (s.pos + r / few.group < 0) row = ~row;
      }
    }
    parts[threadIdx.x] = splits, rows[threadIdx.x] = static_cast<int>(row);
  }
  __syncthreads();
  static_assert(AT_MAX_SPLITS <= WAVE, "a lane for every part");
  const int g = threadIdx.x / tpr, d = 4 * (threadIdx.x & (tpr - 1)), groups = AR_NT / tpr;
#pragma unroll 1
  for (int j = 0; j < rb; ++j) {
    const int splits = abs(parts[j]);
    if (splits <= 1) continue;
    const AttnPlan& p = parts[j] < 0 ? few : many;
    const bool sees = rows[j] >= 0;
    const int64_t row = sees ? rows[j] : ~rows[j], n = row / heads, head = row - n * heads;
    const int64_t place = (place0 + j < by_row ? row : place0 + j - by_row) * p.splits;
    // (every wave for itself)
    float2 st = make_float2(-INFINITY, 0.0f);
    if (lane < splits) st = *reinterpret_cast<const float2*>(p.stat + 2 * (place + lane));
    const float m = wave_reduce(st.x, OpMax());
    const float f = st.x == -INFINITY ? (st.y == 0.0f ? 0.0f : 1.0f) : __builtin_amdgcn_exp2f(st.x - m);
    const float l = wave_reduce(st.y * f, OpAdd());
    if (threadIdx.x == 0 && a.out_lse)
      a.out_lse[row] = l == 0.0f ? -INFINITY : (m == -INFINITY ? l : (m + log2f(l)) * 0.6931471805599453f);
    f32x4 y = {0, 0, 0, 0};
    const float* part = p.part + place * dim + d;
    for (int k0 = 0; k0 < splits; k0 += groups) {   // (the same turns for all lanes: they exchange)
      const int k = k0 + g;
      const float x = __shfl(f, k, WAVE);
      if (k < splits && d < dim && x != 0.0f) y += x * *reinterpret_cast<const f32x4*>(part + static_cast<int64_t>(k) * dim);
    }
    sy[threadIdx.x] = y;
    __syncthreads();
    if (g == 0 && d < dim) {
      for (int k = 1; k < groups; ++k) y += sy[k * tpr + threadIdx.x];
      y *= attn_inverse(l, sees);
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + n * a.out_ld + head * a.out_hs + d) =
          make_uint2(Op::pack(y[0], y[1]), Op::pack(y[2], y[3]));
    }
    __syncthreads();
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

// The launches of a call: sequences of few rows and of many.  Their parts lie apart:
// `by_row` places for every row of the call, if one of them keeps its parts so, and few's
// slots where these are fewer (a prompt's call has a million rows, and its few short
// sequences some thousand).
struct AttnCall {
  AttnPlan few, many;
  bool has_few, has_many;
  int64_t few_places, many_places, by_row, places;   // (places: that the join looks at)
  int64_t parts() const { return few_places * few.splits + many_places * many.splits; }
};

AttnCall attn_call(const fl_attn_args& a) {
  AttnCall c = {};
  const int few_rows = a.cache.dtype == FL_DTYPE_E4M3 ? ATTN_FEW_ROWS8 : ATTN_FEW_ROWS;
  const int64_t G = a.q_heads / a.cache.heads, N = a.rows.tokens, B = a.rows.seqs, Hk = a.cache.heads;
  // The most rows that a sequence can have, and all have where there are no starts.
  const int64_t top = (a.rows.starts ? N : N / B) * G;
  c.has_few = a.rows.starts || top <= few_rows;
  c.has_many = top > few_rows;
  const int64_t keys = a.rows.table_width * a.cache.page_size;
  // Splits: enough that every CU has `work` / 256 work-groups, and `least` of them, so
  // that long and short sequences share the CUs evenly (64 sequences of 1024 to 8192
  // tokens: 2 splits 269 us, 4 243 us, 8 262 us); none shorter than 8 steps of 64 keys
  // of the longest sequence the table (or the window) allows.
  const auto plan = [&](AttnPlan& p, int tr, int64_t groups, int64_t work, int64_t least) {
    p.group = static_cast<int>(G);
    p.tr = tr;
    p.tiles = paged_tiles(a.rows, G, tr, 1, p.each);
    const int64_t seen = a.window > 0 && a.window <= keys
                             ? std::min(keys, a.window + tr / G + std::min(a.sinks, keys) + 3 * AT_BLK) : keys;
    const int64_t blocks = (seen + AT_BLK - 1) / AT_BLK, want = std::max(least, (work + groups - 1) / groups);
    p.splits = static_cast<int>(std::max<int64_t>(
        1, std::min({want, (blocks + AT_MIN_BLKS - 1) / AT_MIN_BLKS, static_cast<int64_t>(AT_MAX_SPLITS)})));
  };
  if (c.has_few) {
    const int64_t rows = std::min<int64_t>(top, few_rows);
    // (ragged: tiles of 16 where the average sequence fits one)
    const int tr = (a.rows.starts ? N * G <= 16 * B : top <= 16) ? 16 : 32;
    c.few.min_rows = 0, c.few.max_rows = few_rows;
    c.few.each = static_cast<int>((rows + tr - 1) / tr);
    plan(c.few, tr, B * Hk, 1024, 4);
    if (c.few.splits > 1) {
      if (N * G > B * rows) c.few.slots = static_cast<int>(rows);
      c.few_places = c.few.slots > 0 ? B * Hk * rows : N * Hk * G;
    }
  }
  if (c.has_many) {
    c.many.min_rows = c.has_few ? few_rows + 1 : 0, c.many.max_rows = 0x7fffffff;
    c.many.each = a.rows.starts ? 0 : static_cast<int>((top + ATTN_WIDE_ROWS - 1) / ATTN_WIDE_ROWS);
    // (ragged: as if all tokens were of sequences of many rows, so that the parts of all
    // rows are at most 2^17, however many of them single tokens' turn out to be)
    const int64_t tiles = a.rows.starts ? (N * G + ATTN_WIDE_ROWS - 1) / ATTN_WIDE_ROWS : B * c.many.each;
    plan(c.many, ATTN_WIDE_ROWS, tiles * Hk, 512, 1);
    if (c.many.splits > 1) c.many_places = N * Hk * G;
  }
  if (!c.has_few) c.few.group = 1, c.few.max_rows = 0;
  c.by_row = std::max(c.many_places, c.few.slots > 0 ? 0 : c.few_places);
  c.places = c.by_row + (c.few.slots > 0 ? c.few_places : 0);
  return c;
}

int64_t attn_rows(const fl_attn_args& a) { return a.rows.seqs == 0 ? 0 : a.rows.tokens * a.q_heads; }

}  // namespace

size_t attn_workspace_bytes(const fl_attn_args& a) {
  if (attn_rows(a) == 0) return 0;
  return static_cast<size_t>(attn_call(a).parts()) * (a.cache.dim + 2) * sizeof(float);
}

int64_t attn_blocks(const fl_attn_args& a) {
  if (attn_rows(a) == 0) return 0;
  const AttnCall c = attn_call(a);
  return std::max({c.few.tiles * c.few.splits * a.cache.heads, c.many.tiles * c.many.splits * a.cache.heads,
                   c.places > 0 ? std::max<int64_t>(c.places / AJ_ROWS, std::min<int64_t>(c.places, 16384)) + 1 : 0});
}

hipError_t launch_attn(const fl_attn_args& args, hipStream_t s) {
  fl_attn_args a = args;
  // (positions are below 2^31: a longer window is none)
  a.window = a.window > 0x7fffffff ? 0 : a.window;
  a.sinks = std::min<int64_t>(a.sinks, 0x7fffffff);
  AttnCall c = attn_call(a);
  // (all parts, then all their maxima and sums: the parts stay 16-byte aligned)
  c.few.part = static_cast<float*>(a.workspace);
  c.many.part = c.few.part + c.few_places * c.few.splits * a.cache.dim;
  c.few.stat = c.few.part + c.parts() * a.cache.dim;
  c.many.stat = c.few.stat + c.few_places * c.few.splits * 2;
  const bool bf = a.dtype == FL_DTYPE_BF16;
  if (c.has_many)
    if (const hipError_t e = launch_attn_wide(a, c.many, s)) return e;
  if (c.has_few) {
    if (a.cache.dtype == FL_DTYPE_E4M3) bf ? ar_dims<Cache8<OpBF16>>(a, c.few, s) : ar_dims<Cache8<OpF16>>(a, c.few, s);
    else bf ? ar_dims<Cache16<OpBF16>>(a, c.few, s) : ar_dims<Cache16<OpF16>>(a, c.few, s);
  }
  if (c.places > 0) {
    // (a row a work-group where that fills the card: most rows of a prompt have no parts)
    const int64_t n = c.places, rb = std::max<int64_t>(1, std::min<int64_t>(n / 8192, AJ_ROWS));
    const dim3 grid(static_cast<unsigned>((n + rb - 1) / rb));
    const int tpr = a.cache.dim <= 64 ? 16 : a.cache.dim <= 128 ? 32 : 64;
    if (bf) hipLaunchKernelGGL(k_attn_join<OpBF16>, grid, dim3(AR_NT), 0, s, a, c.few, c.many, c.by_row, tpr, static_cast<int>(rb));
    else hipLaunchKernelGGL(k_attn_join<OpF16>, grid, dim3(AR_NT), 0, s, a, c.few, c.many, c.by_row, tpr, static_cast<int>(rb));
  }
  return hipGetLastError();
}

}  // namespace fl

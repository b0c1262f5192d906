// Attention over a paged cache for many rows of queries (prompts and their pieces);
// the few rows of decode and verify steps are fl_attn.hip's.
//
// 4 D flops a score for the matrix cores, and beside them the softmax's vector
// instructions, which bound it with them: in one wave they alternate, and registers
// leave two waves a SIMD.  A work-group takes 128 rows, a wave 32 (64: no faster); 64
// keys a step, theirs and their values' tiles in LDS for all four waves, in two turns.
// 16-bit tiles of dim 64, 128 and 256 are loaded past the registers while the other
// turn's are worked on, without padding (aw_swap); 8-bit ones and other dims go through
// registers, 8 bits widened on the way, with rows 16 bytes longer than their data.
// Products as there, transposed: S^T = K Q^T and O^T += V^T P^T with 32x32x16
// instructions, keys assigned to the first product's rows such that a lane's weights are
// the second's operand as they are, and so are the values' tokens as the cache has
// them.  A row's sums and maximum are its column's two lanes'.
//
// 4096 new tokens of 8192, 32 heads over 8, dim 128, bf16: 438 to 448 us, 0.92 to 0.94
// PFLOP/s (a library product reaches 1.59), 5 vector instructions a matrix instruction.
// 12 pieces of up to 1024 tokens over up to 8192, 8 bits: 812 us, 0.69 PFLOP/s, 10 a matrix
// instruction.  (Passes as they are; a profiler's trace has 505 and 876.)
// Before: a step's loads one after another 2857 us (the first), tiles in LDS 889, two
// turns 498, loads past registers 478, instructions in order (aw_reads_ahead) 438.
#include <algorithm>

#include "fl_attn.h"

namespace fl {

namespace {

constexpr int AW_NT = 256, AW_NW = AW_NT / WAVE;

// Bytes of LDS of a work-group: two turns of 64 keys, their values, and 8-bit scales.
constexpr int aw_lds(int DT, bool E8, bool FULL) {
  const int pad = FULL && !E8 ? 0 : 16;
  return 2 * (AT_BLK * (2 * DT + pad) + DT * (2 * AT_BLK + pad) + (E8 ? 2 * AT_BLK * 4 : 0));
}

// Tiles without padding have their rows' chunks exchanged instead (by an exclusive or),
// so that 16 neighbouring rows' chunks of one number lie in different banks (64, of 4
// bytes): rows of 256 bytes and more by the row, of 128 by the pair of rows.
template <int ROW>
__device__ __forceinline__ int aw_swap(int row) {
  return ROW >= 256 ? row & 15 : (row >> 1) & 7;
}

// 16 bytes per lane from base (the wave's) + off to LDS at lds + 16 lane, past the
// registers; the waits are the kernel's (vmcnt).
__device__ __forceinline__ void aw_load_lds(const char* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(off), "s"(base)
               : "memory", "m0");
}
__device__ __forceinline__ void aw_load_lds(const char* src, uint32_t lds) {   // ... each lane from its own address
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(src)
               : "memory", "m0");
}

}  // namespace

// The order of n matrix instructions with an LDS read each: the reads AW_AHEAD before
// (left to itself, the compiler reads, waits and multiplies in turn).
constexpr int AW_AHEAD = 6;
template <int N>
__device__ __forceinline__ void aw_reads_ahead() {
  __builtin_amdgcn_sched_group_barrier(0x100, AW_AHEAD, 0);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
  }
}

// Op: the queries' type, E8: 8-bit cache, DT: channels (a multiple of 64, dim or more),
// FULL: dim == DT, QT: tiles of 32 rows of a wave.
template <class Op, bool E8, int DT, bool FULL, int QT>
__global__ __launch_bounds__(AW_NT, QT == 1 && DT <= 128 ? 2 : 1) void k_attn_wide(const fl_attn_args a, const AttnPlan p) {
  using VOp = OpValues<Op, E8>;
  constexpr bool TWO = TWO_WEIGHTS<Op, E8>;
  constexpr int TR = 32 * QT * AW_NW;
  constexpr int ESZ = E8 ? 1 : 2, EPC = 16 / ESZ;         // the cache's elements, and those of a 16-byte chunk
  // 16-bit tiles go to LDS as they lie, without registers; 8-bit ones and padded rows
  // through registers
  constexpr bool DIRECT = FULL && !E8;
  constexpr int KC = DT / EPC, VC = AT_BLK / EPC;         // chunks of a key's and of a channel's row
  constexpr int NK = AT_BLK * KC / AW_NT, NV = DT * VC / AW_NT;   // chunks of a thread
  constexpr int PAD = DIRECT ? 0 : 16;
  constexpr int KS = 2 * DT + PAD, VS = 2 * AT_BLK + PAD;   // LDS row strides in bytes
  constexpr int KB = AT_BLK * KS, VB = DT * VS, SB = E8 ? 2 * AT_BLK * 4 : 0;
  constexpr int BUF = KB + VB + SB;
  static_assert(aw_lds(DT, E8, FULL) == 2 * BUF, "the launch's LDS");
  constexpr int KSTEPS = DT / 16, DM = DT / 32;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ int flags[2];   // of the steps' turns: 1 << sub-block: no page, 16: a value that is not finite

  const int tid = threadIdx.x, lane = tid & (WAVE - 1), w = tid / WAVE, c = lane & 31, hh = lane >> 5;
  const int Hk = static_cast<int>(a.cache.heads), dim = static_cast<int>(a.cache.dim);
  const int h = blockIdx.x % Hk, rest = blockIdx.x / Hk, split = rest % p.splits;
  // (the last tiles, which see the most keys, first)
  const PagedSeq s = paged_seq(a.rows, static_cast<int>(p.tiles) - 1 - rest / p.splits, p.group, TR, 1, p.each);
  const int rows = s.n * p.group;
  if (rows < p.min_rows || rows > p.max_rows || s.tile >= (rows + TR - 1) / TR) return;
  const AttnSpan v = attn_span(a, p, s, s.tile);
  if (split >= v.splits) return;
  const int b0 = static_cast<uint32_t>(v.blocks) * split / static_cast<uint32_t>(v.splits);
  const int b1 = static_cast<uint32_t>(v.blocks) * (split + 1) / static_cast<uint32_t>(v.splits);

  // a negative scale turns the queries' signs
  // (and one of 0 clears them: a masked score is -inf, which no factor may be 0 to)
  const uint32_t sign = a.scale < 0.0f ? 0x80008000u : 0u, keep = a.scale == 0.0f ? 0u : ~0u;
  const float scale = fabsf(a.scale);
  const float to2 = a.softcap > 0.0f || a.scale == 0.0f ? 1.0f : scale * 1.4426950408889634f;
  const AttnCap cap = attn_cap_of(scale, a.softcap);

  uint4 q[QT][KSTEPS];
  AttnSeen see[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int r = s.tile * TR + 32 * (QT * w + t) + c, i = r / p.group;
    const bool on = r < rows;
    see[t] = attn_seen(a, on ? s.pos + i : -1);
    const char* row = static_cast<const char*>(a.q) + 2 * ((s.row + i) * a.q_ld + (h * p.group + (r - i * p.group)) * a.q_hs);
#pragma unroll
    for (int ks = 0; ks < KSTEPS; ++ks) {
      const int d = 16 * ks + 8 * hh;
      uint4 x = on && d < dim ? ld16(row + 2 * d) : make_uint4(0, 0, 0, 0);
      q[t][ks] = make_uint4((x.x ^ sign) & keep, (x.y ^ sign) & keep, (x.z ^ sign) & keep, (x.w ^ sign) & keep);
    }
  }

  f32x16 o[QT][DM];
  float m[QT], l[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    m[t] = -INFINITY, l[t] = 0.0f;
#pragma unroll
    for (int i = 0; i < DM; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[t][i][e] = 0.0f;
  }

  // ---------------------------------------------------- a step's keys and values
  // (16-key sub-blocks of a step lie each in one page; their pages are looked up a step
  // before they are read)
  const int64_t S = a.cache.page_size;
  const int shift = __builtin_ctzll(a.cache.page_size), mask = static_cast<int>(S) - 1;
  const int* table = a.rows.table + s.b * a.rows.table_ld;
  const int width = static_cast<int>(a.rows.table_width), pages = static_cast<int>(a.cache.pages);
  const int64_t pstride = static_cast<int64_t>(Hk) * S * dim * ESZ;   // bytes from page to page
  const char* kbase = static_cast<const char*>(a.cache.k) + h * S * dim * ESZ;
  const char* vbase = static_cast<const char*>(a.cache.v) + h * S * dim * ESZ;
  int page0, page1, page2, page3;
  const auto look1 = [&](int t) {   // (t is below 2^31, as the table's end)
    const int x = t >> shift, e = __builtin_amdgcn_readfirstlane(table[x < width ? x : width - 1]);
    return x < width && e >= 0 && e < pages ? e : -1;
  };
  auto look = [&](int i) {
    const int t0 = v.key(i);
    page0 = look1(t0), page1 = look1(t0 + 16), page2 = look1(t0 + 32), page3 = look1(t0 + 48);
  };
  const auto pick = [&](int u) {
    const int lo = u & 1 ? page1 : page0, hi = u & 1 ? page3 : page2;
    return max(u & 2 ? hi : lo, 0);
  };
  uint4 kr[NK], vr[NV];
  // 8-bit: a key's scale goes to its values where they are widened, if their type takes
  // it, else to its scores; the values' to the weights
  constexpr bool KSCALE = E8 && Op::SCALES;
  // (codes: nothing waits for them before they are staged)
  uint32_t ks8[KSCALE ? NK : 1], sc8 = 0;
  int bad = 0;
  // DIRECT: the loads of a step into its turn's tiles.  A wave's load fills 64 chunks:
  // keys (or channels) of whole rows.
  const uint32_t lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)smem));
  const int wu = __builtin_amdgcn_readfirstlane(w);
  uint32_t koff[DIRECT ? NK : 1], voff[DIRECT ? NV : 1];
  if constexpr (DIRECT) {
#pragma unroll
    for (int n = 0; n < NK; ++n) {
      const int row = (64 * (AW_NW * n + w) + lane) / KC;
      koff[n] = 2 * (row * DT) + 16 * ((lane % KC) ^ aw_swap<KS>(row));
    }
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int d = (64 * (AW_NW * n + w) + lane) / VC;
      voff[n] = 2 * static_cast<uint32_t>(d * static_cast<int>(S)) + 16 * ((lane % VC) ^ aw_swap<VS>(d));
    }
  }
  auto load = [&](int i, int turn) {
    const int t0 = v.key(i);
    const uint32_t to = lds + turn * BUF;
    bad = (page0 < 0 ? 1 : 0) | (page1 < 0 ? 2 : 0) | (page2 < 0 ? 4 : 0) | (page3 < 0 ? 8 : 0);
    const auto klds = [&](int n) { return to + 1024 * (AW_NW * n + wu); };
    const auto vlds = [&](int n) { return to + KB + 1024 * (AW_NW * n + wu); };
    if (S >= AT_BLK) {   // (one page for all; its tokens side by side)
      const char* ks = kbase + max(page0, 0) * pstride + 2 * (t0 & mask) * DT;
#pragma unroll
      for (int n = 0; n < NK; ++n) aw_load_lds(ks, koff[n], klds(n));
      const char* vs = vbase + max(page0, 0) * pstride + 2 * (t0 & mask);
#pragma unroll
      for (int n = 0; n < NV; ++n) aw_load_lds(vs, voff[n], vlds(n));
    } else {
#pragma unroll
      for (int n = 0; n < NK; ++n) {
        const int u = 64 * (AW_NW * n + wu) / KC / 16;   // the rows' sub-block
        aw_load_lds(kbase + pick(u) * pstride + 2 * (((t0 + 16 * u) & mask) - 16 * u) * DT, koff[n], klds(n));
      }
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        const int d = (64 * (AW_NW * n + w) + lane) / VC, t = 8 * ((lane % VC) ^ aw_swap<VS>(d));
        aw_load_lds(vbase + pick(t >> 4) * pstride + 2 * (d * static_cast<int>(S) + ((t0 + t) & mask)), vlds(n));
      }
    }
  };
  // ... and, once they are there, what stage() does for a step with masks
  auto settle_tile = [&](int turn) {
    char* vb = smem + turn * BUF + KB;
    uint32_t odd = 0;
#pragma unroll
    for (int n = 0; n < NV; ++n) {   // (the chunks that this lane loaded)
      char* at = vb + 1024 * (AW_NW * n + w) + 16 * lane;
      const uint4 x = ld16(at);
      odd |= not_finite<Op>(x);
      st16(at, finite_or_0<Op>(x));
    }
    if (__any(odd != 0) && lane == 0) atomicOr(&flags[turn], 16);
  };
  auto fetch = [&](int i) {
    const int t0 = v.key(i);
    bad = (page0 < 0 ? 1 : 0) | (page1 < 0 ? 2 : 0) | (page2 < 0 ? 4 : 0) | (page3 < 0 ? 8 : 0);
#pragma unroll
    for (int n = 0; n < NK; ++n) {
      // rows tid / KC + n AW_NT / KC: of one sub-block, or of two
      constexpr int STEP = AW_NT / KC;
      const int row = tid / KC + STEP * n, d = tid % KC * EPC;
      const int u = STEP <= 16 ? STEP * n / 16 : STEP / 16 * n + tid / (16 * KC);
      const char* src = kbase + pick(u) * pstride + ESZ * ((((t0 + 16 * u) & mask) + (row & 15)) * dim + d);
      if constexpr (KSCALE)
        ks8[n] = a.cache.k_scale[(static_cast<int64_t>(pick(u)) * Hk + h) * S + ((t0 + 16 * u) & mask) + (row & 15)];
      if constexpr (FULL) kr[n] = ld16(src);
      else {
        kr[n] = make_uint4(0, 0, 0, 0);
        if constexpr (E8) {   // (a row may start at any multiple of 8 bytes)
          if (d < dim) {
            const uint2 x = *reinterpret_cast<const uint2*>(src);
            kr[n].x = x.x, kr[n].y = x.y;
          }
          if (d + 8 < dim) {
            const uint2 x = *reinterpret_cast<const uint2*>(src + 8);
            kr[n].z = x.x, kr[n].w = x.y;
          }
        } else if (d < dim) kr[n] = ld16(src);
      }
    }
    {
      const int t = tid % VC * EPC;   // this thread's tokens of the step
      const char* src = vbase + pick(t >> 4) * pstride + ESZ * (tid / VC * static_cast<int>(S) + ((t0 + t) & mask));
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        vr[n] = FULL || tid / VC + AW_NT / VC * n < dim ? ld16(src) : make_uint4(0, 0, 0, 0);
        src += ESZ * static_cast<int>(S) * (AW_NT / VC);
        asm("" : "+v"(src));   // (one address that moves, not one for every chunk)
      }
    }
    if constexpr (E8) {
      if (tid < 2 * AT_BLK) {   // keys' scales, values' scales
        const int t = tid & (AT_BLK - 1);
        const uint8_t* src = tid < AT_BLK ? a.cache.k_scale : a.cache.v_scale;
        sc8 = src[(static_cast<int64_t>(pick(t >> 4)) * Hk + h) * S + ((t0 + t) & mask)];
      }
    }
  };
  auto stage = [&](int turn, bool whole) {
    char* buf = smem + turn * BUF;
    uint32_t odd = 0;
#pragma unroll
    for (int n = 0; n < NK; ++n) {
      const int id = tid + AW_NT * n, row = id / KC;
      char* dst = buf + row * KS + id % KC * EPC * 2;
      if constexpr (E8) {
        const float f = KSCALE ? scale_of(ks8[KSCALE ? n : 0]) : 1.0f;
        const uint2 y0 = Op::widen(kr[n].x, f), y1 = Op::widen(kr[n].y, f), y2 = Op::widen(kr[n].z, f), y3 = Op::widen(kr[n].w, f);
        st16(dst, make_uint4(y0.x, y0.y, y1.x, y1.y));
        st16(dst + 16, make_uint4(y2.x, y2.y, y3.x, y3.y));
      } else st16(dst, kr[n]);
    }
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int id = tid + AW_NT * n, d = id / VC;
      char* dst = buf + KB + d * VS + id % VC * EPC * 2;
      // A value that is not finite would reach the rows that do not see its key (0 times
      // it is NaN): in a step with masks such values are taken out here, and added to
      // the rows that see them.
      const auto put = [&](char* to, uint4 x) {
        if (!whole) {
          odd |= not_finite<VOp>(x);
          x = finite_or_0<VOp>(x);
        }
        st16(to, x);
      };
      if constexpr (E8) {
        const uint2 y0 = VOp::widen(vr[n].x), y1 = VOp::widen(vr[n].y), y2 = VOp::widen(vr[n].z), y3 = VOp::widen(vr[n].w);
        put(dst, make_uint4(y0.x, y0.y, y1.x, y1.y));
        put(dst + 16, make_uint4(y2.x, y2.y, y3.x, y3.y));
      } else put(dst, vr[n]);
    }
    if constexpr (E8)
      if (tid < 2 * AT_BLK) reinterpret_cast<float*>(buf + KB + VB)[tid] = scale_of(sc8);
    if (!whole && __any(odd != 0) && lane == 0) atomicOr(&flags[turn], 16);
    if (bad != 0 && tid == 0) atomicOr(&flags[turn], bad);
  };

  if (tid < 2) flags[tid] = 0;
  if (b0 < b1) {
    look(b0);
    if constexpr (DIRECT) load(b0, 0);
    else fetch(b0);
    if (b0 + 1 < b1) look(b0 + 1);
  }
  __syncthreads();
  for (int i = b0; i < b1; ++i) {
    const int turn = (i - b0) & 1;
    const int t0 = v.key(i);
    const bool whole = v.whole(t0);
    if constexpr (DIRECT) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      if (!whole) settle_tile(turn);
      if (bad != 0 && tid == 0) atomicOr(&flags[turn], bad);
      lds_barrier();
      // (all waves are done with the other turn's tiles)
      if (i + 1 < b1) load(i + 1, turn ^ 1);
      if (i + 2 < b1) look(i + 2);
    } else {
      stage(turn, whole);
      if (i + 1 < b1) fetch(i + 1);
      if (i + 2 < b1) look(i + 2);
      lds_barrier();
    }
    const char* kb = smem + turn * BUF;
    const char* vb = kb + KB;
    const int fl = flags[turn];
    const bool masked = !whole || fl != 0;

    // -------------------------------------------------- S^T = K Q^T
    // row m = 8 j + 4 h' + r of a tile of 32 holds key 16 (j / 2) + 8 h' + 4 (j % 2) + r
    const int krow = (c >> 4) * 16 + ((c >> 2) & 1) * 8 + ((c >> 3) & 1) * 4 + (c & 3);
    f32x16 st[QT][2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
      for (int t = 0; t < QT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) st[t][kt][e] = 0.0f;
#pragma unroll
      for (int ks = 0; ks < KSTEPS; ++ks) {
        const int chunk = DIRECT ? (2 * ks + hh) ^ aw_swap<KS>(krow) : 2 * ks + hh;   // (32 more rows change nothing)
        const uint4 kf = ld16(kb + (32 * kt + krow) * KS + 16 * chunk);
#pragma unroll
        for (int t = 0; t < QT; ++t) st[t][kt] = Op::mfma32(kf, q[t][ks], st[t][kt]);
      }
    }
    aw_reads_ahead<2 * KSTEPS>();

    // -------------------------------------------------- the weights
    // (value e of a tile: key 16 (e / 8) + 8 hh + e % 8)
    if constexpr (E8 && !KSCALE) {
      const float* sk = reinterpret_cast<const float*>(vb + VB);
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float f = sk[32 * kt + 16 * (e >> 3) + 8 * hh + (e & 7)];
#pragma unroll
          for (int t = 0; t < QT; ++t) st[t][kt][e] *= f;
        }
    }
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      if (a.softcap > 0.0f) {
        attn_cap(st[t][0], cap);
        attn_cap(st[t][1], cap);
      }
      if (masked) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int k = t0 + 32 * kt + 16 * (e >> 3) + 8 * hh + (e & 7);
            const bool seen = (k <= see[t].last) & ((k >= see[t].from) | (k < v.sinks));
            const float y = fl >> (2 * kt + (e >> 3)) & 1 ? __builtin_nanf("") : st[t][kt][e];
            st[t][kt][e] = seen ? y : -INFINITY;
          }
      }
      float top = -INFINITY;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, st[t][kt][e]);
      top *= to2;
      if (__any(top > m[t] + AT_LAZY)) {
        top = fmaxf(top, shfl_xor(top, 32));
        const float to = top > m[t] + AT_LAZY ? top : m[t];   // (each row by its own scores)
        const float f = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[t] - to);
        m[t] = to;
        l[t] *= f;
#pragma unroll
        for (int dm = 0; dm < DM; ++dm)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[t][dm][e] *= f;
      }
    }

    // -------------------------------------------------- O^T += V^T P^T
    // 16 keys a time: the next 16's weights and values beside this 16's products
    uint4 pf[QT][4], pr[TWO ? QT : 1][2], vf[2][DM];
    const auto weights = [&](int u) {
      const int kt = u >> 1, e0 = 8 * (u & 1);
      float x[QT][8];
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        const float mm = m[t] == -INFINITY ? 0.0f : m[t];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[t][e] = __builtin_amdgcn_exp2f(fmaf(st[t][kt][e0 + e], to2, -mm));
          l[t] += x[t][e];
        }
      }
      if constexpr (E8) {   // (the values' scales)
        const float* sv = reinterpret_cast<const float*>(vb + VB) + AT_BLK + 16 * u + 8 * hh;
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int t = 0; t < QT; ++t) x[t][e] *= sv[e];
      }
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        const auto packed = [&](auto f) {
          return make_uint4(f(x[t][0], x[t][1]), f(x[t][2], x[t][3]), f(x[t][4], x[t][5]), f(x[t][6], x[t][7]));
        };
        if constexpr (TWO) {
          pf[t][u] = packed(weights_first);
          pr[t][u & 1] = packed(weights_rest);
        } else pf[t][u] = packed(VOp::pack);
      }
    };
    const auto values = [&](int u) {
#pragma unroll
      for (int dm = 0; dm < DM; ++dm) {
        const int chunk = DIRECT ? (2 * u + hh) ^ aw_swap<VS>(c) : 2 * u + hh;
        vf[u & 1][dm] = ld16(vb + (32 * dm + c) * VS + 16 * chunk);
      }
    };
    values(0);
    weights(0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (u < 3) values(u + 1);
#pragma unroll
      for (int dm = 0; dm < DM; ++dm)
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          o[t][dm] = VOp::mfma32(vf[u & 1][dm], pf[t][u], o[t][dm]);
          if constexpr (TWO) o[t][dm] = VOp::mfma32(vf[u & 1][dm], pr[t][u & 1], o[t][dm]);
        }
      if (u < 3) {
        weights(u + 1);
        __builtin_amdgcn_sched_group_barrier(0x100, DM, 0);
#pragma unroll
        for (int i = 0; i < DM * QT * (TWO ? 2 : 1); ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x002, 36 / DM, 0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }

    if (fl & 16) {   // (the same for all waves)
      float* wl = reinterpret_cast<float*>(smem + turn * BUF) + w * 16 * 32;   // in the keys' place: [16 keys][32 rows]
      static_assert(AW_NW * 16 * 32 * 4 <= KB, "the waves' weights of 16 keys fit");
#pragma unroll
      for (int t = 0; t < QT; ++t) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          __syncthreads();   // (the keys, or the last weights, have been read)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int k = t0 + 16 * u + 8 * hh + e;
            const bool seen = (k <= see[t].last) & ((k >= see[t].from) | (k < v.sinks));
            const uint32_t x = e < 2 ? pf[t][u].x : e < 4 ? pf[t][u].y : e < 6 ? pf[t][u].z : pf[t][u].w;
            wl[(8 * hh + e) * 32 + c] = seen ? VOp::D::to_f32((e & 1 ? x >> 16 : x) & 0xFFFFu) : -1.0f;
          }
          __syncthreads();
          const int page = paged_page(a.rows, a.cache, s.b, t0 + 16 * u);
          if (page < 0) continue;
          const char* col = static_cast<const char*>(a.cache.v) +
                            ESZ * ((static_cast<int64_t>(page) * Hk + h) * dim * S + ((t0 + 16 * u) & (S - 1)));
#pragma unroll 1
          for (int k = 0; k < 16; ++k) {
            const float x = wl[k * 32 + c];
            if (!(x >= 0.0f)) continue;   // (a NaN weight is in the sums already)
            const char* src = col + ESZ * (4 * hh * S + k);
#pragma unroll
            for (int dm = 0; dm < DM; ++dm)
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                // (one load at a time: this path is rare, the registers are the kernel's)
                asm volatile("" : "+v"(src) : : "memory");
                if (FULL || 32 * dm + 8 * (e >> 2) + 4 * hh + (e & 3) < dim) {
                  float y;
                  if constexpr (E8) y = __builtin_amdgcn_cvt_f32_fp8(static_cast<uint8_t>(*src), 0);
                  else y = Op::D::to_f32(*reinterpret_cast<const uint16_t*>(src));
                  if (!(fabsf(y) < INFINITY)) o[t][dm][e] += x * y;
                }
                src += ESZ * S * ((e & 3) == 3 ? 5 : 1);
              }
          }
        }
      }
      __syncthreads();
    }
    if (fl != 0) {
      __syncthreads();   // (all waves have read the flags)
      if (tid == 0) flags[turn] = 0;
      // (two barriers before the turn's next stage)
    }
  }

  // ---------------------------------------------------- results
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    float ll = l[t] + shfl_xor(l[t], 32);
    const int r = s.tile * TR + 32 * (QT * w + t) + c;
    if (r >= rows) continue;
    const int i = r / p.group;
    if (s.pos + i >= a.rows.table_width * S) ll = __builtin_nanf("");
    const int64_t head = h * p.group + (r - i * p.group), row = (s.row + i) * a.q_heads + head;
    const float inv = v.splits > 1 ? 1.0f : attn_inverse(ll, s.pos + i >= 0);
#pragma unroll
    for (int dm = 0; dm < DM; ++dm)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int d = 32 * dm + 8 * j + 4 * hh;
        if (!FULL && d >= dim) continue;
        const f32x4 y = (f32x4){o[t][dm][4 * j], o[t][dm][4 * j + 1], o[t][dm][4 * j + 2], o[t][dm][4 * j + 3]} * inv;
        if (v.splits > 1) *reinterpret_cast<f32x4*>(p.part + (row * p.splits + split) * dim + d) = y;
        else
          *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + (s.row + i) * a.out_ld + head * a.out_hs + d) =
              make_uint2(Op::pack(y[0], y[1]), Op::pack(y[2], y[3]));
      }
    if (hh == 0) {
      if (v.splits > 1) *reinterpret_cast<float2*>(p.stat + 2 * (row * p.splits + split)) = make_float2(m[t], ll);
      else if (a.out_lse) a.out_lse[row] = ll == 0.0f ? -INFINITY : m[t] == -INFINITY ? ll : (m[t] + log2f(ll)) * 0.6931471805599453f;
    }
  }
}

namespace {

template <class Op, bool E8, int DT, bool FULL>
hipError_t aw_launch(const fl_attn_args& a, const AttnPlan& p, hipStream_t s) {
  constexpr int QT = ATTN_WIDE_QT;
  constexpr int LDS = aw_lds(DT, E8, FULL);
  if (LDS > 65536) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&k_attn_wide<Op, E8, DT, FULL, QT>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((k_attn_wide<Op, E8, DT, FULL, QT>), dim3(static_cast<unsigned>(p.tiles * p.splits * a.cache.heads)), dim3(AW_NT),
                     LDS, s, a, p);
  return hipGetLastError();
}
template <class Op, bool E8>
hipError_t aw_dims(const fl_attn_args& a, const AttnPlan& p, hipStream_t s) {
  switch (a.cache.dim) {
    case 64: return aw_launch<Op, E8, 64, true>(a, p, s);
    case 128: return aw_launch<Op, E8, 128, true>(a, p, s);
    case 256: return aw_launch<Op, E8, 256, true>(a, p, s);
  }
  if (a.cache.dim < 64) return aw_launch<Op, E8, 64, false>(a, p, s);
  if (a.cache.dim < 128) return aw_launch<Op, E8, 128, false>(a, p, s);
  return aw_launch<Op, E8, 256, false>(a, p, s);
}

}  // namespace

hipError_t launch_attn_wide(const fl_attn_args& a, const AttnPlan& p, hipStream_t s) {
  const bool bf = a.dtype == FL_DTYPE_BF16;
  if (a.cache.dtype == FL_DTYPE_E4M3) return bf ? aw_dims<OpBF16, true>(a, p, s) : aw_dims<OpF16, true>(a, p, s);
  return bf ? aw_dims<OpBF16, false>(a, p, s) : aw_dims<OpF16, false>(a, p, s);
}

}  // namespace fl

// Log-probabilities, entropy and log-sum-exp of given tokens from hidden states
// and the lm_head weight, and their gradients, without the [rows, vocab] logits
// in memory.  With logits x[n, v] = sum_d hidden[n, d] weight[v, d] (float32
// accumulators, never rounded to 16 bits) and p = softmax(x[n, :]):
//
//   forward   per row (max, sum e, sum e (x - max)) of each tile of 256
//             vocabulary rows from the product's registers, joined per row;
//   backward  g[n, v] = a (1[v = t] - p) - b p (log p + H) + c p for upstream
//             a, b, c of logprob, entropy, lse; then
//             dhidden[n, d] = sum_v g[n, v] weight[v, d],
//             dweight[v, d] = sum_n g[n, v] hidden[n, d].
//
// Four products of one main loop.  The gradient g of a chunk of the vocabulary
// is written once, in bfloat16, the largest chunk that a bounded workspace holds;
// each product then reads it as its matrix operand.  Its rounding, of at most 2^-8
// relative, is independent from entry to entry, so that a sum of many terms moves
// by as much relative to its terms' norm as rounding the result does; but a row's
// largest entry is its token's, most of the row's dhidden and of that token's
// dweight.  What the rounding took of it is kept in float32 and added to both sums.
// Distance from 64 bits against that of rounding the results alone: of a training
// step of few rows up to 2.3 times without that; with it, of random batches, 1.00 to
// 1.07 times for 4099 tokens and more (255x1024x50257 and 4096x4096x128256: 1.00), up
// to 1.35 for 64 to 512, where a row has several large entries.  A row whose
// probability sits on another token has that one's entry rounded: up to 2.4 times
// in dhidden and 1.55 in that token's dweight, where g lies half way between two
// bf16 values.  (A linear layer in bfloat16 is handed every entry so.)
//
// What bounds them: with few rows the weight's bytes (64x4096x128256: 170 to 217 us
// for 1.05 GB, 6.2 to 4.8 TB/s, by the clock the card holds), with many LDS: the
// fragments of a stage (64 k) of a 256 x 256 tile are 192 KiB read beside 64 KiB
// written, 2048 cycles at 128 bytes a cycle, as many as its matrix instructions
// take.  4096x4096x128256, per product of 4.3 TFLOP: statistics 3.51 ms, g 3.83,
// dhidden 3.48, dweight 3.75 ms (1.12 to 1.24 PFLOP/s; the matrix units busy for 57
// to 65 % of the cycles, LDS without bank conflicts but for the stores' 2 %); a
// library product of that shape, which writes the logits, reaches 1.41 PFLOP/s.
// Tried and slower: 4 waves of 128 x 128, which read a third less of LDS (dweight
// 4.4 ms, dhidden 4.0, g 4.8; the statistics spill); s_setprio around the matrix
// instructions (no change).  255x1024x50257: 35 to 38, 42 to 44, 49 to 52 (with the
// parts' sum) and 56 to 60 us, where the operations of each take 19: 197 tiles of 256
// vocabulary rows on 256 CUs make 19 to 24 in the first two, and as one work-group
// fills a CU's LDS (also with tiles of 64 or 128), nothing runs beside its first
// loads, 16 stages of k (dweight: 4) and its results (dweight: 103 MB written).
#include <algorithm>
#include <type_traits>

#include "fl_device.h"
#include "fl_kernels.h"

namespace fl {

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef short short8v __attribute__((ext_vector_type(8)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef int int32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_8 __attribute__((ext_vector_type(4), aligned(8)));   // (what a caller's results are aligned to,
typedef float floatx4_4 __attribute__((ext_vector_type(4), aligned(4)));    // and `saved`)

constexpr float HL_LOG2E = 1.44269504088896340736f;

// ---------------------------------------------------------------- main loop
// A work-group of 8 waves computes out[j, i] = sum_k A(i, k) B(j, k) for HL_I =
// 256 values of i and BJ of j, with v_mfma_f32_32x32x16_bf16: lane l holds
// column j = l % 32 of a 32 x 32 block and its rows i = 8 (r / 4) + 4 (l / 32) +
// r % 4, r = 0 .. 15, so that a lane's four consecutive results lie side by
// side along i.  Each operand lies in memory either with k contiguous
// ("rows": A(i, k) = p[i * ld + k]) or with i (j) contiguous ("cols":
// p[k * ld + i]).
//
// A stage is 64 k of both tiles, loaded straight into LDS (16 bytes a lane) NST -
// 1 stages ahead.  LDS holds 16-byte granules with an exclusive-or of the row in
// their place, applied to the address each lane loads from, so that the fragment
// reads spread over all banks:
//   rows: granule g (of 8) of row r at r 8 + (g ^ ((r >> 1) & 7)); a lane's 8
//         k of a 32 x 16 fragment are one ds_read_b128;
//   cols: granule g (of BJ / 8) of k-row k at k BJ / 8 + (g ^ (4 (k & 3))), of 8
//         granules 4 (k & 1); a
//         16-lane group's ds_read_b64_tr_b16 takes 4 k-rows of 16 columns and
//         leaves each lane 4 k of its column.
constexpr int HL_I = 256, HL_K = 64, HL_NT = 512, HL_NW = HL_NT / WAVE;

// One operand: a tile's first element, and what may be read from it.
struct Operand {
  const uint16_t* p;   // rows: element (row 0 of the tile, k 0); cols: (k 0, column 0)
  int64_t ld;          // elements
  int rows;            // rows of the tile that exist (rows), k-rows left (cols)
  int width;           // rows: k; cols: columns left from column 0
};

__device__ __forceinline__ int32x4 hl_rsrc(const void* p, uint32_t bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(p);
  int32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane(static_cast<int>(a));
  r[1] = __builtin_amdgcn_readfirstlane(static_cast<int>(a >> 32) & 0xFFFF);
  r[2] = __builtin_amdgcn_readfirstlane(static_cast<int>(bytes));
  r[3] = 0x00020000;
  return r;
}

// 16 bytes per lane from r (voff bytes per lane, soff) to LDS at lds + 16 lane.
// No register is written (m0, which the compiler sets before each use of its own,
// apart); completion is counted in vmcnt.  m0 is read a wait state after it is set.
__device__ __forceinline__ void hl_load_lds(int32x4 r, uint32_t voff, uint32_t soff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(voff), "s"(r), "s"(__builtin_amdgcn_readfirstlane(soff))
               : "memory");
}
template <int N>
__device__ __forceinline__ void hl_wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}

// bytes from the first element to the end of what may be read (below 2^31:
// checked by the host for every shape)
__device__ __forceinline__ uint32_t hl_bytes(int64_t rows, int64_t ld, int64_t width) {
  return rows <= 0 || width <= 0 ? 0u : static_cast<uint32_t>(2 * ((rows - 1) * ld + width));
}

// COLS: the layout; T: rows i (j) of the tile
template <bool COLS, int T>
struct Loader {
  static constexpr int LOADS = T * HL_K * 2 / (HL_NT * 16);   // per thread and stage
  static_assert(LOADS >= 1 && T * HL_K * 2 % (HL_NT * 16) == 0, "whole loads");
  static constexpr int BYTES = T * HL_K * 2;
  Operand o;
  uint32_t voff[LOADS];

  __device__ __forceinline__ void init(const Operand& op) {
    o = op;
    const int lane = threadIdx.x & (WAVE - 1), w = threadIdx.x / WAVE;
#pragma unroll
    for (int p = 0; p < LOADS; ++p) {
      const int q = p * HL_NW + w;   // 1 KiB piece of the tile
      if constexpr (!COLS) {
        const int row = q * 8 + (lane >> 3), g = (lane & 7) ^ ((row >> 1) & 7);
        // (a row that does not exist lies past the range, whatever ld is)
        const uint32_t v = 2u * (static_cast<uint32_t>(row) * static_cast<uint32_t>(o.ld) + 8u * g);
        voff[p] = row < o.rows ? v : 0x80000000u;
      } else {
        constexpr int GR = T / 8;                  // granules of a k-row
        const int k = q * (WAVE / GR) + lane / GR, g = (lane % GR) ^ (4 * (k & 3) & (GR - 1));
        voff[p] = 2u * (static_cast<uint32_t>(k) * static_cast<uint32_t>(o.ld) + 8u * g);
      }
    }
  }
  // what stage s's loads have in common
  struct Stage {
    int32x4 r;
    uint32_t soff;
  };
  __device__ __forceinline__ Stage stage(int s) const {
    if constexpr (!COLS) {
      return {hl_rsrc(o.p, hl_bytes(o.rows, o.ld, o.width)), static_cast<uint32_t>(2 * HL_K * s)};
    } else {
      const int64_t k0 = static_cast<int64_t>(s) * HL_K, left = o.rows - k0;
      return {hl_rsrc(o.p + k0 * o.ld, hl_bytes(left < HL_K ? left : HL_K, o.ld, o.width)), 0u};
    }
  }
  // load p of the stage into the tile in LDS at lds + 1024 times the wave
  __device__ __forceinline__ void load(const Stage& st, int p, uint32_t lds) const {
    hl_load_lds(st.r, voff[p], st.soff, lds + 1024 * p * HL_NW);
  }
};

// The fragments of 32 rows i0 + 32 f .. of a tile in LDS, 16 k from 16 ks.
template <bool COLS, int T, int F>
struct Reader {
  uint32_t at[COLS ? F : 4];
  __device__ __forceinline__ void init(int i0) {
    const int lane = threadIdx.x & (WAVE - 1);
    if constexpr (!COLS) {
      const int row = i0 + (lane & 31);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) at[ks] = 16 * (row * 8 + ((2 * ks + (lane >> 5)) ^ ((row >> 1) & 7)));
    } else {
      const int j = lane & 15, g = lane >> 4;
      const int k = 8 * (g >> 1) + (j >> 2);
#pragma unroll
      for (int f = 0; f < F; ++f) {
        const int col = i0 + 32 * f + 16 * (g & 1) + 4 * (j & 3);
        at[f] = 16 * (k * (T / 8) + ((col >> 3) ^ (4 * (k & 3) & (T / 8 - 1)))) + 2 * (col & 7);
      }
    }
  }
  __device__ __forceinline__ bf16x8 read(const char* tile, int f, int ks) const {
    if constexpr (!COLS) {
      return *reinterpret_cast<const bf16x8*>(tile + at[ks] + f * 32 * 128);
    } else {
      typedef __attribute__((address_space(3))) short4v* lds4;
      const char* p = tile + at[f] + ks * 16 * T * 2;
      const short4v a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p));
      const short4v b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p + 4 * T * 2));
      return __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
};

// Wave grid WI x WJ of FI x FJ blocks of 32 x 32 per wave; NST stages in LDS, and
// beside them an area for the epilogues.
template <int BJ_>
struct Shape {
  static constexpr int BJ = BJ_, WJ = BJ / 64, WI = HL_NW / WJ, FI = HL_I / (32 * WI), FJ = BJ / (32 * WJ);
  static constexpr int STAGE = (HL_I + BJ) * HL_K * 2;
  static constexpr int NST = BJ == 256 ? 2 : 3;
  static constexpr int AREA_W = BJ == 128 ? 2048 : 4096;   // per wave
  static constexpr int LDS = NST * STAGE + HL_NW * AREA_W;
  static_assert(LDS <= 160 * 1024, "LDS");
};

// Tiles of a launch: ni of 256 along i, nj of BJ along j, nz ranges of k.  Work-group
// b of a grid of at most one per CU takes every (grid / 8)-th tile of its XCD's
// share (work-groups go round the 8 XCDs): a contiguous range of an order in
// which 8 j-tiles share each i-tile, so that the work-groups of an XCD read the
// same few rows through its L2.
struct Tiles {
  int ni, nj, nz;
  __device__ __forceinline__ int count() const { return ni * nj * nz; }
  __device__ __forceinline__ void at(int t, int& i, int& j, int& z) const {
    z = t / (ni * nj);
    t -= z * ni * nj;
    const int per = 8 * ni, grp = t / per, in = t - grp * per, gj = min(8, nj - 8 * grp);
    i = in / gj;
    j = 8 * grp + in % gj;
  }
};
// The tiles of one work-group: first, first + step, ... below end.
struct Share {
  int t, end, step;
};
__device__ __forceinline__ Share hl_share(const Tiles& ts) {
  const int n = ts.count(), x = blockIdx.x % 8, q = blockIdx.x / 8;
  const int lo = x * (n / 8) + min(x, n % 8);
  // (work-groups of XCD x in the grid)
  const int step = (static_cast<int>(gridDim.x) - x + 7) / 8;
  return {lo + q, lo + n / 8 + (x < n % 8 ? 1 : 0), step};
}

// The products of a work-group's tiles, one after another without a gap in the
// loads: operands(t, A, B) says what tile t reads and returns its stages (one or
// more); epilogue(t, acc) takes its results.  A stage's last fragments are in
// registers when the work-group meets (all have read the stage, the next has
// landed); the next stage's first fragments are read, and the loads into the
// stage's place issued, ahead of the last quarter of its matrix instructions.
// While an epilogue runs, the next tile's first stages are on their way: it calls
// hl_wait_vm<0>() before its first store, so that no later wait for a load waits
// for a store.
template <bool ACOLS, bool BCOLS, class S, class OPS, class EPI>
__device__ __forceinline__ void hl_products(const Tiles& ts, char* smem, OPS&& operands, EPI&& epilogue) {
  constexpr int NST = S::NST, BJ = S::BJ;
  using LA = Loader<ACOLS, HL_I>;
  using LB = Loader<BCOLS, BJ>;
  constexpr int L = LA::LOADS + LB::LOADS;
  const Share sh = hl_share(ts);
  if (sh.t >= sh.end) return;
  const int w = threadIdx.x / WAVE;
  Reader<ACOLS, HL_I, S::FI> ra;
  Reader<BCOLS, BJ, S::FJ> rb;
  ra.init((w / S::WJ) * 32 * S::FI);
  rb.init((w % S::WJ) * 32 * S::FJ);
  const uint32_t lds = static_cast<uint32_t>(
      reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)(smem)));

  // the load cursor: tile lt, its next stage ls of ln, into buffer lbuf
  LA la;
  LB lb;
  int lt = sh.t, ls = 0, ln = 0, lbuf = 0;
  auto open = [&]() {
    Operand A, B;
    ln = operands(lt, A, B);
    la.init(A);
    lb.init(B);
    ls = 0;
  };
  typename LA::Stage sa;
  typename LB::Stage sb;
  uint32_t to = 0;
  auto aim = [&](bool on) {   // at the cursor's stage; past the last, at nothing (zeros into a free place)
    sa = la.stage(ls);
    sb = lb.stage(ls);
    sa.r[2] = on ? sa.r[2] : 0;
    sb.r[2] = on ? sb.r[2] : 0;
    to = lds + lbuf * S::STAGE + 1024 * __builtin_amdgcn_readfirstlane(w);
  };
  auto load = [&](int p) {
    if (p < LA::LOADS) la.load(sa, p, to);
    else lb.load(sb, p - LA::LOADS, to + LA::BYTES);
  };
  auto advance = [&]() {
    lbuf = lbuf == NST - 1 ? 0 : lbuf + 1;
    if (++ls == ln) {
      lt += sh.step;
      if (lt < sh.end) open();
    }
  };
  open();
  int stages = ln;     // of the current tile
  int ahead = 0;       // stages issued past the current one ...
  int landed = 0;      // ... and how many of them this wave has waited for
#pragma unroll 1
  for (int s = 0; s < NST && lt < sh.end; ++s) {
    aim(true);
#pragma unroll
    for (int p = 0; p < L; ++p) load(p);
    advance();
    if (s == 0) hl_wait_vm<0>();
    else ++ahead;
  }
  lds_barrier();

  bf16x8 fa[2][S::FI], fb[2][S::FJ];
  int buf = 0;
  auto read = [&](int slot, int b, int ks) {
    const char* ta = smem + b * S::STAGE;
    const char* tb = ta + LA::BYTES;
#pragma unroll
    for (int i = 0; i < S::FI; ++i) fa[slot][i] = ra.read(ta, i, ks);
#pragma unroll
    for (int j = 0; j < S::FJ; ++j) fb[slot][j] = rb.read(tb, j, ks);
  };
  constexpr int M = S::FI * S::FJ, KS = HL_K / 16;
#pragma unroll 1
  for (int t = sh.t; t < sh.end; t += sh.step) {
    floatx16 acc[S::FI][S::FJ];
#pragma unroll
    for (int i = 0; i < S::FI; ++i)
#pragma unroll
      for (int j = 0; j < S::FJ; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
    auto mfma = [&](int slot, int m) {
      const int i = m / S::FJ, j = m % S::FJ;
      acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[slot][i], fb[slot][j], acc[i][j], 0, 0, 0);
    };
    read(0, buf, 0);
#pragma unroll 1
    for (int s = 0; s < stages; ++s) {
#pragma unroll
      for (int ks = 0; ks < KS - 1; ++ks) {
        // (the next fragments are on their way while these are multiplied)
        read((ks + 1) & 1, buf, ks + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int m = 0; m < M; ++m) mfma(ks & 1, m);
        __builtin_amdgcn_sched_barrier(0);
      }
      constexpr int last = (KS - 1) & 1;
      if (ahead > 0) {
        if (landed > 0) --landed;
        else if (NST > 2 && ahead > 1) hl_wait_vm<L>();   // (the newest stage may be on its way)
        else hl_wait_vm<0>();
        lds_barrier();
        --ahead;
        buf = buf == NST - 1 ? 0 : buf + 1;
        if (s + 1 < stages) read(0, buf, 0);   // (a tile's first ones after the epilogue, which needs the registers)
      }
      // (also past the last stage, without a branch: into the place of one that
      // every wave has read)
      const bool more = lt < sh.end;
      aim(more);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int m = 0; m < M; ++m) {
        mfma(last, m);
#pragma unroll
        for (int p = m * L / M; p < (m + 1) * L / M; ++p) load(p);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (more) {
        advance();
        ++ahead;
      }
    }
    epilogue(t, acc);
    landed = ahead;
    if (t + sh.step < sh.end) {
      Operand A, B;
      stages = operands(t + sh.step, A, B);
    }
  }
}

// A wave's results as bfloat16 rows: out[j, i0 ...] for its 32 x 32 blocks,
// through its area of LDS, so that every store is 16 bytes of rows of 64 or 128.
// row(j) is the row's first element of the wave's i range, NULL for none; left: the
// elements of the range that exist, a multiple of 8.  Called by whole waves.
template <class S, class ROW>
__device__ __forceinline__ void hl_store_rows(const floatx16 (&acc)[S::FI][S::FJ], char* area, int left, ROW&& row) {
  constexpr int PI = S::FI < S::AREA_W / 2048 ? S::FI : S::AREA_W / 2048;   // i-blocks of a turn: rows of 64 PI bytes
  constexpr int GR = 4 * PI;                  // 16-byte granules of a row
  static_assert(32 * GR * 16 <= S::AREA_W, "the wave's area");
  int lane = threadIdx.x & (WAVE - 1);
  asm volatile("" : "+v"(lane));   // (what follows from it is not kept over the product's loop)
  const int r = lane & 31, h = lane >> 5;
#pragma unroll
  for (int j = 0; j < S::FJ; ++j)
#pragma unroll
    for (int ib = 0; ib < S::FI; ib += PI) {
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int i = 0; i < PI; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t o[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = BF16::from_f32(acc[ib + i][j][4 * q + e]);
          const int g = (4 * i + q) ^ (r & (GR - 1));
          *reinterpret_cast<uint2*>(area + 16 * (r * GR + g) + 8 * h) = make_uint2(o[0] | (o[1] << 16), o[2] | (o[3] << 16));
        }
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int p = 0; p < 32 * GR / WAVE; ++p) {
        const int rr = p * (WAVE / GR) + lane / GR, g = lane % GR;
        const uint4 v = *reinterpret_cast<const uint4*>(area + 16 * (rr * GR + (g ^ (rr & (GR - 1)))));
        uint16_t* out = row(32 * j + rr);
        const int i = 32 * ib + 8 * g;
        if (out != nullptr && i < left) *reinterpret_cast<u32x4_8*>(out + i) = u32x4_8{v.x, v.y, v.z, v.w};
        __builtin_amdgcn_sched_barrier(0);   // (one address live at a time)
      }
    }
}

// ---------------------------------------------------------------- forward
struct HlArgs {
  const uint16_t* hidden;   // [rows, dim], ld
  const uint16_t* weight;   // [vocab, dim]
  int64_t ld;
  int rows, dim, vocab;
  const int64_t* tokens;
  int64_t ignore_index;
};

// Operands of the logits' product: vocabulary rows v0 .., rows n0 ..; the stages.
template <int BJ>
__device__ __forceinline__ int hl_logits_operands(const HlArgs& a, int v0, int n0, Operand& A, Operand& B) {
  A = {a.weight + static_cast<int64_t>(v0) * a.dim, a.dim, min(HL_I, a.vocab - v0), a.dim};
  B = {a.hidden + n0 * a.ld, a.ld, min(BJ, a.rows - n0), a.dim};
  return a.dim / HL_K;
}

}  // namespace

// part[tile rows + n]: max, sum e, sum e d2 of the tile's vocabulary rows, in the
// order rows run so that a join's loads are coalesced
template <int BJ>
__global__ __launch_bounds__(HL_NT) __attribute__((amdgpu_waves_per_eu(2, 2))) void k_head_stats(const HlArgs a, float4* part,
                                                                                               float* xt, const Tiles ts) {
  using S = Shape<BJ>;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  float* wave_part = reinterpret_cast<float*>(smem + S::NST * S::STAGE);   // [WI][BJ][3]
  static_assert(S::WI * BJ * 12 <= HL_NW * S::AREA_W, "the area");
  const int lane = threadIdx.x & (WAVE - 1), w = threadIdx.x / WAVE;
  const int wi = w / S::WJ, wj = w % S::WJ;
  constexpr float NINF = -__builtin_inff();
  hl_products<false, false, S>(
      ts, smem,
      [&](int t, Operand& A, Operand& B) {
        int i, j, z;
        ts.at(t, i, j, z);
        return hl_logits_operands<BJ>(a, i * HL_I, j * BJ, A, B);
      },
      [&](int t, floatx16 (&acc)[S::FI][S::FJ]) {
        int ti, tj, z;
        ts.at(t, ti, tj, z);
        const int v0 = ti * HL_I, n0 = tj * BJ;
        const int vw = v0 + wi * 32 * S::FI + 4 * (lane >> 5);   // the lane's first vocabulary row
        lds_barrier();   // (the last tile's parts are read)
        if (v0 + HL_I > a.vocab) {
#pragma unroll
          for (int i = 0; i < S::FI; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (vw + 32 * i + 8 * (r / 4) + r % 4 >= a.vocab) {
#pragma unroll
                for (int j = 0; j < S::FJ; ++j) acc[i][j][r] = NINF;
              }
        }
#pragma unroll
        for (int j = 0; j < S::FJ; ++j) {
          float m = NINF;
#pragma unroll
          for (int i = 0; i < S::FI; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) m = fmaxf(m, acc[i][j][r]);
          m = fmaxf(m, __shfl_xor(m, 32, WAVE));
          const float ref = m == NINF ? 0.0f : m;
          float s[2] = {0.0f, 0.0f}, u[2] = {0.0f, 0.0f};
#pragma unroll
          for (int i = 0; i < S::FI; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const float d2 = (acc[i][j][r] - ref) * HL_LOG2E;
              const float e = __builtin_amdgcn_exp2f(d2);
              s[r & 1] += e;
              u[r & 1] = fmaf(e, fmaxf(d2, -200.0f), u[r & 1]);   // (e is 0 there)
            }
          float ss = s[0] + s[1], uu = u[0] + u[1];
          ss += __shfl_xor(ss, 32, WAVE);
          uu += __shfl_xor(uu, 32, WAVE);
          if (lane < 32) {
            float* wp = wave_part + 3 * (wi * BJ + wj * 32 * S::FJ + 32 * j + lane);
            wp[0] = m;
            wp[1] = ss;
            wp[2] = uu;
          }
        }
        hl_wait_vm<0>();
        // the tokens' logits, by the lanes that have them
#pragma unroll
        for (int j = 0; j < S::FJ; ++j) {
          const int n = n0 + wj * 32 * S::FJ + 32 * j + (lane & 31);
          const int64_t tk = a.tokens && n < a.rows ? a.tokens[n] : -1;
          const int64_t d = tk - vw;
          if (tk >= 0 && tk < a.vocab && d >= 0 && d < 32 * S::FI) {
#pragma unroll
            for (int i = 0; i < S::FI; ++i)
#pragma unroll
              for (int r = 0; r < 16; ++r) {
                if (d == 32 * i + 8 * (r / 4) + r % 4) xt[n] = acc[i][j][r];
                __builtin_amdgcn_sched_barrier(0);   // (one comparison live at a time)
              }
          }
        }
        lds_barrier();
        // the tile's part of each row: the waves' joined
        const int q = threadIdx.x;
        if (q < BJ && n0 + q < a.rows) {
          float m = NINF, s = 0.0f, u = 0.0f;
#pragma unroll
          for (int i = 0; i < S::WI; ++i) m = fmaxf(m, wave_part[3 * (i * BJ + q)]);
          const float ref = m == NINF ? 0.0f : m;
#pragma unroll
          for (int i = 0; i < S::WI; ++i) {
            const float* wp = wave_part + 3 * (i * BJ + q);
            const float d = (wp[0] - ref) * HL_LOG2E, f = __builtin_amdgcn_exp2f(d);
            s = fmaf(wp[1], f, s);
            u = fmaf(fmaf(wp[1], fmaxf(d, -200.0f), wp[2]), f, u);
          }
          part[static_cast<int64_t>(ti) * a.rows + n0 + q] = make_float4(m, s, u, 0.0f);
        }
      });
}

// The parts of each row joined: 8 rows per work-group, 32 threads each, in
// float64 and in a fixed order.
constexpr int HJ_R = 8, HJ_P = 32;
__global__ __launch_bounds__(HJ_R * HJ_P) void k_head_join(const fl_head_args a, const float4* part, const float* xt,
                                                           int parts) {
  __shared__ float sm[HJ_P / 8][HJ_R];
  __shared__ double ss[HJ_P / 8][HJ_R], su[HJ_P / 8][HJ_R];
  const int r = threadIdx.x % HJ_R, p0 = threadIdx.x / HJ_R, w = threadIdx.x / WAVE;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * HJ_R + r;
  const bool on = n < a.rows;
  const float ninf = -__builtin_inff();
  // (a thread's parts relative to its own maximum; of -inf alone m stays -inf,
  // and a NaN sum stays NaN)
  float m = ninf;
  double s = 0.0, u = 0.0;
  if (on) {
#pragma unroll 4
    for (int p = p0; p < parts; p += HJ_P) {
      const float4 q = part[static_cast<int64_t>(p) * a.rows + n];
      const float nm = fmaxf(m, q.x), ref = nm == ninf ? 0.0f : nm;
      const float d0 = (m - ref) * HL_LOG2E, d1 = (q.x - ref) * HL_LOG2E;
      const double f0 = __builtin_amdgcn_exp2f(d0), f1 = __builtin_amdgcn_exp2f(d1);
      u = (u + s * static_cast<double>(fmaxf(d0, -200.0f))) * f0 + (static_cast<double>(q.z) + q.y * fmaxf(d1, -200.0f)) * f1;
      s = s * f0 + q.y * f1;
      m = nm;
    }
  }
  float M = m;
  for (int x = HJ_R; x < WAVE; x <<= 1) M = fmaxf(M, __shfl_xor(M, x, WAVE));
  if ((threadIdx.x & (WAVE - 1)) < HJ_R) sm[w][r] = M;
  __syncthreads();
  M = sm[0][r];
#pragma unroll
  for (int i = 1; i < HJ_P / 8; ++i) M = fmaxf(M, sm[i][r]);
  {
    const float ref = M == ninf ? 0.0f : M, d = (m - ref) * HL_LOG2E;
    const double f = __builtin_amdgcn_exp2f(d);
    u = (u + s * static_cast<double>(fmaxf(d, -200.0f))) * f;
    s *= f;
  }
  for (int x = HJ_R; x < WAVE; x <<= 1) {
    s += __shfl_xor(s, x, WAVE);
    u += __shfl_xor(u, x, WAVE);
  }
  if ((threadIdx.x & (WAVE - 1)) < HJ_R) {
    ss[w][r] = s;
    su[w][r] = u;
  }
  __syncthreads();
  if (p0 != 0 || !on) return;
  m = M;
  s = ss[0][r];
  u = su[0][r];
#pragma unroll
  for (int i = 1; i < HJ_P / 8; ++i) {
    s += ss[i][r];
    u += su[i][r];
  }
  const float nan = __builtin_nanf("");
  const bool okr = s > 0.0 && s < static_cast<double>(__builtin_inff());
  const double logs = log(s), ref = static_cast<double>(m);
  const float ent = okr ? static_cast<float>(logs - u / s / static_cast<double>(HL_LOG2E)) : nan;
  if (a.out_entropy) a.out_entropy[n] = ent;
  if (a.out_lse) a.out_lse[n] = okr ? static_cast<float>(ref + logs) : s == 0.0 ? ninf : nan;
  if (a.tokens && a.out_logprob) {
    const int64_t t = a.tokens[n];
    const bool bad = t < 0 || t >= a.vocab || !okr;
    a.out_logprob[n] = t == a.ignore_index ? -0.0f : bad ? nan : static_cast<float>((static_cast<double>(xt[n]) - ref) - logs);
  }
  if (a.out_saved) {   // as fl_score_tokens
    float* sv = a.out_saved + 4 * n;
    sv[0] = okr ? m : nan;
    sv[1] = okr ? static_cast<float>(logs) : nan;
    sv[2] = a.out_entropy ? ent : nan;
    const int64_t t = a.tokens ? a.tokens[n] : -1;
    sv[3] = t >= 0 && t < a.vocab ? xt[n] : nan;   // (0 there)
  }
}

// ---------------------------------------------------------------- backward
namespace {
struct HlGrad {
  const float* saved;
  const float *ga, *gb, *gc;   // upstream of logprob, entropy, lse (NULL: 0)
};
// What rounding took of g at a row's token v, if that lies in a chunk that was
// written (else -1).
struct HlFix {
  int v;
  float r;
};
// acc += r x for a lane's column of a wave's blocks and the bf16 x[first ...] of
// width elements (those past it go to results that nobody stores; all loads ahead
// of the first use).
template <int FI>
__device__ __forceinline__ void hl_add(floatx16 (&acc)[FI], float r, const uint16_t* x, int first, int width) {
  uint2 w[FI][4];
#pragma unroll
  for (int i = 0; i < FI; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) w[i][q] = *reinterpret_cast<const uint2*>(x + min(first + 32 * i + 8 * q, width - 4));
#pragma unroll
  for (int i = 0; i < FI; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint32_t u[2] = {w[i][q].x, w[i][q].y};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        acc[i][4 * q + e] = fmaf(r, BF16::to_f32(e % 2 == 0 ? u[e / 2] & 0xFFFFu : u[e / 2] >> 16), acc[i][4 * q + e]);
    }
}
}  // namespace

// g of the vocabulary rows c0 .. c0 + cn - 1 (cn a multiple of 64; those past
// the vocabulary 0), bfloat16 [rows, cn]
template <int BJ>
__global__ __launch_bounds__(HL_NT) __attribute__((amdgpu_waves_per_eu(2, 2))) void k_head_g(const HlArgs a, const HlGrad gr,
                                                                                           uint16_t* g, int c0, int cn,
                                                                                           const Tiles ts) {
  using S = Shape<BJ>;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int lane = threadIdx.x & (WAVE - 1), w = threadIdx.x / WAVE;
  const int wi = w / S::WJ, wj = w % S::WJ;
  char* area = smem + S::NST * S::STAGE + w * S::AREA_W;
  hl_products<false, false, S>(
      ts, smem,
      [&](int t, Operand& A, Operand& B) {
        int i, j, z;
        ts.at(t, i, j, z);
        return hl_logits_operands<BJ>(a, c0 + i * HL_I, j * BJ, A, B);
      },
      [&](int t, floatx16 (&acc)[S::FI][S::FJ]) {
        int ti, tj, z;
        ts.at(t, ti, tj, z);
        const int i0 = ti * HL_I + wi * 32 * S::FI, n0 = tj * BJ + wj * 32 * S::FJ;   // of the wave
        const int vw = c0 + i0 + 4 * (lane >> 5);                                     // the lane's first vocabulary row
#pragma unroll
        for (int j = 0; j < S::FJ; ++j) {
          const int n = min(n0 + 32 * j + (lane & 31), a.rows - 1);   // (rows past the last are not stored)
          const float hi = gr.saved[4 * n], lo = gr.saved[4 * n + 1], H = gr.saved[4 * n + 2];
          const float gb = gr.gb ? gr.gb[n] : 0.0f, gc = gr.gc ? gr.gc[n] : 0.0f;
          float ga = gr.ga ? gr.ga[n] : 0.0f;
          int d = -1;   // the token's place from the lane's first row
          if (a.tokens) {
            const int64_t tk = a.tokens[n];
            if (tk == a.ignore_index) ga = 0.0f;
            else if (tk < 0 || tk >= a.vocab) ga = ga == 0.0f ? 0.0f : __builtin_nanf("");
            else d = static_cast<int>(tk) - vw;
          }
          const bool zero = ga == 0.0f && gb == 0.0f && gc == 0.0f;
          const float k0 = gc - ga, h = gb == 0.0f ? 0.0f : H;
#pragma unroll
          for (int i = 0; i < S::FI; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int at = 32 * i + 8 * (r / 4) + r % 4;
              const float l = (acc[i][j][r] - hi) - lo;
              const float p = __builtin_amdgcn_exp2f(l * HL_LOG2E);
              float v = p * (k0 - gb * (fmaxf(l, -200.0f) + h));
              if (at == d) v += ga;
              acc[i][j][r] = zero || vw + at >= a.vocab ? 0.0f : v;
              if (r % 4 == 3) __builtin_amdgcn_sched_barrier(0);   // (four results' temporaries live at a time)
            }
        }
        hl_wait_vm<0>();
        uint16_t* out = g + static_cast<int64_t>(n0) * cn + i0;
        const int rows = a.rows - n0;
        hl_store_rows<S>(acc, area, cn - i0, [&](int q) { return q < rows ? out + static_cast<int64_t>(q) * cn : nullptr; });
      });
}

// What rounding took of g at the rows' tokens in a chunk: g in float32 from the
// token's logit that the forward pass left, less what k_head_g wrote.  No more than
// a rounding: of a forward call with other tokens it is 0 or as small.  A wave takes
// 64 vocabulary rows and looks for them among the tokens: fix by row, for dhidden,
// and list by vocabulary row, for dweight: the 64 first rows with such a token, v
// their number times 64 and the place, 0 behind the last.
// 255x1024x50257 5 us, 4096x4096x128256 13 us for each of two chunks; what dweight
// does with the list is 4 of its 56 us at the first size and not seen at the second.
constexpr int HL_LIST = 64;
__global__ __launch_bounds__(256) void k_head_fix(const HlArgs a, const HlGrad gr, const uint16_t* g, HlFix* fix, HlFix* list,
                                                  int c0, int cn) {
  const int lane = threadIdx.x & (WAVE - 1), bin = blockIdx.x * (256 / WAVE) + threadIdx.x / WAVE;
  if (bin >= cn / HL_LIST) return;
  const int v0 = c0 + bin * HL_LIST, v1 = min(a.vocab, v0 + HL_LIST);
  int count = 0;
  constexpr int U = 8;
#pragma unroll 1
  for (int nb = 0; nb < a.rows; nb += U * WAVE) {
    int64_t tk[U];
#pragma unroll
    for (int u = 0; u < U; ++u) tk[u] = a.tokens ? a.tokens[min(nb + u * WAVE + lane, a.rows - 1)] : -1;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int n = nb + u * WAVE + lane;
      // (the first wave of the first chunk: rows whose token lies in no chunk yet have none)
      if (c0 == 0 && bin == 0 && n < a.rows && (tk[u] < 0 || tk[u] >= min(a.vocab, cn))) fix[n] = HlFix{-1, 0.0f};
      const bool in = n < a.rows && tk[u] >= v0 && tk[u] < v1;
      const uint64_t hits = __ballot(in);
      if (hits == 0) continue;
      if (in) {
        const float ga = gr.ga && tk[u] != a.ignore_index ? gr.ga[n] : 0.0f;
        const float gb = gr.gb ? gr.gb[n] : 0.0f, gc = gr.gc ? gr.gc[n] : 0.0f;
        const floatx4_4 sv = reinterpret_cast<const floatx4_4*>(gr.saved)[n];
        const float l = (sv.w - sv.x) - sv.y, p = __builtin_amdgcn_exp2f(l * HL_LOG2E);
        const float v = p * (gc - ga - gb * (fmaxf(l, -200.0f) + (gb == 0.0f ? 0.0f : sv.z))) + ga;
        const float was = BF16::to_f32(g[static_cast<int64_t>(n) * cn + (tk[u] - c0)]), lost = v - was;
        const float r = __builtin_fabsf(lost) <= __builtin_fabsf(was) * 0x1.02p-8f ? lost : 0.0f;   // (NaN: 0)
        fix[n] = HlFix{static_cast<int>(tk[u]), r};
        const int at = count + __popcll(hits & ((1ull << lane) - 1ull));
        if (at < HL_LIST) list[bin * HL_LIST + at] = HlFix{n * HL_LIST + static_cast<int>(tk[u] - v0), r};
      }
      count += __popcll(hits);
    }
  }
  if (lane >= count) list[bin * HL_LIST + lane] = HlFix{0, 0.0f};
}

// dweight[c0 + v, d] = sum_n g[n, v] hidden[n, d]: i = d, j = v.  (Tiles of 128 or
// 64 vocabulary rows are slower where those of 256 fill the CUs, also for few rows:
// 255x1024x50257 58, 61, 73 us.)
// What rounding took of g at the rows' tokens comes to the sums of the tokens'
// rows: a wave's 64 vocabulary rows take one row's part each at a time, in the
// order of the rows, in HL_FIXES turns at most, which bounds the time where many
// rows have one token (more rows' roundings are as independent as any; 4096 rows
// of one token in a vocabulary of 64 would be 4096 turns of about a microsecond).
constexpr int HL_FIXES = 16;
template <int BJ>
__global__ __launch_bounds__(HL_NT) __attribute__((amdgpu_waves_per_eu(2, 2))) void k_head_dw(const HlArgs a, const uint16_t* g,
                                                                                            const HlFix* list, uint16_t* dw,
                                                                                            int c0, int cn, const Tiles ts) {
  using S = Shape<BJ>;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int w = threadIdx.x / WAVE;
  char* area = smem + S::NST * S::STAGE + w * S::AREA_W;
  hl_products<true, true, S>(
      ts, smem,
      [&](int t, Operand& A, Operand& B) {
        int i, j, z;
        ts.at(t, i, j, z);
        A = {a.hidden + i * HL_I, a.ld, a.rows, a.dim - i * HL_I};
        B = {g + j * S::BJ, cn, a.rows, cn - j * S::BJ};
        return (a.rows + HL_K - 1) / HL_K;
      },
      [&](int t, floatx16 (&acc)[S::FI][S::FJ]) {
        int ti, tj, z;
        ts.at(t, ti, tj, z);
        const int d0 = ti * HL_I + (w / S::WJ) * 32 * S::FI, v0 = c0 + tj * S::BJ + (w % S::WJ) * 32 * S::FJ;
        uint16_t* out = dw + static_cast<int64_t>(v0) * a.dim + d0;
        const int rows = min(a.vocab, c0 + cn) - v0;
        const int lane = threadIdx.x & (WAVE - 1);
        static_assert(32 * S::FJ == HL_LIST, "a wave's vocabulary rows are a list's");
        const HlFix f = rows > 0 ? list[v0 - c0 + lane] : HlFix{0, 0.0f};   // (beside the next tile's loads)
        hl_wait_vm<0>();
        int qn[2] = {0, 0}, turns = 0;
        float qr[2] = {0.0f, 0.0f};   // the lane's columns' parts that wait; 0: none
        uint64_t wait = 0;            // the columns that have one
        uint64_t hits = __ballot(f.r != 0.0f);
#pragma unroll 1
        while ((hits | wait) != 0 && turns < HL_FIXES) {   // (the same way for the whole wave)
          const bool end = hits == 0;
          const int b = end ? 0 : __builtin_ctzll(hits);
          const int e = __builtin_amdgcn_readlane(f.v, b), v = e % HL_LIST;
          if (end || (wait >> v & 1)) {
#pragma unroll
            for (int j = 0; j < S::FJ; ++j) {
              if (qr[j] != 0.0f) {
                floatx16 col[S::FI];
#pragma unroll
                for (int i = 0; i < S::FI; ++i) col[i] = acc[i][j];
                hl_add<S::FI>(col, qr[j], a.hidden + qn[j] * a.ld, d0 + 4 * (lane >> 5), a.dim);
#pragma unroll
                for (int i = 0; i < S::FI; ++i) acc[i][j] = col[i];
              }
              qr[j] = 0.0f;
            }
            wait = 0;
            ++turns;
          } else {
            hits &= hits - 1;
            wait |= 1ull << v;
            const float r = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f.r), b));
#pragma unroll
            for (int j = 0; j < S::FJ; ++j)
              if (v - 32 * j == (lane & 31)) {
                qn[j] = e / HL_LIST;
                qr[j] = r;
              }
          }
        }
        hl_store_rows<S>(acc, area, a.dim - d0, [&](int q) { return q < rows ? out + static_cast<int64_t>(q) * a.dim : nullptr; });
      });
}

// dhidden's part z: sum over the z-th of nz ranges of the chunk's vocabulary
// rows of g[n, v] weight[c0 + v, d]: i = d, j = n.  The part is written, or (for a
// chunk after the first) added to; DIRECT: one part in all, rounded into dhidden.
template <int BJ, bool DIRECT>
__global__ __launch_bounds__(HL_NT) __attribute__((amdgpu_waves_per_eu(2, 2))) void k_head_dh(const HlArgs a, const uint16_t* g,
                                                                                            const HlFix* fix, float* sum,
                                                                                            uint16_t* dh, int c0, int cn,
                                                                                            const Tiles ts, int per, int first) {
  using S = Shape<BJ>;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int lane = threadIdx.x & (WAVE - 1), w = threadIdx.x / WAVE;
  char* area = smem + S::NST * S::STAGE + w * S::AREA_W;
  hl_products<true, false, S>(
      ts, smem,
      [&](int t, Operand& A, Operand& B) {
        int i, j, z;
        ts.at(t, i, j, z);
        // (the host's nz leaves no range empty)
        const int k0 = z * per * HL_K, stages = min(cn / HL_K - z * per, per);
        A = {a.weight + static_cast<int64_t>(c0 + k0) * a.dim + i * HL_I, a.dim, min(stages * HL_K, a.vocab - c0 - k0),
             a.dim - i * HL_I};
        B = {g + static_cast<int64_t>(j) * BJ * cn + k0, cn, min(BJ, a.rows - j * BJ), stages * HL_K};
        return stages;
      },
      [&](int t, floatx16 (&acc)[S::FI][S::FJ]) {
        int ti, tj, z;
        ts.at(t, ti, tj, z);
        const int d0 = ti * HL_I + (w / S::WJ) * 32 * S::FI, n0 = tj * BJ + (w % S::WJ) * 32 * S::FJ;
        const int rows = a.rows - n0;
        hl_wait_vm<0>();
        if constexpr (DIRECT) {
#pragma unroll
          for (int j = 0; j < S::FJ; ++j) {
            const int n = 32 * j + (lane & 31), d = d0 + 4 * (lane >> 5);
            const HlFix f = fix[n0 + min(n, rows - 1)];
            if (f.r == 0.0f || n >= rows) continue;
            floatx16 col[S::FI];
#pragma unroll
            for (int i = 0; i < S::FI; ++i) col[i] = acc[i][j];
            hl_add<S::FI>(col, f.r, a.weight + static_cast<int64_t>(f.v) * a.dim, d, a.dim);
#pragma unroll
            for (int i = 0; i < S::FI; ++i) acc[i][j] = col[i];
          }
          uint16_t* out = dh + static_cast<int64_t>(n0) * a.dim + d0;
          hl_store_rows<S>(acc, area, a.dim - d0,
                           [&](int q) { return q < rows ? out + static_cast<int64_t>(q) * a.dim : nullptr; });
        } else {
          const int d = d0 + 4 * (lane >> 5);
#pragma unroll
          for (int j = 0; j < S::FJ; ++j) {
            const int n = 32 * j + (lane & 31);
            if (n >= rows) continue;
            float* out = sum + (static_cast<int64_t>(z) * a.rows + n0 + n) * a.dim + d;
#pragma unroll
            for (int i = 0; i < S::FI; ++i)
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                if (d + 32 * i + 8 * q >= a.dim) continue;   // (dim is a multiple of 64)
                float4* o = reinterpret_cast<float4*>(out + 32 * i + 8 * q);
                float4 v = make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
                if (!first) {
                  const float4 b = *o;
                  v = make_float4(v.x + b.x, v.y + b.y, v.z + b.z, v.w + b.w);
                }
                *o = v;
              }
          }
        }
      });
}

// dhidden = the parts' sum and what rounding took of g at the row's token times the
// token's weights, rounded once; four values per thread (of dim / 4 a row)
__global__ __launch_bounds__(256) void k_head_dh_join(const HlArgs a, const HlFix* fix, const float4* part, uint2* out,
                                                      int splits) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, n4 = static_cast<int64_t>(a.rows) * (a.dim / 4);
  if (i >= n4) return;
  const int64_t n = i / (a.dim / 4);
  const HlFix f = fix[n];
  float4 v = part[i];
  for (int z = 1; z < splits; ++z) {
    const float4 b = part[z * n4 + i];
    v = make_float4(v.x + b.x, v.y + b.y, v.z + b.z, v.w + b.w);
  }
  if (f.r != 0.0f) {
    const uint2 w = *reinterpret_cast<const uint2*>(a.weight + static_cast<int64_t>(f.v) * a.dim + 4 * (i - n * (a.dim / 4)));
    v = make_float4(fmaf(f.r, BF16::to_f32(w.x & 0xFFFFu), v.x), fmaf(f.r, BF16::to_f32(w.x >> 16), v.y),
                    fmaf(f.r, BF16::to_f32(w.y & 0xFFFFu), v.z), fmaf(f.r, BF16::to_f32(w.y >> 16), v.w));
  }
  out[i] = make_uint2(BF16::from_f32(v.x) | (BF16::from_f32(v.y) << 16), BF16::from_f32(v.z) | (BF16::from_f32(v.w) << 16));
}

// ---------------------------------------------------------------- launches
namespace {

int cdiv(int64_t a, int64_t b) { return static_cast<int>((a + b - 1) / b); }
size_t al(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }

// j-tile of the logits' products: the rows' own size up to 128, so that a few rows
// do not pay for 256, and smaller while that leaves half the CUs or more idle
// (calls, 4096x4096x1000: 93 us with 64 tiles of 256, 54 with 256 of 64; 255x768x32000
// 32 and, 250 of 128, 24).
constexpr int HL_CUS = 256;
int hl_few(int64_t ni, int64_t nj, int bj = 256) {
  while (bj > 64 && 2 * ni * cdiv(nj, bj) <= HL_CUS) bj /= 2;
  return bj;
}
int hl_bj(int64_t rows, int64_t vocab) { return hl_few(cdiv(vocab, HL_I), rows, rows <= 64 ? 64 : rows <= 128 ? 128 : 256); }
int hl_parts(int64_t vocab) { return cdiv(vocab, HL_I); }

// Vocabulary rows of a backward chunk: g's bytes stay within HL_G_BYTES, but a
// chunk has at least HL_CHUNK rows, so that the products of many rows have k
// enough beside the sums they read and write.
constexpr int64_t HL_G_BYTES = 512ll << 20, HL_CHUNK = 16384;
int hl_chunk(int64_t rows, int64_t vocab) {
  const int64_t fit = std::max<int64_t>(HL_CHUNK, HL_G_BYTES / (2 * std::max<int64_t>(rows, 1)) / HL_I * HL_I);
  const int64_t all = (vocab + HL_K - 1) / HL_K * HL_K;
  if (all <= fit) return static_cast<int>(all);
  // chunks of about one size
  const int64_t n = (all + fit - 1) / fit;
  return static_cast<int>(std::min(all, ((all + n - 1) / n + HL_I - 1) / HL_I * HL_I));
}
// j-tile of dhidden's product: few tiles mean many parts, 4 bytes a value each
// written and read, so smaller ones where they are fewer than 32 (255x1024x50257:
// 4 tiles of 256 in 61 parts 64 us with their sum, 16 of 64 in 16 parts 47 us).
int hl_dh_bj(int64_t rows, int64_t dim) {
  const int64_t nd = cdiv(dim, HL_I);
  return rows > 128 && cdiv(rows, 256) * nd >= 32 ? 256 : rows > 64 && cdiv(rows, 128) * nd >= 32 ? 128 : 64;
}
// Ranges of a chunk's vocabulary rows that dhidden's product is split into: as
// many as give every CU a tile, of 8 stages or more; each but the last `per`
// stages, none empty.
struct Split {
  int nz, per;
};
Split hl_split(int64_t rows, int64_t dim, int64_t chunk) {
  const int64_t tiles = std::max<int64_t>(1, static_cast<int64_t>(cdiv(rows, hl_dh_bj(rows, dim))) * cdiv(dim, HL_I));
  const int64_t st = chunk / HL_K, want = std::max<int64_t>(1, std::min(HL_CUS / tiles, st / 8));
  const int per = cdiv(st, want);
  return {cdiv(st, per), per};
}

HlArgs hl_args(const void* hidden, const void* weight, int64_t ld, int64_t rows, int64_t dim, int64_t vocab,
               const int64_t* tokens, int64_t ignore_index) {
  return {static_cast<const uint16_t*>(hidden), static_cast<const uint16_t*>(weight), ld, static_cast<int>(rows),
          static_cast<int>(dim), static_cast<int>(vocab), tokens, ignore_index};
}

// f(bj) as a constant
template <class F>
void hl_by(int bj, F&& f) {
  if (bj == 64) f(std::integral_constant<int, 64>{});
  else if (bj == 128) f(std::integral_constant<int, 128>{});
  else f(std::integral_constant<int, 256>{});
}

// Launch of a persistent kernel over the tiles: a work-group per CU at most (each
// fills a CU's LDS).  Above 64 KiB a kernel's dynamic LDS has to be asked for.
template <class S, class K, class... A>
hipError_t hl_launch(K k, const Tiles& ts, hipStream_t s, A... args) {
  const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, S::LDS);
  if (e != hipSuccess) return e;
  const int64_t n = static_cast<int64_t>(ts.ni) * ts.nj * ts.nz;
  hipLaunchKernelGGL(k, dim3(static_cast<unsigned>(std::min<int64_t>(n, HL_CUS))), dim3(HL_NT), S::LDS, s, args...);
  return hipGetLastError();
}

}  // namespace

size_t head_workspace_bytes(int64_t rows, int64_t vocab) {
  const size_t R = static_cast<size_t>(rows);
  return al(16 * R * static_cast<size_t>(hl_parts(vocab))) + al(4 * R);
}

size_t head_grad_workspace_bytes(int64_t rows, int64_t dim, int64_t vocab, bool dhidden) {
  const int64_t cn = hl_chunk(rows, vocab);
  const size_t R = static_cast<size_t>(rows);
  return al(2 * R * static_cast<size_t>(cn)) + al(sizeof(HlFix) * R) + al(sizeof(HlFix) * static_cast<size_t>(cn)) +
         (dhidden ? al(4 * R * static_cast<size_t>(dim) * static_cast<size_t>(hl_split(rows, dim, cn).nz)) : 0);
}

hipError_t launch_head(const fl_head_args& a, hipStream_t s) {
  const HlArgs h = hl_args(a.hidden, a.weight, a.ld_hidden, a.rows, a.dim, a.vocab, a.tokens, a.ignore_index);
  float4* part = static_cast<float4*>(a.workspace);
  const int parts = hl_parts(a.vocab);
  float* xt = reinterpret_cast<float*>(static_cast<char*>(a.workspace) + al(16 * static_cast<size_t>(a.rows) * parts));
  hipError_t e = hipSuccess;
  hl_by(hl_bj(a.rows, a.vocab), [&](auto bj) {
    constexpr int BJ = decltype(bj)::value;
    const Tiles ts = {cdiv(a.vocab, HL_I), cdiv(a.rows, BJ), 1};
    e = hl_launch<Shape<BJ>>(k_head_stats<BJ>, ts, s, h, part, xt, ts);
  });
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(k_head_join, dim3(cdiv(a.rows, HJ_R)), dim3(HJ_R * HJ_P), 0, s, a, part, xt, parts);
  return hipGetLastError();
}

hipError_t launch_head_grad(const fl_head_grad_args& a, hipStream_t s) {
  const HlArgs h = hl_args(a.hidden, a.weight, a.ld_hidden, a.rows, a.dim, a.vocab, a.tokens, a.ignore_index);
  const HlGrad gr = {a.saved, a.grad_logprob, a.grad_entropy, a.grad_lse};
  const int chunk = hl_chunk(a.rows, a.vocab), nd = cdiv(a.dim, HL_I);
  uint16_t* g = static_cast<uint16_t*>(a.workspace);
  char* behind = static_cast<char*>(a.workspace) + al(2 * static_cast<size_t>(a.rows) * chunk);
  HlFix* fix = reinterpret_cast<HlFix*>(behind);
  HlFix* list = reinterpret_cast<HlFix*>(behind + al(sizeof(HlFix) * static_cast<size_t>(a.rows)));
  float* sum = reinterpret_cast<float*>(reinterpret_cast<char*>(list) + al(sizeof(HlFix) * static_cast<size_t>(chunk)));
  uint16_t* dh = static_cast<uint16_t*>(a.out_dhidden);
  const bool direct = chunk >= a.vocab && hl_split(a.rows, a.dim, chunk).nz == 1;
  hipError_t e = hipSuccess;
  for (int c0 = 0; c0 < a.vocab && e == hipSuccess; c0 += chunk) {
    const int cn = static_cast<int>(std::min<int64_t>(chunk, (a.vocab - c0 + HL_K - 1) / HL_K * HL_K));
    const int nc = cdiv(cn, HL_I);
    hl_by(hl_bj(a.rows, cn), [&](auto bj) {
      constexpr int BJ = decltype(bj)::value;
      using S = Shape<BJ>;
      const Tiles tg = {nc, cdiv(a.rows, BJ), 1};
      e = hl_launch<S>(k_head_g<BJ>, tg, s, h, gr, g, c0, cn, tg);
    });
    if (e != hipSuccess) break;
    hipLaunchKernelGGL(k_head_fix, dim3(cdiv(cn / HL_LIST, 256 / WAVE)), dim3(256), 0, s, h, gr, g, fix, list, c0, cn);
    e = hipGetLastError();
    if (e == hipSuccess && dh != nullptr)
      hl_by(hl_dh_bj(a.rows, a.dim), [&](auto bj) {
        constexpr int BJ = decltype(bj)::value;
        using S = Shape<BJ>;
        // (ranges of the first chunk's size, so that a later one has no more of them:
        // every part that it adds to was written)
        const Split sp = hl_split(a.rows, a.dim, chunk);
        const Tiles td = {nd, cdiv(a.rows, BJ), cdiv(cn / HL_K, sp.per)};
        if (direct) e = hl_launch<S>(k_head_dh<BJ, true>, td, s, h, g, fix, sum, dh, c0, cn, td, sp.per, 1);
        else e = hl_launch<S>(k_head_dh<BJ, false>, td, s, h, g, fix, sum, dh, c0, cn, td, sp.per, c0 == 0 ? 1 : 0);
      });
    if (e == hipSuccess && a.out_dweight) hl_by(hl_few(nd, cn), [&](auto bj) {
      constexpr int BJ = decltype(bj)::value;
      const Tiles tw = {nd, cdiv(cn, BJ), 1};
      e = hl_launch<Shape<BJ>>(k_head_dw<BJ>, tw, s, h, g, list, static_cast<uint16_t*>(a.out_dweight), c0, cn, tw);
    });
  }
  if (e != hipSuccess) return e;
  if (dh != nullptr && !direct) {
    const int64_t n4 = a.rows * a.dim / 4;
    hipLaunchKernelGGL(k_head_dh_join, dim3(static_cast<unsigned>(cdiv(n4, 256))), dim3(256), 0, s, h, fix,
                       reinterpret_cast<const float4*>(sum), reinterpret_cast<uint2*>(dh),
                       hl_split(a.rows, a.dim, chunk).nz);
  }
  return hipGetLastError();
}

}  // namespace fl

// Scores of given tokens from logits rows, and their gradient.
//
//   lse      = log sum_i exp x_i
//   logprob  = x_t - lse                       (the row's token t)
//   entropy  = lse - sum_i p_i x_i             (p_i = exp(x_i - lse); a masked
//                                               value, -inf, adds nothing)
//   rank     = #{i : x_i > x_t}
//   top k    : the k largest values, ties by the lowest index, each x - lse
//
//   d x_i    = a (1[i = t] - p_i) - b p_i (log p_i + entropy) + c p_i
//              for upstream gradients a, b, c of logprob, entropy and lse.
//
// Forward: a row is cut into slices of SC_SLICE values, one work-group each,
// whatever the number of rows: a decode step's few rows spread over the CUs,
// and a row's results are a function of the row alone.  A thread holds its 64
// values of the slice in registers, so every step (maximum, sums, rank count,
// the largest values) reads HBM once; the join of a row's slices is a second
// kernel (none for a row of one slice).  bf16 4096x128256 (1.05 GB), whole calls:
// 170 us for the log-probability (6.2 TB/s), 179 with the entropy, 201 with 5
// alternatives too, 203 with all that and the rank: bound by HBM, and past that by
// the vector instructions and the meetings of the search.  12x128256 with 20
// alternatives and the rank: 12.0 us + 4.7 us for the join, a chain of a load, eight
// barriers and the list; 1x50257: 7.6 + 3.5 us.  A slice costs the instructions of
// 16384 values whatever it holds: 4096 bf16 rows of 512, 4099, 8192 and 16384 take
// 26, 28, 26 and 22 us with the entropy, for 4 to 134 MB.  (Fewer registers for 7
// or 8 waves per SIMD spill: 238 us with the entropy; slices streamed by one
// work-group per row: 289 us with 5 alternatives.)
#include <type_traits>

#include "fl_device.h"
#include "fl_kernels.h"

namespace fl {

namespace {

constexpr int SC_NT = 256;                    // threads of a slice's work-group
constexpr int SC_NW = SC_NT / WAVE;
constexpr int SC_VALS = 64;                   // values per thread
constexpr int SC_SLICE = SC_NT * SC_VALS;     // 16384
constexpr int SC_MAX_SLICES = FL_MAX_VOCAB_F32 / SC_SLICE;
// Candidates for a slice's largest values: those at or above the k-th largest
// of the threads' maxima, at most a few more than k unless the large values lie
// side by side (a vocabulary sorted by frequency: 8 per thread, 505 for k = 64)
// or are equal (then the exact path below).
constexpr int SC_CAP = 1024;
constexpr int SC_MAX_TOP = FL_SCORE_MAX_TOPK;
static_assert(SC_MAX_SLICES * SC_MAX_TOP <= SC_CAP, "the join holds every slice's list");
static_assert(SC_MAX_TOP <= SC_NT, "one maximum per thread bounds the k-th largest");

constexpr float SC_LOG2E = 1.44269504088896340736f;
constexpr double SC_INV_LOG2E = 1.0 / static_cast<double>(SC_LOG2E);  // (of the float: exact for base-2 differences over it)

// A slice's part of its row: sums of e = exp(x - ref) over the slice.
struct ScPart {
  double ref;   // -inf: every value is -inf
  double s;     // sum e
  double u;     // sum e (x - ref)
  float xt;     // the token's logit (the same in every slice)
  int32_t rank; // values above it
};

struct ScWs {
  ScPart* part;     // [rows, S]
  uint64_t* list;   // [rows, S, top_k]: (key << 32) | ~index, descending, 0 past the slice's values
  int S;
};

// Ascending key of a value with -0 as +0, and a candidate's 64 bits: greater
// for a larger value and, of equal values, for a lower index.
__device__ __forceinline__ uint64_t sc_key(float x, uint32_t i) {
  return (static_cast<uint64_t>(f32_key(x + 0.0f)) << 32) | static_cast<uint32_t>(~i);
}

// What a row's outputs are made of.
struct ScRow {
  double ref, logs;   // lse = ref + logs (apart: beside a reference of -3e38 the logarithm would be lost)
  bool ok;            // the row has a distribution (no NaN, no +inf, not all -inf)
  __device__ __forceinline__ float logprob(float x) const {
    return ok ? static_cast<float>((static_cast<double>(x) - ref) - logs) : __builtin_nanf("");
  }
};

// The outputs that need no list, by one thread.
__device__ __forceinline__ ScRow sc_finish(const fl_score_args& a, int64_t r, double ref, double s, double u, float xt,
                                           int rank) {
  const float nan = __builtin_nanf("");
  const double logs = log(s);
  const ScRow out = {ref, logs, s > 0.0 && s < static_cast<double>(__builtin_inff())};
  const float ent = out.ok ? static_cast<float>(logs - u / s) : nan;
  if (a.out_entropy) a.out_entropy[r] = ent;
  if (a.out_lse) a.out_lse[r] = out.ok ? static_cast<float>(ref + logs) : s == 0.0 ? -__builtin_inff() : nan;
  if (a.tokens) {
    const int64_t t = a.tokens[r];
    const bool ignored = t == a.ignore_index, bad = t < 0 || t >= a.vocab;
    if (a.out_logprob) a.out_logprob[r] = ignored ? -0.0f : bad ? nan : out.logprob(xt);
    if (a.out_rank) a.out_rank[r] = ignored || bad || !out.ok ? -1 : rank;
  }
  if (a.out_saved) {
    // lse in two floats: of logits in the thousands, one float's rounding
    // would be 1e-4 of every probability in the gradient
    float* sv = a.out_saved + 4 * r;
    const float hi = static_cast<float>(ref);
    sv[0] = out.ok ? hi : nan;
    sv[1] = out.ok ? static_cast<float>((ref - static_cast<double>(hi)) + logs) : nan;
    sv[2] = a.out_entropy ? ent : nan;   // (a gradient of it without it is NaN, not another number)
    sv[3] = 0.0f;
  }
  return out;
}

// Entry q of the row's list (key 0: past the row's values; never for k <= V).
__device__ __forceinline__ void sc_emit(const fl_score_args& a, int64_t r, int q, uint64_t key, const ScRow& row) {
  const int64_t o = r * a.top_k + q;
  const float x = f32_of_key(static_cast<uint32_t>(key >> 32));
  if (a.out_top_ids) a.out_top_ids[o] = row.ok ? static_cast<int64_t>(~static_cast<uint32_t>(key)) : -1;
  if (a.out_top_logprobs) a.out_top_logprobs[o] = row.logprob(x);
}

// n candidates to their places by counting the greater ones (they are
// distinct), eight a turn; put(place, key) for places below k.  Called by the
// whole work-group of NT threads, cand written and met on.
template <int NT, class P>
__device__ __forceinline__ void sc_place(uint64_t* cand, int n, int k, P&& put) {
  const int n8 = (n + 7) & ~7;
  if (static_cast<int>(threadIdx.x) < n8 - n) cand[n + threadIdx.x] = 0u;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += NT) {
    const uint64_t mine = cand[i];
    int above = 0;
    for (int j = 0; j < n8; j += 8) {
      const ulonglong2* c = reinterpret_cast<const ulonglong2*>(cand + j);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const ulonglong2 v = c[e];
        above += (v.x > mine ? 1 : 0) + (v.y > mine ? 1 : 0);
      }
    }
    if (above < k) put(above, mine);
  }
}

}  // namespace

// One slice of a row.  ENT: the entropy's sum; RANK: count the values above
// the token's.
template <class D, bool ENT, bool RANK>
__global__ __launch_bounds__(SC_NT) void k_score_slice(const fl_score_args a, const ScWs ws) {
  using C = RowChunk<D>;
  constexpr int N = C::N, NCH = SC_VALS / N;
  constexpr size_t ESZ = D::id == FL_DTYPE_F32 ? 4 : 2;
  // low bits of a value's key that its type leaves at 0 (1, for a negative value)
  constexpr int LOW = D::id == FL_DTYPE_F32 ? 0 : D::id == FL_DTYPE_BF16 ? 16 : 13;
  __shared__ __attribute__((aligned(16))) uint64_t cand[SC_CAP];
  __shared__ uint32_t tkey[SC_NT];
  __shared__ float red[SC_NW], red_s[SC_NW], red_u[SC_NW];
  __shared__ uint32_t red_c[SC_NW];
  __shared__ uint32_t s_key, s_n;
  __shared__ ScRow s_row;
  const int tid = threadIdx.x, lane = tid & (WAVE - 1), w = tid / WAVE;
  const int S = ws.S, V = static_cast<int>(a.vocab), K = static_cast<int>(a.top_k);
  const int64_t r = blockIdx.x / static_cast<unsigned>(S);
  const int sl = static_cast<int>(blockIdx.x - static_cast<unsigned>(r) * static_cast<unsigned>(S));
  const int base = sl * SC_SLICE, nval = min(SC_SLICE, V - base);
  const char* row = static_cast<const char*>(a.logits) + r * a.ld * static_cast<int64_t>(ESZ);
  const __amdgpu_buffer_rsrc_t rs = row_rsrc(row + base * ESZ, static_cast<uint32_t>(nval * ESZ));

  uint4 q[NCH];
#pragma unroll
  for (int k = 0; k < NCH; ++k) q[k] = buf_load16_once(rs, 16u * static_cast<uint32_t>(tid + k * SC_NT), 0u);
  // the token's logit (+inf, which nothing is above, without a token)
  float xt = __builtin_inff();
  if (a.tokens) {
    const int64_t t = a.tokens[r];
    if (t >= 0 && t < V && t != a.ignore_index)
      xt = C::elem(row_rsrc(row, static_cast<uint32_t>(V * ESZ)), static_cast<int>(t));
  }
  // Past the slice's values a chunk takes the pattern `fill`; the last value of
  // an odd 16-bit row by itself (the range check goes by dwords).
  const bool part = nval < SC_SLICE;
  constexpr uint32_t NINF = D::id == FL_DTYPE_F32 ? 0xFF800000u : D::id == FL_DTYPE_BF16 ? 0xFF80u : 0xFC00u;
  uint32_t last = 0;
  if (D::id != FL_DTYPE_F32 && part && (nval & 1))
    last = static_cast<uint16_t>(__builtin_amdgcn_raw_buffer_load_b16(rs, 2 * (nval - 1), 0, 0));
  auto pad = [&](uint4 v, int k, uint32_t fill) {
    uint32_t wd[4] = {v.x, v.y, v.z, v.w};
    const int f = N * (tid + k * SC_NT);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (D::id == FL_DTYPE_F32) {
        wd[j] = f + j >= nval ? fill : wd[j];
      } else {
        wd[j] = f + 2 * j + 1 == nval ? (last | (fill << 16)) : wd[j];
        wd[j] = f + 2 * j >= nval ? (fill | (fill << 16)) : wd[j];
      }
    }
    return make_uint4(wd[0], wd[1], wd[2], wd[3]);
  };
  auto pad_all = [&](uint32_t fill) {
#pragma unroll
    for (int k = 0; k < NCH; ++k) q[k] = pad(q[k], k, fill);
  };
  if (part) pad_all(NINF);
  // (chunk k from memory again, for the rare paths: rolled loops, small code)
  auto fetch = [&](float (&x)[N], int k) {
    C::unpack(pad(buf_load16(rs, 16u * static_cast<uint32_t>(tid + k * SC_NT), 0u), k, NINF), x);
  };
  // (the steps below unpack the values again each, rather than hold both forms)
  auto fence = [&]() {
#pragma unroll
    for (int k = 0; k < NCH; ++k) asm volatile("" : "+v"(q[k].x), "+v"(q[k].y), "+v"(q[k].z), "+v"(q[k].w));
  };

  // Maxima: chunk, thread, slice.  Of the values' bits as signed integers, two
  // 16-bit values at a time: right as soon as one value is not negative, else
  // it finds the one farthest from 0 (a value of the chunk still).  Only where
  // that matters are they taken again as floats: a slice of negative values,
  // fewer than K threads with one that is not, or a K-th value of 0 (-0, which
  // is equal to it, is the least of the integers).
  float cm[NCH];
  int tb = -0x7FFFFFFF - 1;
#pragma unroll
  for (int k = 0; k < NCH; ++k) {
    int c;
    if constexpr (D::id == FL_DTYPE_F32) {
      c = max(max(static_cast<int>(q[k].x), static_cast<int>(q[k].y)), max(static_cast<int>(q[k].z), static_cast<int>(q[k].w)));
      cm[k] = __uint_as_float(static_cast<uint32_t>(c));
    } else {
      typedef short short2v __attribute__((ext_vector_type(2)));
      const short2v m2 = __builtin_elementwise_max(
          __builtin_elementwise_max(__builtin_bit_cast(short2v, q[k].x), __builtin_bit_cast(short2v, q[k].y)),
          __builtin_elementwise_max(__builtin_bit_cast(short2v, q[k].z), __builtin_bit_cast(short2v, q[k].w)));
      const uint32_t b = __builtin_bit_cast(uint32_t, m2);
      c = max(static_cast<int>(b << 16), static_cast<int>(b & 0xFFFF0000u));
      cm[k] = D::to_f32(static_cast<uint32_t>(c) >> 16);
    }
    tb = max(tb, c);
  }
  auto as_float = [](int b) {
    if constexpr (D::id == FL_DTYPE_F32) return __uint_as_float(static_cast<uint32_t>(b));
    else return D::to_f32(static_cast<uint32_t>(b) >> 16);
  };
  auto exact_maxima = [&]() {   // (of the thread)
    fence();
    float t = -__builtin_inff();
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      float x[N];
      C::unpack(q[k], x);
      float c = x[0];
#pragma unroll
      for (int e = 1; e < N; ++e) c = fmaxf(c, x[e]);
      cm[k] = c;
      t = fmaxf(t, c);
    }
    fence();
    return t;
  };
  if (tid == 0) s_n = 0u;
  tkey[tid] = f32_key(as_float(tb) + 0.0f);
  const int wb = wave_reduce(tb, OpMax());
  if (lane == 0) red[w] = as_float(wb);
  __syncthreads();
  float m = red[0];
#pragma unroll
  for (int i = 1; i < SC_NW; ++i) m = fmaxf(m, red[i]);
  // (a wave of negative values alone left a lower one: no matter beside a
  // wave that has one which is not)
  bool exact = !(m >= 0.0f);
  if (exact) {   // (for the whole work-group)
    const float t = exact_maxima();
    const float wm = wave_reduce(t, OpMax());
    __syncthreads();
    tkey[tid] = f32_key(t + 0.0f);
    if (lane == 0) red[w] = wm;
    __syncthreads();
    m = red[0];
#pragma unroll
    for (int i = 1; i < SC_NW; ++i) m = fmaxf(m, red[i]);
  }
  m = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(m)));
  fence();

  // Sums relative to the slice's maximum, exponents in base 2.  d2 =
  // fma(x, log2(e), -mb) has one rounding; it is relative to mb / log2(e),
  // which is what `ref` says.  From |mb| = 2^31 on (a mask of the type's lowest
  // value) that would not do, and d2 = (x - m) log2(e).  A term of the entropy
  // is e d2, which for a -inf value, or one the exponent leaves the float range
  // for, is 0 * -inf: a wave that finds a NaN takes its sums again with
  // e max(d2, -200), 0 there.
  const float mb = m == -__builtin_inff() ? 0.0f : m * SC_LOG2E;
  // Past the slice's values a finite fill far below m, so that the fast sums of
  // a row's last slice have no NaN (float16 has none below a mask of its lowest).
  constexpr uint32_t FILL = D::id == FL_DTYPE_F32 ? 0xF149F2CAu : D::id == FL_DTYPE_BF16 ? 0xF149u : 0xFBFFu;   // -1e30; -65504
  const bool plain = __builtin_fabsf(mb) < 0x1p31f && !(D::id == FL_DTYPE_F16 && part && m < -60000.0f);
  if (part && plain) pad_all(FILL);
  const double ref = m == -__builtin_inff() ? static_cast<double>(m)
                     : plain                ? static_cast<double>(mb) * SC_INV_LOG2E
                                            : static_cast<double>(m);   // (as the sums below take it)
  float fs[2] = {0.0f, 0.0f}, fu[2] = {0.0f, 0.0f};
  uint32_t above = 0;
  if (plain) {
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      float x[N];
      C::unpack(q[k], x);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float d2 = fmaf(x[e], SC_LOG2E, -mb);
        const float ex = __builtin_amdgcn_exp2f(d2);
        fs[e & 1] += ex;
        if (ENT) fu[e & 1] = fmaf(ex, d2, fu[e & 1]);
        if (RANK) above += static_cast<uint32_t>(__popcll(__ballot(x[e] > xt)));
      }
      __builtin_amdgcn_sched_barrier(0);   // (one chunk's comparisons live at a time)
    }
    // (a token below the fill, a masked one, has counted the wave's places past
    // the slice; summing its slice again instead, with -inf there: 318 us for
    // bf16 4096x128256 with every token masked, 190 of other tokens)
    if (RANK && part && xt < as_float(static_cast<int>(D::id == FL_DTYPE_F32 ? FILL : FILL << 16))) {
#pragma unroll 1
      for (int k = 0; k < NCH; ++k)
        above -= static_cast<uint32_t>(min(max(N * (tid - lane + WAVE + k * SC_NT) - nval, 0), N * WAVE));
    }
  }
  const float u0 = fu[0] + fu[1];
  if (!plain || (ENT && __any(u0 != u0))) {   // (for the whole wave)
    const float ref0 = m == -__builtin_inff() ? 0.0f : m;
    fs[0] = fs[1] = fu[0] = fu[1] = 0.0f;
    above = 0;
#pragma unroll 1
    for (int k = 0; k < NCH; ++k) {
      float x[N];
      fetch(x, k);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float d2 = plain ? fmaf(x[e], SC_LOG2E, -mb) : (x[e] - ref0) * SC_LOG2E;
        const float ex = __builtin_amdgcn_exp2f(d2);
        fs[e & 1] += ex;
        if (ENT) fu[e & 1] = fmaf(ex, fmaxf(d2, -200.0f), fu[e & 1]);
        if (RANK) above += static_cast<uint32_t>(__popcll(__ballot(x[e] > xt)));
      }
    }
  }
  const float ws_s = wave_reduce(fs[0] + fs[1], OpAdd());
  const float ws_u = ENT ? wave_reduce(fu[0] + fu[1], OpAdd()) : 0.0f;
  if (lane == 0) {
    red_s[w] = ws_s;
    red_u[w] = ws_u;
    red_c[w] = above;
  }
  auto bound = [&]() {
    // the K-th largest of the threads' maxima: K values of the slice reach it
    // (past the slice's values the maxima are -inf)
    uint32_t kk[SC_NW];
#pragma unroll
    for (int i = 0; i < SC_NW; ++i) kk[i] = tkey[lane + WAVE * i];
    uint32_t T = 0;
#pragma unroll 1
    for (int b = 31; b >= LOW; --b) {
      const uint32_t t = T | (1u << b);
      int c = 0;
#pragma unroll
      for (int i = 0; i < SC_NW; ++i) c += __popcll(__ballot(kk[i] >= t));
      if (c >= K) T = t;
    }
    if (LOW > 0 && !(T & 0x80000000u)) T |= (1u << LOW) - 1u;
    if (lane == 0) s_key = T;
  };
  if (K > 0 && w == 0) bound();
  __syncthreads();
  if (tid == 0) {
    double s = 0.0, u = 0.0;
    int c = 0;
#pragma unroll
    for (int i = 0; i < SC_NW; ++i) {
      s += static_cast<double>(red_s[i]);
      u += static_cast<double>(red_u[i]);
      c += static_cast<int>(red_c[i]);
    }
    u *= SC_INV_LOG2E;
    if (S == 1) s_row = sc_finish(a, r, ref, s, u, xt, c);
    else ws.part[r * S + sl] = ScPart{ref, s, u, xt, c};
  }
  if (K == 0) return;

  // ---- the slice's K largest values
  fence();
  if (!exact && s_key <= 0x80000000u) {   // (a negative bound, or 0, by integer maxima)
    __syncthreads();
    if (part) pad_all(NINF);
    tkey[tid] = f32_key(exact_maxima() + 0.0f);
    __syncthreads();
    if (w == 0) bound();
    __syncthreads();
  }
  float tf = f32_of_key(s_key);
  auto append = [&](const float (&x)[N], int k, auto&& in) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int i = N * (tid + k * SC_NT) + e;
      if (in(x[e]) && i < nval) {
        const uint32_t slot = atomicAdd(&s_n, 1u);
        if (slot < SC_CAP) cand[slot] = sc_key(x[e], static_cast<uint32_t>(base + i));
      }
    }
  };
#pragma unroll
  for (int k = 0; k < NCH; ++k) {
    if (__any(cm[k] >= tf)) {
      float x[N];
      C::unpack(q[k], x);
      append(x, k, [&](float v) { return v >= tf; });
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  __syncthreads();
  int n = static_cast<int>(s_n);
  if (n > SC_CAP) {
    // Many values at or above the bound.  The exact K-th largest value: the
    // bound itself if fewer than K values are above it (many equal values: a
    // mask), else by bisection over the keys.  Then the values above it, and of
    // those equal to it the first ones.
    auto count = [&](auto&& in) {   // (over the slice; the same for every thread)
      uint32_t c = 0;
#pragma unroll 1
      for (int k = 0; k < NCH; ++k) {
        float x[N];
        fetch(x, k);
#pragma unroll
        for (int e = 0; e < N; ++e) c += (in(x[e]) && N * (tid + k * SC_NT) + e < nval) ? 1u : 0u;
      }
      c = wave_reduce(c, OpAdd());
      __syncthreads();
      if (lane == 0) red_c[w] = c;
      __syncthreads();
      uint32_t t = 0;
#pragma unroll
      for (int i = 0; i < SC_NW; ++i) t += red_c[i];
      return static_cast<int>(t);
    };
    if (count([&](float x) { return x > tf; }) >= K) {
      // count(key >= lo) >= K > count(key >= hi), hi past +inf's key
      uint32_t lo = f32_key(tf), hi = 0xFF800001u;
#pragma unroll 1
      while (hi - lo > 1u) {
        const uint32_t mid = lo + (hi - lo) / 2u;
        const float mf = f32_of_key(mid);
        if (count([&](float x) { return x >= mf; }) >= K) lo = mid;
        else hi = mid;
      }
      tf = f32_of_key(lo);
    }
    if (tid == 0) s_n = 0u;
    __syncthreads();
#pragma unroll 1
    for (int k = 0; k < NCH; ++k) {
      float x[N];
      fetch(x, k);
      append(x, k, [&](float v) { return v > tf; });
    }
    __syncthreads();
    n = min(static_cast<int>(s_n), SC_CAP);
    // equal values in index order: chunk by chunk, thread by thread
#pragma unroll 1
    for (int k = 0; k < NCH && n < K; ++k) {   // (n is the same for every thread)
      float x[N];
      fetch(x, k);
      uint32_t mine = 0;
#pragma unroll
      for (int e = 0; e < N; ++e) mine += (x[e] == tf && N * (tid + k * SC_NT) + e < nval) ? 1u : 0u;
      const uint32_t incl = wave_incl_scan(mine);
      if (lane == WAVE - 1) red_c[w] = incl;
      __syncthreads();
      uint32_t before = 0, total = 0;
#pragma unroll
      for (int i = 0; i < SC_NW; ++i) {
        before += i < w ? red_c[i] : 0u;
        total += red_c[i];
      }
      int at = n + static_cast<int>(before + incl - mine);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int i = N * (tid + k * SC_NT) + e;
        if (x[e] == tf && i < nval) {
          if (at < K) cand[at] = sc_key(x[e], static_cast<uint32_t>(base + i));
          ++at;
        }
      }
      n = min(K, n + static_cast<int>(total));
      __syncthreads();
    }
  }
  if (S == 1) {
    const ScRow rw = s_row;
    sc_place<SC_NT>(cand, n, K, [&](int p, uint64_t key) { sc_emit(a, r, p, key, rw); });
    // (fewer than K values found: NaN values, whose row has no distribution)
    for (int p = n + tid; p < K; p += SC_NT) sc_emit(a, r, p, 0u, rw);
  } else {
    uint64_t* out = ws.list + (r * S + sl) * static_cast<int64_t>(K);
    sc_place<SC_NT>(cand, n, K, [&](int p, uint64_t key) { out[p] = key; });
    for (int p = n + tid; p < K; p += SC_NT) out[p] = 0u;
  }
}

// A row's slices joined; one work-group per row: of one wave where its lists hold
// no more than an entry a lane (bf16 4096x128256, K = 5: 8.8 us, 13.5 of four
// waves), else of SC_NT threads (12x128256, K = 20, 160 entries: 4.9 us, 6.3 of one
// wave).
template <int NT>
__global__ __launch_bounds__(NT) void k_score_join(const fl_score_args a, const ScWs ws) {
  __shared__ __attribute__((aligned(16))) uint64_t cand[NT == SC_NT ? SC_CAP : NT];
  __shared__ ScRow s_row;
  __shared__ uint32_t s_n;
  const int tid = threadIdx.x;
  const int S = ws.S, K = static_cast<int>(a.top_k);
  const int64_t r = blockIdx.x;
  const uint64_t* list = ws.list + r * S * K;
  if (tid == 0) s_n = 0u;
  // Bounds that the row's K-th value reaches: the largest of the lists' K-th
  // entries, and the smallest over the slices of n values of their ceil(K n /
  // V)-th (together they hold K values).  The second is the close one: with the
  // first alone a row of 151936 had 550 candidates for K = 64, 14 us for 37 rows.
  // (The loads go beside the statistics.)
  const int sl = tid & (WAVE - 1), V = static_cast<int>(a.vocab);
  const bool has = K > 0 && sl < S;
  const int nth = static_cast<int>((static_cast<int64_t>(K) * min(SC_SLICE, V - sl * SC_SLICE) + V - 1) / V);
  const uint64_t kth = has ? list[sl * K + K - 1] : 0u, share = has ? list[sl * K + nth - 1] : ~0ull;
  constexpr int PER = NT == SC_NT ? SC_CAP / SC_NT : 1;   // (the host's choice of NT)
  uint64_t mine[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) mine[i] = tid + i * NT < S * K ? list[tid + i * NT] : 0u;
  if (tid < WAVE) {
    constexpr int G = SC_MAX_SLICES;   // lanes of the fixed tree
    static_assert(G <= WAVE && (G & (G - 1)) == 0, "one lane per slice");
    const double ninf = -static_cast<double>(__builtin_inff());
    ScPart p = {ninf, 0.0, 0.0, 0.0f, 0};
    if (tid < S) p = ws.part[r * S + tid];
    double R = wave_reduce<double, OpMax, G>(p.ref, OpMax());
    const double d = p.ref - R;
    const bool on = p.ref != ninf;
    const double f = on ? exp(d) : 0.0;
    // (a slice of -inf alone adds nothing; a NaN sum, of any slice, stays)
    const double s = wave_reduce<double, OpAdd, G>(on ? p.s * f : p.s, OpAdd());
    const double u = wave_reduce<double, OpAdd, G>(on ? (p.u + p.s * (f > 0.0 ? d : 0.0)) * f : p.u, OpAdd());
    const int c = wave_reduce<int, OpAdd, G>(p.rank, OpAdd());
    if (tid == 0) s_row = sc_finish(a, r, R, s, u, p.xt, c);
  }
  if (K == 0) return;
  __syncthreads();
  const ScRow rw = s_row;
  const uint64_t bound = max(wave_reduce(kth, OpMax()), wave_reduce(share, OpMin()));   // (every wave's the same)
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (mine[i] >= bound && mine[i] != 0u) cand[atomicAdd(&s_n, 1u)] = mine[i];   // (at most S K)
  __syncthreads();
  const int n = static_cast<int>(s_n);
  sc_place<NT>(cand, n, K, [&](int p, uint64_t key) { sc_emit(a, r, p, key, rw); });
  for (int p = n + tid; p < K; p += NT) sc_emit(a, r, p, 0u, rw);
}

// ---------------------------------------------------------------- gradient
// Element by element: a read and a write of every value, which HBM bounds.
// One work-group per piece of GR_NT x GR_U chunks of a row.  bf16 4096x128256 (2.1
// GB): 355 to 419 us, 5.0 to 5.9 TB/s; f32 255x50257 (103 MB): 18.5 to 20 us.
namespace {
constexpr int GR_NT = 256, GR_U = 4;
}

template <class D>
__global__ __launch_bounds__(GR_NT) void k_score_grad(const fl_score_grad_args a, int pieces) {
  using C = RowChunk<D>;
  constexpr int N = C::N;
  constexpr size_t ESZ = D::id == FL_DTYPE_F32 ? 4 : 2;
  const int tid = threadIdx.x;
  const int V = static_cast<int>(a.vocab);
  const int64_t r = blockIdx.x / static_cast<unsigned>(pieces);
  const int pc = static_cast<int>(blockIdx.x - static_cast<unsigned>(r) * static_cast<unsigned>(pieces));
  constexpr int PIECE = GR_NT * GR_U * N;
  const int base = pc * PIECE, nval = min(PIECE, V - base);
  const __amdgpu_buffer_rsrc_t rx = row_rsrc(
      static_cast<const char*>(a.logits) + (r * a.ld + base) * static_cast<int64_t>(ESZ), static_cast<uint32_t>(nval * ESZ));
  const __amdgpu_buffer_rsrc_t ro = row_rsrc(
      static_cast<char*>(a.out_grad) + (r * a.out_ld + base) * static_cast<int64_t>(ESZ), static_cast<uint32_t>(nval * ESZ));
  uint4 q[GR_U];
#pragma unroll
  for (int k = 0; k < GR_U; ++k) q[k] = buf_load16_once(rx, 16u * static_cast<uint32_t>(tid + k * GR_NT), 0u);
  const float hi = a.saved[4 * r], lo = a.saved[4 * r + 1], H = a.saved[4 * r + 2];
  const float gb = a.grad_entropy ? a.grad_entropy[r] : 0.0f, gc = a.grad_lse ? a.grad_lse[r] : 0.0f;
  float ga = a.grad_logprob ? a.grad_logprob[r] : 0.0f;
  int t = -1;   // the token's place in the piece
  if (a.tokens) {
    const int64_t tk = a.tokens[r];
    if (tk == a.ignore_index) ga = 0.0f;
    else if (tk < 0 || tk >= V) ga = ga == 0.0f ? 0.0f : __builtin_nanf("");   // (as its log-probability)
    else t = static_cast<int>(tk) - base;
  }
  // (a row whose upstream gradients are all 0 has gradient 0, also one without
  // a distribution, as a padded batch's rows may be)
  const bool zero = ga == 0.0f && gb == 0.0f && gc == 0.0f;
  const float k0 = gc - ga, h = gb == 0.0f ? 0.0f : H;
#pragma unroll
  for (int k = 0; k < GR_U; ++k) {
    const int i0 = N * (tid + k * GR_NT);
    if (i0 >= nval) continue;
    float x[N];
    C::unpack(q[k], x);
    if (D::id != FL_DTYPE_F32 && nval - i0 < N) {
      const int last = nval - 1 - i0;   // the last value of an odd row by itself
#pragma unroll
      for (int e = 0; e < N; e += 2)
        if (e == last) x[e] = C::elem(rx, nval - 1);
    }
    float d[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float l = (x[e] - hi) - lo;
      const float p = __builtin_amdgcn_exp2f(l * SC_LOG2E);
      // (log p no lower than -200, where p is 0: 0, not 0 * -inf)
      float g = p * (k0 - gb * (fmaxf(l, -200.0f) + h));
      if (i0 + e == t) g += ga;
      d[e] = zero ? 0.0f : g;
    }
    uint4 o;
    if constexpr (D::id == FL_DTYPE_F32) {
      o = make_uint4(__float_as_uint(d[0]), __float_as_uint(d[1]), __float_as_uint(d[2]), __float_as_uint(d[3]));
    } else {
      uint32_t wd[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) wd[j] = D::from_f32(d[2 * j]) | (D::from_f32(d[2 * j + 1]) << 16);
      o = make_uint4(wd[0], wd[1], wd[2], wd[3]);
    }
    if (nval - i0 >= N) {
      typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
      __builtin_amdgcn_raw_buffer_store_b128(u32x4{o.x, o.y, o.z, o.w}, ro, static_cast<int>(ESZ) * i0, 0, 0);
    } else {   // the row's last chunk, value by value
#pragma unroll
      for (int e = 0; e < N; ++e) {
        if (i0 + e >= nval) break;
        if constexpr (D::id == FL_DTYPE_F32)
          __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(d[e]), ro, 4 * (i0 + e), 0, 0);
        else
          __builtin_amdgcn_raw_buffer_store_b16(static_cast<short>(D::from_f32(d[e])), ro, 2 * (i0 + e), 0, 0);
      }
    }
  }
}

// ---------------------------------------------------------------- launches
namespace {
int sc_slices(int64_t vocab) { return static_cast<int>((vocab + SC_SLICE - 1) / SC_SLICE); }
}  // namespace

size_t score_workspace_bytes(int64_t rows, int64_t vocab, int64_t top_k) {
  const int S = sc_slices(vocab);
  if (S == 1) return 0;
  return static_cast<size_t>(rows) * S * (sizeof(ScPart) + 8 * static_cast<size_t>(top_k));
}

int64_t score_blocks(int64_t rows, int64_t vocab) { return rows * sc_slices(vocab); }
int64_t score_grad_blocks(int64_t rows, int64_t vocab, int dtype) {
  const int64_t piece = static_cast<int64_t>(GR_NT) * GR_U * (dtype == FL_DTYPE_F32 ? 4 : 8);
  return rows * ((vocab + piece - 1) / piece);
}

hipError_t launch_score(const fl_score_args& a, hipStream_t s) {
  ScWs ws;
  ws.S = sc_slices(a.vocab);
  ws.part = static_cast<ScPart*>(a.workspace);
  ws.list = reinterpret_cast<uint64_t*>(ws.part + a.rows * ws.S);
  const dim3 grid(static_cast<unsigned>(a.rows * ws.S));
  const bool ent = a.out_entropy != nullptr, rank = a.out_rank != nullptr;
  auto run = [&](auto d) {
    using D = decltype(d);
    if (ent && rank) hipLaunchKernelGGL((k_score_slice<D, true, true>), grid, dim3(SC_NT), 0, s, a, ws);
    else if (ent) hipLaunchKernelGGL((k_score_slice<D, true, false>), grid, dim3(SC_NT), 0, s, a, ws);
    else if (rank) hipLaunchKernelGGL((k_score_slice<D, false, true>), grid, dim3(SC_NT), 0, s, a, ws);
    else hipLaunchKernelGGL((k_score_slice<D, false, false>), grid, dim3(SC_NT), 0, s, a, ws);
  };
  if (a.dtype == FL_DTYPE_F32) run(F32{});
  else if (a.dtype == FL_DTYPE_BF16) run(BF16{});
  else run(F16{});
  if (ws.S > 1) {
    const dim3 rows(static_cast<unsigned>(a.rows));
    if (ws.S * a.top_k <= WAVE) hipLaunchKernelGGL(k_score_join<WAVE>, rows, dim3(WAVE), 0, s, a, ws);
    else hipLaunchKernelGGL(k_score_join<SC_NT>, rows, dim3(SC_NT), 0, s, a, ws);
  }
  return hipGetLastError();
}

hipError_t launch_score_grad(const fl_score_grad_args& a, hipStream_t s) {
  const int64_t blocks = score_grad_blocks(a.rows, a.vocab, a.dtype);
  const int pieces = static_cast<int>(blocks / a.rows);
  const dim3 grid(static_cast<unsigned>(blocks));
  if (a.dtype == FL_DTYPE_F32) hipLaunchKernelGGL(k_score_grad<F32>, grid, dim3(GR_NT), 0, s, a, pieces);
  else if (a.dtype == FL_DTYPE_BF16) hipLaunchKernelGGL(k_score_grad<BF16>, grid, dim3(GR_NT), 0, s, a, pieces);
  else hipLaunchKernelGGL(k_score_grad<F16>, grid, dim3(GR_NT), 0, s, a, pieces);
  return hipGetLastError();
}

}  // namespace fl

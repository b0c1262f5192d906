// Which tokens, keys and pages a work-group of a call on a paged cache works on: the
// arithmetic alone, for the device and for a host's checks.
#pragma once

#include <stdint.h>

#include "../../include/fl_sampler.h"

#ifdef __HIPCC__
#define FL_HD __host__ __device__ __forceinline__
#else
#define FL_HD inline
#endif

namespace fl {

FL_HD int64_t least(int64_t a, int64_t b) { return a < b ? a : b; }
FL_HD int64_t most(int64_t a, int64_t b) { return a < b ? b : a; }

// A work-group's sequence: its rows row .. row + n - 1 hold the tokens at positions
// pos .. pos + n - 1, and `tile` is the work-group's number among the sequence's.
struct PagedSeq {
  int b, n, tile;
  int64_t row;
  int64_t pos;
};

// Tiles of a launch, `per` of the sequences' rows x mul each: `each` of every sequence
// if it is above 0; else sequence b's begin at starts[b] mul / per + extra b, which
// leaves it floor(n mul / per) + extra of them at least.  (The host has checked that
// tokens x mul and the tiles stay below 2^31.)
FL_HD int64_t paged_tiles(const fl_cache_rows& r, int64_t mul, int64_t per, int64_t extra, int64_t each) {
  return each > 0 ? r.seqs * each : r.tokens * mul / per + extra * r.seqs;
}

// The last of n sequences whose base, base(b), is x or below (or the first): they
// ascend, or x belongs to none.
template <class F>
FL_HD int paged_find(int n, int x, F base) {
  int a = 0, z = n - 1;
  while (a < z) {
    const int m = (a + z + 1) / 2;
    if (base(m) <= x) a = m;
    else z = m - 1;
  }
  return a;
}

// Sequence b, as its rows and positions; what starts and lengths hold cannot lead
// outside the rows.
FL_HD PagedSeq paged_rows(const fl_cache_rows& r, int b) {
  PagedSeq s;
  const int tokens = static_cast<int>(r.tokens), n = tokens / static_cast<int>(r.seqs);
  const int64_t lo = r.starts == nullptr ? n * b : least(most(r.starts[b], 0), tokens);
  const int64_t hi = r.starts == nullptr ? lo + n : least(most(r.starts[b + 1], lo), tokens);
  s.b = b;
  s.tile = 0;
  s.row = lo;
  s.n = static_cast<int>(hi - lo);
  s.pos = static_cast<int64_t>(r.lengths[b]) - s.n;
  return s;
}

// The sequence of tile x.
FL_HD PagedSeq paged_seq(const fl_cache_rows& r, int x, uint32_t mul, uint32_t per, int extra, int each) {
  if (each > 0) {
    PagedSeq s = paged_rows(r, x / each);
    s.tile = x % each;
    return s;
  }
  // (unsigned: what starts holds is below 2^31 / mul, or no matter)
  const auto base = [&](int m) { return static_cast<int>(static_cast<uint32_t>(r.starts[m]) * mul / per + extra * m); };
  PagedSeq s = paged_rows(r, paged_find(static_cast<int>(r.seqs), x, base));
  s.tile = static_cast<int>(most(static_cast<int64_t>(x) - base(s.b), 0));
  return s;
}

// The page of position t (0 <= t), or -1.
FL_HD int paged_page(const fl_cache_rows& r, const fl_cache& c, int b, int64_t t) {
  const int64_t i = t >> __builtin_ctzll(c.page_size);   // (a power of two)
  if (i >= r.table_width) return -1;
  const int p = r.table[b * r.table_ld + i];
  return p >= 0 && p < c.pages ? p : -1;
}

// What a work-group of a write or a read works on: 16 neighbouring slots of one page
// (or -1), slot up, aligned; those from t0 to t1 - 1 hold tokens of the call, slot + t
// the one of row row0 + t.
constexpr int KV_T = 16;
struct KvTile {
  int page, slot, t0, t1;
  int64_t row0;
};
FL_HD int64_t kv_tiles(const fl_cache_rows& r, int* each) {
  // (n tokens touch at most (n + 14) / 16 + 1 aligned runs of 16)
  *each = r.starts != nullptr ? 0 : static_cast<int>((r.tokens / r.seqs + KV_T - 2) / KV_T + 1);
  return paged_tiles(r, 1, KV_T, 2, *each);
}
FL_HD bool kv_tile(const fl_cache_rows& r, const fl_cache& c, const PagedSeq& s, KvTile& t) {
  const int64_t first = most(s.pos, 0), base = first / KV_T * KV_T + static_cast<int64_t>(s.tile) * KV_T;
  const int64_t end = s.pos + s.n;
  if (base >= end) return false;
  t.t0 = static_cast<int>(most(first - base, 0));
  t.t1 = static_cast<int>(least(end - base, KV_T));
  t.row0 = s.row + (base - s.pos);
  t.page = paged_page(r, c, s.b, base);
  t.slot = static_cast<int>(base & (c.page_size - 1));
  return true;
}

constexpr int AT_BLK = 64;          // keys of a step
constexpr int AT_MIN_BLKS = 8;      // steps of a split, at least
constexpr int AT_MAX_SPLITS = 64;

// A launch's plan.  Rows of a sequence and cached head: (token, head of the group),
// r = token * group + head; tiles of `tr` rows.
struct AttnPlan {
  int group;          // query heads per cached head
  int tr;             // rows of a tile
  int splits;         // parts that a tile's keys may be split into
  int min_rows;       // sequences of fewer rows, or
  int max_rows;       // more rows, are another launch's
  int each;           // tiles of every sequence, or 0
  int slots;          // rows of a sequence and cached head that have a place for parts, or 0: all of the call's
  int64_t tiles;
  float* part;        // [places][splits][dim]
  float* stat;        // [places][splits][2]: maximum (powers of two) and sum
};

// Where the parts of a sequence's row r of cached head h are, which is the call's row
// `row` (token * q_heads + head).
FL_HD int64_t attn_place(const AttnPlan& p, int b, int64_t heads, int h, int r, int64_t row) {
  return p.slots > 0 ? (b * heads + h) * p.slots + r : row;
}

// The keys that a tile's tokens see, in steps of 64: those of the first `sink` steps
// and of the steps from `low` on, `blocks` in all; and how many splits they make.
// (The host has checked that keys number 2^30 at most.)
struct AttnSpan {
  int64_t pmin, pmax;   // positions of the tile's first and last token
  int end;              // keys end here
  int sink, blocks, splits, low;
  int all, open, sinks;   // every token sees the keys up to `all` that are above `open` or below `sinks`
  FL_HD int key(int i) const { return AT_BLK * (i < sink ? i : low + (i - sink)); }   // the first key of step i
  // Whether every key of the step from t0 on is seen by every token of the tile.
  FL_HD bool whole(int t0) const { return t0 + AT_BLK - 1 <= all && (t0 > open || t0 + AT_BLK <= sinks); }
};

constexpr int64_t AT_FAR = 0x7fffff00;   // beyond any key

FL_HD AttnSpan attn_span(const fl_attn_args& a, const AttnPlan& p, const PagedSeq& s, int tile) {
  AttnSpan v;
  const int r0 = tile * p.tr, r1 = static_cast<int>(least(r0 + p.tr, s.n * p.group)) - 1;
  v.pmin = s.pos + r0 / p.group;
  v.pmax = s.pos + r1 / p.group;
  // (a position past the table is no key's: its query is given NaN)
  v.end = static_cast<int>(least(most(v.pmax + 1, 0), a.rows.table_width * a.cache.page_size));
  v.low = 0;
  v.sink = 0;
  v.all = static_cast<int>(least(most(v.pmin, -1), AT_FAR));
  v.open = a.window > 0 ? static_cast<int>(least(most(v.pmax - a.window, -1), AT_FAR)) : -1;
  v.sinks = a.window > 0 ? static_cast<int>(least(a.sinks, AT_FAR)) : 0;
  if (a.window > 0) {
    v.low = static_cast<int>(least(most(v.pmin - a.window + 1, 0), AT_FAR)) / AT_BLK;
    v.sink = static_cast<int>(least((least(v.sinks, v.end) + AT_BLK - 1) / AT_BLK, v.low));
  }
  const int last = (v.end + AT_BLK - 1) / AT_BLK;
  v.blocks = static_cast<int>(v.sink + most(last - v.low, 0));
  v.splits = static_cast<int>(most(1, least(p.splits, (v.blocks + AT_MIN_BLKS - 1) / AT_MIN_BLKS)));
  return v;
}

// The keys that a token at position `at` sees: t <= last and (t >= from or t < sinks).
struct AttnSeen {
  int last, from;
};
FL_HD AttnSeen attn_seen(const fl_attn_args& a, int64_t at) {
  return {static_cast<int>(least(most(at, -1), AT_FAR)),
          a.window > 0 ? static_cast<int>(least(most(at - a.window + 1, 0), AT_FAR)) : 0};
}

}  // namespace fl

// paged_schedule.h — how attention over a paged cache is dealt to the CTAs of a launch, as arithmetic that every CTA repeats.
//
// The host knows neither the lengths nor how many new tokens a sequence has, so the split is made on the device.  The work of
// a launch is laid out on a line: sequence after sequence, kv head after kv head, tile after tile of query tokens; a UNIT (one
// tile of one kv head of one sequence) covers as many points as it has keys to walk, plus `overhead` for starting and ending it.
// CTA c of G takes the points [cut(c), cut(c + 1)): equal shares whatever the lengths are, one sequence of 30000 keys or a
// thousand of 30.  A cut inside a unit falls between two of its key blocks (paged_block); the two CTAs beside it compute it by
// the same integer arithmetic.  A CTA that has only part of a unit's blocks parks what it has, in one of its TWO slots — it can
// hold the end of one unit and the beginning of another, never more — and a second kernel joins the parts of a unit in order.
// So the scratch depends on G alone, and the result on the batch alone: no atomics, no order of arrival.
#pragma once
#include <cstdint>

#ifdef __CUDACC__
#define OPS_HD __host__ __device__ __forceinline__
#else
#define OPS_HD inline
#endif

namespace ops {

typedef long long i64;

// A sequence's rows [row, row + n) of the step and its cache slots [0, len).
struct PagedSeq {
  int row, n, len;
};

struct PagedLine {
  int nkvh, group, causal;
  int rows_lo, rows_hi;  // the sequences on this line: rows_lo <= n * group <= rows_hi (n > 0)
  int max_seq;           // ... and n <= max_seq
  int tokens;            // query tokens of a unit
  int block;             // keys of a block
  int overhead;          // points in front of a unit's keys
  int min_share;         // no CTA gets fewer points than this, as long as one has any
  int ctas;
};

// What one sequence puts on the line: per kv head `tiles` units, the p-th of overhead + base + ramp * (p + 1) points.  (Causal
// tiles see `tokens` keys more each; the last one may see fewer, which the line does not bother to know.)
struct PagedSpan {
  int tiles, base, ramp;
  i64 head;  // points of one kv head
};

OPS_HD PagedSpan paged_span(const PagedLine &l, const PagedSeq &s) {
  PagedSpan p;
  const i64 rows = (i64)s.n * l.group;
  if (s.n <= 0 || s.n > l.max_seq || rows < l.rows_lo || rows > l.rows_hi) {
    p.tiles = p.base = p.ramp = 0;
    p.head = 0;
    return p;
  }
  p.tiles = (s.n + l.tokens - 1) / l.tokens;
  const bool ramped = l.causal && p.tiles > 1;
  p.base = ramped ? (s.len > s.n ? s.len - s.n : 0) : (s.len > 0 ? s.len : 1);
  p.ramp = ramped ? l.tokens : 0;
  p.head = (i64)p.tiles * (l.overhead + p.base) + (i64)p.ramp * ((i64)p.tiles * (p.tiles + 1) / 2);
  return p;
}

struct PagedUnit {
  int head, tile;
  i64 begin, cost;  // on the sequence's stretch of the line
};

OPS_HD i64 paged_tile_begin(const PagedLine &l, const PagedSpan &p, i64 tile) {
  return tile * (l.overhead + p.base) + (i64)p.ramp * (tile * (tile + 1) / 2);
}

// The unit that holds point `at` of the sequence's stretch, 0 <= at < nkvh * head.
OPS_HD PagedUnit paged_unit(const PagedLine &l, const PagedSpan &p, i64 at) {
  PagedUnit u;
  u.head = (int)(at / p.head);
  const i64 in_head = at - (i64)u.head * p.head;
  int lo = 0, hi = p.tiles;  // begin(lo) <= in_head < begin(hi)
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (paged_tile_begin(l, p, mid) <= in_head) lo = mid;
    else hi = mid;
  }
  u.tile = lo;
  u.begin = (i64)u.head * p.head + paged_tile_begin(l, p, lo);
  u.cost = l.overhead + p.base + (i64)p.ramp * (lo + 1);
  return u;
}

// Keys that tokens [t0, t1) of a sequence see at most, and the blocks they fill: one at least, so that rows that see nothing are
// written all the same.
OPS_HD int paged_keys(const PagedLine &l, const PagedSeq &s, int t1) {
  if (!l.causal) return s.len;
  const int k = s.len - s.n + (t1 < s.n ? t1 : s.n);
  return k > 0 ? k : 0;
}
OPS_HD int paged_blocks(const PagedLine &l, const PagedSeq &s, int tile) {
  const int k = paged_keys(l, s, (tile + 1) * l.tokens);
  return k > 0 ? (k + l.block - 1) / l.block : 1;
}

// First block behind a cut at point `at` (of the sequence's stretch) of unit u.
OPS_HD int paged_block(const PagedLine &l, const PagedUnit &u, int blocks, i64 at) {
  if (at <= u.begin) return 0;
  if (at >= u.begin + u.cost) return blocks;
  const i64 t = at - u.begin - l.overhead;
  return t <= 0 ? 0 : (int)(t * blocks / (u.cost - l.overhead));
}

// CTAs that get anything, and where CTA c's share begins.
OPS_HD int paged_active(const PagedLine &l, i64 total) {
  const i64 most = (total + l.min_share - 1) / l.min_share;
  return (int)(most < l.ctas ? most : l.ctas);
}
OPS_HD i64 paged_cut(i64 total, int active, int c) { return total / active * c + total % active * c / active; }

// The first CTA whose share begins at or behind point x, 0 < x <= total (`active` if there is none).
OPS_HD int paged_first_behind(i64 total, int active, i64 x) {
  int c = (int)((double)x * active / (double)total);
  while (c > 0 && paged_cut(total, active, c) >= x) --c;
  while (c < active && paged_cut(total, active, c) < x) ++c;
  return c;
}

// A CTA's part of a unit.
struct PagedPiece {
  int seq;  // -1: no more
  PagedSeq s;
  int head, tile;
  int lo, hi, blocks;  // key blocks [lo, hi) of `blocks`
  OPS_HD bool whole() const { return lo == 0 && hi == blocks; }
  OPS_HD int slot() const { return lo > 0 ? 0 : 1; }
};

// Where a CTA is on its share: sequence `seq` begins at point `begin` of the line.
struct PagedWalk {
  int seq;
  i64 begin, at, end;
};

// The next piece of the share (an empty one is passed over).  Seqs: seq index -> PagedSeq.
template <class Seqs> OPS_HD PagedPiece paged_next(const PagedLine &l, int nseq, PagedWalk &w, const Seqs &seqs) {
  PagedPiece q;
  q.seq = -1;
  while (w.at < w.end && w.seq < nseq) {
    const PagedSeq s = seqs(w.seq);
    const PagedSpan p = paged_span(l, s);
    const i64 all = p.head * l.nkvh;
    if (w.at >= w.begin + all) {
      w.begin += all;
      ++w.seq;
      continue;
    }
    const PagedUnit u = paged_unit(l, p, w.at - w.begin);
    const int blocks = paged_blocks(l, s, u.tile);
    const i64 stop = w.begin + u.begin + u.cost < w.end ? w.begin + u.begin + u.cost : w.end;
    const int lo = paged_block(l, u, blocks, w.at - w.begin), hi = paged_block(l, u, blocks, stop - w.begin);
    w.at = stop;
    if (lo == hi) continue;
    q.seq = w.seq;
    q.s = s;
    q.head = u.head;
    q.tile = u.tile;
    q.lo = lo;
    q.hi = hi;
    q.blocks = blocks;
    break;
  }
  return q;
}

}  // namespace ops

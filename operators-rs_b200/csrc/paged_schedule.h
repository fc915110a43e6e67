// paged_schedule.h — how attention over a paged cache is dealt to the CTAs of a launch, as arithmetic that every CTA repeats.
//
// The host knows neither the lengths nor how many new tokens a sequence has, so the split is made on the device.  The work of
// a launch is laid out on a line: sequence after sequence, kv head after kv head, tile after tile of query tokens; a UNIT (one
// tile of one kv head of one sequence) covers as many points as it has keys to walk, plus `overhead` for starting and ending it.
// CTA c of G takes the points [cut(c), cut(c + 1)): equal shares whatever the lengths are, one sequence of 30000 keys or a
// thousand of 30.  A cut inside a unit falls between two of its key blocks (paged_block); the two CTAs beside it compute it by
// the same integer arithmetic.  A CTA that has only part of a unit's blocks parks what it has, in one of its TWO slots — it can
// hold the end of one unit and the beginning of another, never more.  The parts of a unit are joined by
// the last to come, or with its help (nobody's result waits for a CTA that is not there yet), always in the same order: the
// scratch depends on G alone, the result on the batch alone, not on the order of arrival.
//
// A point is 2^shift keys, with the least shift that keeps every line the host can expect within 31 bits: the arithmetic is
// 32-bit throughout, without a division by anything but what the host knows, and one warp of a CTA does it.  What the others
// wait for at the start of a launch is this.
#pragma once
#include <algorithm>
#include <cmath>
#include <cstddef>
#include <cstdint>

#ifdef __CUDACC__
#define OPS_HD __host__ __device__ __forceinline__
#define OPS_ROLLED _Pragma("unroll 1")
#else
#define OPS_HD inline
#define OPS_ROLLED
#endif

namespace ops {

// n / d for 0 <= n < 2^31 with a divisor that the host knows: a multiplication and a shift.  (A division by a variable takes some
// 200 clocks, and a thread that finds a CTA's share is what all others wait for.)
struct PagedDiv {
  uint32_t mul;
  int shift;
};
inline PagedDiv paged_div_by(uint32_t d) {  // mul = ceil(2^(31 + shift) / d), 2^(shift - 1) < d <= 2^shift
  PagedDiv v;
  v.shift = 0;
  while ((1ull << v.shift) < d) ++v.shift;
  v.mul = (uint32_t)(((1ull << (31 + v.shift)) + d - 1) / d);
  return v;
}
// near enough to be put right by one
OPS_HD int paged_guess(float a, float b) {
#ifdef __CUDA_ARCH__
  return (int)__fdividef(a, b);
#else
  return (int)(a / b);
#endif
}
OPS_HD int paged_div(int n, const PagedDiv &d) { return (int)(((unsigned long long)(unsigned)n * d.mul) >> (31 + d.shift)); }

// A sequence's rows [row, row + n) of the step and its cache slots [0, len).
struct PagedSeq {
  int row, n, len;
};

struct PagedLine {
  int nkvh, group, causal;
  int rows_lo, rows_hi;  // the sequences on this line: rows_lo <= n * group <= rows_hi (n > 0); 0x7fffffff: no upper bound
  int max_seq;           // ... and n <= max_seq
  int tokens;            // query tokens of a unit
  int block_log2;        // keys of a block
  int shift;             // log2 of the keys of a point
  int overhead;          // points in front of a unit's keys
  int min_share, min_share_log2;  // no CTA gets fewer points than this, a power of two and a block at least, as long as there are any
  int ctas;
  PagedDiv by_group, by_tokens, by_ctas;
};

constexpr int AP_MAX_CTAS = 256;  // of a kernel
constexpr int AP_SHARES = 16;     // the few-rows line gets k / 16 of the CTAs where both have work
constexpr int AP_FEW_JOIN = 16, AP_LEVELS = 2;  // parts are joined in groups, the groups in turn: 16^2 is AP_MAX_CTAS
constexpr int AP_FEW_BLOCK_LOG2 = 5, AP_FEW_BLOCK = 32, AP_TILE_BLOCK_LOG2 = 7, AP_TILE_BLOCK = 128;  // keys of a block
constexpr int AP_TILE_ROWS = 256;                       // query rows of a unit of the tile kernel: two tiles

// The few-rows line's CTAs for k of 16 shares; the tiles get the others.
OPS_HD int paged_share(int ctas, int k) { return ctas * k / AP_SHARES > 0 ? ctas * k / AP_SHARES : 1; }

// The lines of a launch.  A sequence goes to the line of few rows when its new tokens times the query heads of a kv head fit;
// sequences with more go to the tiles.
struct PagedLines {
  PagedLine few, tile;  // ctas == 0: nothing can be on it
  int few_rows;
  bool fit;  // whatever the device finds in the batch, both fit in 31 bits
};

// The least shift with which a line cannot pass 31 bits: units, at most all rows in tiles and one more per sequence with rows, of at
// most all slots and rows; false: there is none.  `overhead`, `min_share`: keys.
inline bool paged_line_scale(PagedLine *l, size_t nt, size_t nseq, size_t slots, int overhead, int min_share) {
  const double units = ((double)(nt / (size_t)l->tokens) + (double)std::min(nseq, nt)) * l->nkvh, keys = (double)slots + (double)nt + l->tokens + overhead;
  auto fits = [&] { return units * (std::ldexp(keys, -l->shift) + 4.0) <= 2147483647.0; };
  l->shift = 0;
  while (l->shift < 30 && !fits()) ++l->shift;
  l->overhead = std::max(1, overhead >> l->shift);
  l->min_share = std::max(1, min_share >> l->shift);  // a power of two
  l->min_share_log2 = 0;
  while ((1 << l->min_share_log2) < l->min_share) ++l->min_share_log2;
  l->by_tokens = paged_div_by((uint32_t)l->tokens);
  l->by_ctas = paged_div_by((uint32_t)l->ctas);
  return fits();
}

// For nt rows and nseq sequences of up to `slots` slots; max_seq: 0xffffffff when unknown.
inline PagedLines paged_lines(int sm_count, size_t nh, size_t nkvh, bool causal, uint32_t max_seq, size_t nt, size_t nseq, size_t slots) {
  PagedLines p = PagedLines();
  p.fit = true;
  const size_t group = nh / nkvh, most = max_seq == 0xffffffffu ? 0xffffffffull : (size_t)max_seq * group;
  // 16 rows cost the kernel a third of its ring; 8 are enough for one token of up to 8 heads
  p.few_rows = group <= 8 && !(most > 8 && most <= 16) ? 8 : 16;
  PagedLine l = PagedLine();
  l.nkvh = (int)nkvh;
  l.group = (int)group;
  l.by_group = paged_div_by((uint32_t)group);
  l.causal = causal;
  l.max_seq = max_seq > 0x7fffffffu ? 0x7fffffff : (int)max_seq;
  p.few = p.tile = l;
  if (group <= (size_t)p.few_rows) {
    p.few.rows_lo = 1;
    p.few.rows_hi = p.few_rows;
    p.few.tokens = p.few_rows;
    p.few.block_log2 = AP_FEW_BLOCK_LOG2;
    p.few.ctas = std::min(sm_count, AP_MAX_CTAS);  // one a SM: the ring takes its shared memory
    p.fit = paged_line_scale(&p.few, nt, nseq, slots, 128, 128);
    p.tile.rows_lo = p.few_rows + 1;
  } else {
    p.tile.rows_lo = 1;
  }
  if (most >= (size_t)p.tile.rows_lo) {
    p.tile.rows_hi = 0x7fffffff;
    p.tile.tokens = AP_TILE_ROWS / 2 / (int)group * 2;
    p.tile.block_log2 = AP_TILE_BLOCK_LOG2;
    p.tile.ctas = std::min(sm_count, AP_MAX_CTAS);
    p.fit = paged_line_scale(&p.tile, nt, nseq, slots, 512, 512) && p.fit;
  }
  return p;
}

// What one sequence puts on the line: per kv head `tiles` units, the p-th of base + ramp * (p + 1) points, the overhead among
// them.  (Causal tiles see `tokens` keys more each; the last one may see fewer, which the line does not bother to know.)
struct PagedSpan {
  int tiles, base, ramp;
  int head;  // points of one kv head
};

OPS_HD int paged_points(const PagedLine &l, int keys) { return (int)(((unsigned)keys + ((1u << l.shift) - 1u)) >> l.shift); }

OPS_HD int paged_tile_begin(const PagedSpan &p, int tile) { return tile * p.base + p.ramp * (int)((long long)tile * (tile + 1) / 2); }

OPS_HD PagedSpan paged_span(const PagedLine &l, const PagedSeq &s) {
  PagedSpan p;
  p.tiles = p.base = p.ramp = p.head = 0;
  const long long rows = (long long)s.n * l.group;
  if (s.n <= 0 || s.n > l.max_seq || rows < l.rows_lo || (rows > l.rows_hi && l.rows_hi != 0x7fffffff)) return p;
  p.tiles = s.n <= l.tokens ? 1 : paged_div(s.n + l.tokens - 1, l.by_tokens);
  const bool ramped = l.causal && p.tiles > 1;
  p.base = l.overhead + paged_points(l, ramped ? (s.len > s.n ? s.len - s.n : 0) : (s.len > 0 ? s.len : 1));
  p.ramp = ramped ? l.tokens >> l.shift : 0;
  p.head = paged_tile_begin(p, p.tiles);
  return p;
}

struct PagedUnit {
  int head, tile;
  int begin, cost;  // on the sequence's stretch of the line
};

// The unit that holds point `at` of the sequence's stretch, 0 <= at < nkvh * head.
OPS_HD PagedUnit paged_unit(const PagedSpan &p, int at) {
  PagedUnit u;
  u.head = paged_guess((float)at, (float)p.head);  // heads are few: off by one at most
  if (u.head * p.head > at) --u.head;
  else if (at - u.head * p.head >= p.head) ++u.head;
  const int in_head = at - u.head * p.head;
  int lo = 0, hi = p.tiles;  // begin(lo) <= in_head < begin(hi)
  OPS_ROLLED while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (paged_tile_begin(p, mid) <= in_head) lo = mid;
    else hi = mid;
  }
  u.tile = lo;
  u.begin = u.head * p.head + paged_tile_begin(p, lo);
  u.cost = p.base + p.ramp * (lo + 1);
  return u;
}

// Keys that the tokens of a sequence in front of token t1 see at most, and the blocks they fill: one at least, so that rows that
// see nothing are written all the same.
OPS_HD int paged_keys(const PagedLine &l, const PagedSeq &s, int t1) {
  if (!l.causal) return s.len;
  const int k = s.len - s.n + (t1 < s.n ? t1 : s.n);
  return k > 0 ? k : 0;
}
OPS_HD int paged_blocks(const PagedLine &l, const PagedSeq &s, int tile) {
  const int k = paged_keys(l, s, (tile + 1) * l.tokens);
  return k > 0 ? (k + (1 << l.block_log2) - 1) >> l.block_log2 : 1;
}

// First block behind a cut `at` points behind the beginning of a unit.  (The points of a ramped unit may stand for a few keys more
// than its last blocks hold: those cuts fall behind its end.)
OPS_HD int paged_block(const PagedLine &l, int cost, int blocks, int at) {
  if (at >= cost) return blocks;
  const int t = at - l.overhead;
  if (t <= 0) return 0;
  const int b = l.shift <= l.block_log2 ? t >> (l.block_log2 - l.shift) : t << (l.shift - l.block_log2);
  return b < blocks ? b : blocks;
}

// Shares: equal ones if every CTA gets min_share points at least, else shares of min_share for as many as there are points for.
// CTAs that get anything, and where CTA c's share begins.
OPS_HD bool paged_all(const PagedLine &l, int total) { return total >= l.min_share * l.ctas; }
OPS_HD int paged_active(const PagedLine &l, int total) {
  if (paged_all(l, total)) return l.ctas;
  return (total + l.min_share - 1) >> l.min_share_log2;
}
OPS_HD int paged_cut(const PagedLine &l, int total, int c) {
  if (paged_all(l, total)) {
    const int each = paged_div(total, l.by_ctas);
    return each * c + paged_div((total - each * l.ctas) * c, l.by_ctas);
  }
  const int cut = c * l.min_share;
  return cut < total ? cut : total;
}

// The first CTA whose share begins at or behind point x, 0 < x <= total (`active` if there is none).
OPS_HD int paged_first_behind(const PagedLine &l, int total, int x) {
  const int active = paged_active(l, total);
  int c = paged_guess((float)x * (float)active, (float)total);
  if (c > active) c = active;
  OPS_ROLLED while (c > 0 && paged_cut(l, total, c) >= x) --c;
  OPS_ROLLED while (c < active && paged_cut(l, total, c) < x) ++c;
  return c;
}

// A CTA's part of a unit.
struct PagedPiece {
  int seq;  // -1: no more
  PagedSeq s;
  int head, tile;
  int lo, hi, blocks;  // key blocks [lo, hi) of `blocks`
  int begin, cost;     // of the unit, on the line
};

// The CTAs [first, first + count) that have blocks of the unit, each some; 1: the piece is all of it.  (The unit's points may lie
// in the shares of more, whose cuts leave them none: in front of its overhead's end, or behind its last block.)
struct PagedParts {
  int first, count;
};
OPS_HD PagedParts paged_parts(const PagedLine &l, int total, int cta, const PagedPiece &q) {
  PagedParts p;
  p.first = cta;
  p.count = 1;
  if (q.lo == 0 && q.hi == q.blocks) return p;
  if (q.lo > 0) {
    p.first = paged_first_behind(l, total, q.begin + 1) - 1;
    OPS_ROLLED while (paged_block(l, q.cost, q.blocks, paged_cut(l, total, p.first + 1) - q.begin) == 0) ++p.first;
  }
  int end = cta + 1;
  if (q.hi < q.blocks) {
    end = paged_first_behind(l, total, q.begin + q.cost);
    OPS_ROLLED while (paged_block(l, q.cost, q.blocks, paged_cut(l, total, end - 1) - q.begin) == q.blocks) --end;
  }
  p.count = end - p.first;
  return p;
}
// The slot of the k-th part of a unit: its first is the end of its CTA's share, the others are the beginnings of theirs.
OPS_HD int paged_slot(int first, int k) { return (first + k) * 2 + (k == 0 ? 1 : 0); }
// The slot of parts [k, k + size) joined, behind the slots of the parts: the CTA of the k-th part has one.  (A group of one stays where
// it is: the CTA of a unit's last part may be the first of the next unit, whose first group has that slot.  In larger groups that
// CTA is not the first.)
OPS_HD int paged_group_slot(const PagedLine &l, int first, int k, int size) { return size == 1 ? paged_slot(first, k) : 2 * l.ctas + first + k; }

// Where a CTA is on its share: sequence `seq` begins at point `begin` of the line.
struct PagedWalk {
  int seq;
  int begin, at, end;
};

// Whether a sequence with rows [r0, r1) can have points on the line (max_seq may still rule it out).
OPS_HD bool paged_rows_fit(const PagedLine &l, uint32_t r0, uint32_t r1) {
  if (r1 <= r0) return false;
  const unsigned long long rows = (unsigned long long)(r1 - r0) * (unsigned)l.group;
  return rows >= (unsigned)l.rows_lo && (rows <= (unsigned)l.rows_hi || l.rows_hi == 0x7fffffff);
}

// The next piece of the share (an empty one is passed over).  Seqs: seq index -> PagedSeq.  Skip: the first sequence from the given
// one on that has points on the line, or any in front of it; it is asked when one without any has been met.
template <class Seqs, class Skip> OPS_HD PagedPiece paged_next(const PagedLine &l, int nseq, PagedWalk &w, const Seqs &seqs, const Skip &skip) {
  PagedPiece q;
  q.seq = -1;
  OPS_ROLLED while (w.at < w.end && w.seq < nseq) {
    q.s = seqs(w.seq);
    const PagedSpan p = paged_span(l, q.s);
    const int all = p.head * l.nkvh;
    if (w.at >= w.begin + all) {
      w.begin += all;
      ++w.seq;
      if (all == 0) w.seq = skip(w.seq);
      continue;
    }
    const PagedUnit u = paged_unit(p, w.at - w.begin);
    q.head = u.head;
    q.tile = u.tile;
    q.begin = w.begin + u.begin;
    q.cost = u.cost;
    q.blocks = paged_blocks(l, q.s, u.tile);
    q.lo = paged_block(l, u.cost, q.blocks, w.at - q.begin);
    w.at = q.begin + u.cost < w.end ? q.begin + u.cost : w.end;
    q.hi = paged_block(l, u.cost, q.blocks, w.at - q.begin);
    if (q.lo == q.hi) continue;
    q.seq = w.seq;
    break;
  }
  return q;
}
template <class Seqs> OPS_HD PagedPiece paged_next(const PagedLine &l, int nseq, PagedWalk &w, const Seqs &seqs) {
  return paged_next(l, nseq, w, seqs, [](int seq) { return seq; });
}

}  // namespace ops

// Walks the schedule of random batches on the CPU: every key block of every unit belongs to exactly one CTA, a CTA parks at most
// one part in each of its two slots, shares are even, and every part of a unit knows which CTAs have the others.
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <tuple>
#include <vector>

#include "../operators-rs_b200/csrc/paged_schedule.h"

using namespace ops;

#define CHECK(x)                                                            \
  do {                                                                      \
    if (!(x)) {                                                             \
      printf("round %d: %s failed (line %d)\n", round_no, #x, __LINE__);    \
      return 1;                                                             \
    }                                                                       \
  } while (0)

int main() {
  std::mt19937 rng(7);
  const int round_no = -1;
  for (uint32_t d = 1; d <= 70000; d += d < 300 ? 1 : 97)
    for (uint32_t n : {0u, 1u, d - 1, d, d + 1, 2 * d - 1, 1000 * d - 1, 1000 * d, 0x7fffffffu, 0x7fffffffu - d, 0x7fffffffu / d * d, 0x7fffffffu / d * d - 1, (uint32_t)(rng() >> 1)})
      if (n <= 0x7fffffffu) CHECK(paged_div((int)n, paged_div_by(d)) == (int)(n / d));
  auto pick = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
  for (int round_no = 0; round_no < 3000; ++round_no) {
    PagedLine l;
    l.group = std::vector<int>{1, 2, 4, 7, 8, 16, 32}[pick(0, 6)];
    l.nkvh = pick(1, 9);
    l.causal = pick(0, 3) > 0;
    const bool tile = pick(0, 1);
    const int few = 16;
    l.rows_lo = tile ? few + 1 : 1;
    l.rows_hi = tile ? 0x7fffffff : few;
    l.max_seq = pick(0, 4) ? 0x7fffffff : pick(1, 40);
    l.tokens = tile ? 2 * (128 / l.group) : few;
    l.block_log2 = tile ? 7 : 6;
    const int block = 1 << l.block_log2;
    // (a share holds a block at least: no CTA in the middle of a unit goes without)
    const int overhead = pick(1, 600), min_share = pick(1 << l.block_log2, 900);
    l.ctas = std::vector<int>{1, 3, 148, 296}[pick(0, 3)];
    std::vector<PagedSeq> seqs(pick(0, round_no % 10 ? 12 : 400));
    const int big = round_no % 7 ? 300 : 20000;
    int row = 0;
    for (auto &s : seqs) {
      s.n = pick(0, 2) ? pick(0, 3) : pick(0, big);
      s.len = pick(0, 9) ? s.n + pick(0, big) : pick(0, 5);
      s.row = row;
      row += s.n;
    }
    const int nseq = (int)seqs.size();
    // the host's bound: all rows in tiles and one more unit per sequence, each of all slots and rows
    int slots = 1;
    for (auto &s : seqs) slots = std::max(slots, s.len);
    const double count = ((double)row / l.tokens + nseq) * l.nkvh, most = (double)slots + row + l.tokens + overhead;
    l.shift = pick(0, 3) ? 0 : pick(0, 7);
    while (count * (most / (1 << l.shift) + 4.0) > 2147483647.0) ++l.shift;
    l.overhead = std::max(1, overhead >> l.shift);
    l.min_share = 1;
    while (l.min_share * 2 <= std::max(1, min_share >> l.shift)) l.min_share *= 2;
    l.min_share_log2 = 0;
    while ((1 << l.min_share_log2) < l.min_share) ++l.min_share_log2;
    l.by_group = paged_div_by(l.group);
    l.by_tokens = paged_div_by(l.tokens);
    l.by_ctas = paged_div_by(l.ctas);
    long long sum = 0;
    for (auto &s : seqs) sum += (long long)paged_span(l, s).head * l.nkvh;
    CHECK(sum <= 0x7fffffff);  // the shift below is chosen like the host's
    const int total = (int)sum;
    if (total == 0) continue;
    const int active = paged_active(l, total);
    CHECK(active >= 1 && active <= l.ctas);
    CHECK(paged_cut(l, total, 0) == 0 && paged_cut(l, total, active) == total);
    auto at = [&](int i) { return seqs[i]; };
    struct Part {
      int lo, hi, cta;
      PagedParts parts;
    };
    std::map<std::tuple<int, int, int>, std::vector<Part>> units;  // (seq, head, tile) -> its parts
    std::map<std::tuple<int, int, int>, int> blocks;
    std::map<int, int> parked;
    for (int c = 0; c < active; ++c) {
      PagedWalk w{0, 0, paged_cut(l, total, c), paged_cut(l, total, c + 1)};
      long long keys = 0;
      int steps = 0;
      for (PagedPiece q = paged_next(l, nseq, w, at); q.seq >= 0; q = paged_next(l, nseq, w, at)) {
        CHECK(++steps < 1000000);
        CHECK(q.lo < q.hi && q.hi <= q.blocks && q.lo >= 0);
        const PagedParts parts = paged_parts(l, total, c, q);
        CHECK((parts.count == 1) == (q.lo == 0 && q.hi == q.blocks));
        if (parts.count > 1) CHECK(++parked[paged_slot(parts.first, c - parts.first)] == 1 && paged_slot(parts.first, c - parts.first) / 2 == c);
        units[{q.seq, q.head, q.tile}].push_back({q.lo, q.hi, c, parts});
        blocks[{q.seq, q.head, q.tile}] = q.blocks;
        keys += (q.hi - q.lo);
      }
      // a share is its points' blocks, to within the roundings at its two ends and the short last block and tile of a unit (a point
      // of several keys rounds the ramp of a causal unit down)
      if (l.shift == 0) CHECK(keys <= ((long long)(paged_cut(l, total, c + 1) - paged_cut(l, total, c)) / block + 2 + 2 * steps) * 9 / 8);
    }
    size_t want = 0;
    for (int i = 0; i < nseq; ++i) {
      const PagedSpan p = paged_span(l, seqs[i]);
      const long long rows = (long long)seqs[i].n * l.group;
      CHECK((p.tiles > 0) == (seqs[i].n > 0 && rows >= l.rows_lo && rows <= l.rows_hi && seqs[i].n <= l.max_seq));
      if (p.tiles) CHECK((long long)p.tiles * l.tokens >= seqs[i].n && (long long)(p.tiles - 1) * l.tokens < seqs[i].n);
      want += (size_t)p.tiles * l.nkvh;
    }
    CHECK(units.size() == want);
    // the few-rows kernel joins a unit's parts 16 at a time: no two groups share a slot, or a slot with a part
    std::map<int, int> joined;
    for (auto &u : units) {
      const int count = (int)u.second.size(), first = u.second[0].parts.first;
      for (int k = 0; count > 16 && k < count; k += 16) {
        const int size = std::min(16, count - k), slot = paged_group_slot(l, first, k, size);
        if (size == 1) CHECK(slot == paged_slot(first, k));
        else CHECK(slot >= 2 * l.ctas && slot < 3 * l.ctas && ++joined[slot] == 1);
      }
    }
    for (auto &u : units) {
      int next = 0, k = 0;
      for (auto &part : u.second) {
        CHECK(part.lo == next && part.parts.count == (int)u.second.size() && part.parts.first + k++ == part.cta);
        next = part.hi;
      }
      CHECK(next == blocks[u.first]);
      const PagedSeq &s = seqs[std::get<0>(u.first)];
      const int keys = paged_keys(l, s, (std::get<2>(u.first) + 1) * l.tokens);
      CHECK((long long)blocks[u.first] * block >= keys && (keys == 0 || (long long)(blocks[u.first] - 1) * block < keys));
    }
    for (int k = 0; k < 20; ++k) {
      const int x = k ? 1 + (int)(rng() % (unsigned)total) : total;
      int c = 0;
      while (c < active && paged_cut(l, total, c) < x) ++c;
      CHECK(paged_first_behind(l, total, x) == c);
    }
  }
  printf("schedule ok\n");
  return 0;
}

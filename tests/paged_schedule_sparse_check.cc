// Walks batches of a few sequences with work between thousands without: the pieces are those of the plain walk, and the number of
// sequences looked at one by one does not grow with those that have none.
#include <cstdio>
#include <random>
#include <vector>

#include "../operators-rs_b200/csrc/paged_schedule.h"

using namespace ops;

#define CHECK(x)                                                         \
  do {                                                                   \
    if (!(x)) {                                                          \
      printf("round %d: %s failed (line %d)\n", round_no, #x, __LINE__); \
      return 1;                                                          \
    }                                                                    \
  } while (0)

int main() {
  std::mt19937 rng(5);
  auto pick = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
  for (int round_no = 0; round_no < 200; ++round_no) {
    PagedLine l;
    l.nkvh = pick(1, 4);
    l.group = 4;
    l.causal = 1;
    l.rows_lo = 17;
    l.rows_hi = l.max_seq = 0x7fffffff;
    l.tokens = 64;
    l.block_log2 = 7;
    l.shift = 0;
    l.overhead = l.min_share = 512;
    l.min_share_log2 = 9;
    l.ctas = pick(1, 148);
    l.by_group = paged_div_by(l.group);
    l.by_tokens = paged_div_by(l.tokens);
    l.by_ctas = paged_div_by(l.ctas);
    // chunks, idle sequences and single tokens (which are not on this line), in runs
    std::vector<PagedSeq> seqs;
    int row = 0, chunks = 0;
    for (int run = pick(1, 8); run > 0; --run) {
      const int kind = pick(0, 2), count = kind == 0 ? pick(1, 3) : pick(0, 3000);
      for (int k = 0; k < count; ++k) {
        PagedSeq s;
        s.row = row;
        s.n = kind == 0 ? pick(5, 300) : kind - 1;
        s.len = s.n + pick(0, 300);
        row += s.n;
        chunks += kind == 0;
        seqs.push_back(s);
      }
    }
    const int nseq = (int)seqs.size();
    long long sum = 0;
    for (auto &s : seqs) sum += (long long)paged_span(l, s).head * l.nkvh;
    const int total = (int)sum, active = total ? paged_active(l, total) : 0;
    for (int c = 0; c < active; ++c) {
      // where the share begins, as the kernels look for it
      const int lo = paged_cut(l, total, c);
      int seq = 0, begin = 0;
      while (begin + paged_span(l, seqs[seq]).head * l.nkvh <= lo) begin += paged_span(l, seqs[seq++]).head * l.nkvh;
      PagedWalk plain{seq, begin, lo, paged_cut(l, total, c + 1)}, fast = plain;
      int looked = 0, skips = 0, pieces = 0;
      auto counted = [&](int i) { return ++looked, seqs[i]; };
      auto skip = [&](int i) {
        ++skips;
        while (i < nseq && !paged_rows_fit(l, seqs[i].row, seqs[i].row + seqs[i].n)) ++i;
        return i;
      };
      while (true) {
        const PagedPiece p = paged_next(l, nseq, plain, [&](int i) { return seqs[i]; });
        const PagedPiece q = paged_next(l, nseq, fast, counted, skip);
        CHECK(p.seq == q.seq);
        if (p.seq < 0) break;
        ++pieces;
        CHECK(p.head == q.head && p.tile == q.tile && p.lo == q.lo && p.hi == q.hi && p.blocks == q.blocks && p.begin == q.begin && p.cost == q.cost);
      }
      CHECK(looked <= 2 * pieces + 2 * chunks + 2 && skips <= chunks + 1);
    }
  }
  printf("schedule ok\n");
  return 0;
}

// Walks random batches through the lines that a launch uses (paged_lines: its blocks, rows, overheads, smallest shares and scale),
// whole and split between the two kinds of work, and checks what the kernels rely on: every key block belongs to one CTA, every part
// of a unit knows where the others are, and no two units, groups or levels share a slot, a counter or a mark.
#include <cstdio>
#include <map>
#include <random>
#include <set>
#include <tuple>
#include <vector>

#include "../operators-rs_b200/csrc/paged_schedule.h"

using namespace ops;

static int round_no = 0;
#define CHECK(x)                                                         \
  do {                                                                   \
    if (!(x)) {                                                          \
      printf("round %d: %s failed (line %d)\n", round_no, #x, __LINE__); \
      return 1;                                                          \
    }                                                                    \
  } while (0)

// `line`: as the CTAs of a share of the SMs see it; `ctas`: what the scratch is laid out for
static int check(const PagedLine &line, int ctas, const std::vector<PagedSeq> &seqs, bool tiles) {
  const int nseq = (int)seqs.size();
  long long sum = 0;
  size_t want = 0;
  for (auto &s : seqs) {
    const PagedSpan p = paged_span(line, s);
    sum += (long long)p.head * line.nkvh;
    want += (size_t)p.tiles * line.nkvh;
  }
  CHECK(sum <= 0x7fffffff);
  const int total = (int)sum;
  if (total == 0) return 0;
  const int active = paged_active(line, total);
  CHECK(active >= 1 && active <= line.ctas && paged_cut(line, total, active) == total);
  typedef std::tuple<int, int, int> Unit;
  struct Part {
    int lo, hi, blocks, cta;
    PagedParts parts;
  };
  std::map<Unit, std::vector<Part>> units;
  int seq = 0, begin = 0;
  for (int c = 0; c < active; ++c) {
    const int lo = paged_cut(line, total, c), hi = paged_cut(line, total, c + 1);
    CHECK(lo < hi);
    while (begin + paged_span(line, seqs[seq]).head * line.nkvh <= lo) begin += paged_span(line, seqs[seq++]).head * line.nkvh;
    PagedWalk w{seq, begin, lo, hi};
    for (PagedPiece q = paged_next(line, nseq, w, [&](int i) { return seqs[i]; }); q.seq >= 0; q = paged_next(line, nseq, w, [&](int i) { return seqs[i]; }))
      units[Unit(q.seq, q.head, q.tile)].push_back({q.lo, q.hi, q.blocks, c, paged_parts(line, total, c, q)});
  }
  CHECK(units.size() == want);
  std::set<int> slots;     // parked parts and groups
  std::set<int> counters;  // words of `arrived`
  auto take = [](std::set<int> &from, int x, int most) { return x >= 0 && x < most && from.insert(x).second; };
  PagedLine laid = line;  // slots and counters go by the whole line
  laid.ctas = ctas;
  for (auto &u : units) {
    const std::vector<Part> &parts = u.second;
    const int n = (int)parts.size(), first = parts[0].cta;
    for (int k = 0, next = 0; k < n; ++k) {
      CHECK(parts[k].lo == next && parts[k].hi > next && parts[k].cta == first + k && parts[k].parts.first == first && parts[k].parts.count == n);
      next = parts[k].hi;
      if (k == n - 1) CHECK(next == parts[k].blocks);
      if (n > 1) CHECK(take(slots, paged_slot(first, k), 2 * ctas));
    }
    if (n == 1) continue;
    if (tiles) {
      if (n == 2) {
        for (int warp = 0; warp < 8; ++warp) CHECK(take(counters, first * 8 + warp, AP_LEVELS * ctas * 8));
      } else {
        CHECK(take(counters, (ctas + first) * 8, AP_LEVELS * ctas * 8));
        for (int k = 0; k < n; ++k) CHECK(take(counters, (ctas + first + k) * 8 + (k == n - 1 ? 2 : 1), AP_LEVELS * ctas * 8));
      }
      continue;
    }
    // parts in groups of AP_FEW_JOIN, the groups in turn
    int level = 0;
    std::vector<int> at;  // the slots of a level's nodes
    for (int k = 0; k < n; ++k) at.push_back(paged_slot(first, k));
    for (int one = 1; one < n; one *= AP_FEW_JOIN, ++level) {
      CHECK(level < AP_LEVELS);
      const int nodes = (int)at.size();
      std::vector<int> next;
      for (int g0 = 0; g0 < nodes; g0 += AP_FEW_JOIN) {
        const int together = std::min(AP_FEW_JOIN, nodes - g0);
        if (together == 1) {  // passed on where it is
          next.push_back(at[g0]);
          continue;
        }
        CHECK(take(counters, (level * ctas + first + g0 * one) * 8, AP_LEVELS * ctas * 8));
        for (int j = 0; j < together; ++j) CHECK(paged_group_slot(laid, first, (g0 + j) * one, std::min(one, n - (g0 + j) * one)) == at[g0 + j]);
        next.push_back(paged_group_slot(laid, first, g0 * one, together * one));
        if (nodes > AP_FEW_JOIN) CHECK(next.back() >= 2 * ctas && take(slots, next.back(), 3 * ctas));
      }
      at = next;
    }
    CHECK(at.size() == 1);
  }
  return 0;
}

int main() {
  // a sequence of more query rows than 31 bits count, one of them alone and behind a single token
  for (int n : {1 << 24, (1 << 24) + 1, 1 << 26})
    for (int past : {0, 1000}) {
      const PagedLines lines = paged_lines(148, 128, 1, true, 0xffffffffu, (size_t)n + 1, 2, (size_t)n + past);
      const std::vector<PagedSeq> seqs{{0, 1, 1}, {1, n, n + past}};
      CHECK(lines.fit && paged_span(lines.tile, seqs[1]).tiles == (n + lines.tile.tokens - 1) / lines.tile.tokens);
      CHECK(paged_rows_fit(lines.tile, 1, 1 + (uint32_t)n) && !paged_rows_fit(lines.tile, 1, 1));
    }
  std::mt19937 rng(11);
  auto pick = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
  for (round_no = 0; round_no < 1500; ++round_no) {
    const int group = std::vector<int>{1, 2, 3, 4, 7, 8, 16, 24, 128}[pick(0, 8)], nkvh = pick(1, 9);
    const bool causal = pick(0, 3) > 0;
    const int kind = pick(0, 4), nseq = round_no % 25 == 0 ? pick(1000, 2500) : pick(1, 40);
    std::vector<PagedSeq> seqs(nseq);
    int row = 0, longest = 0;
    const int past = std::vector<int>{40, 300, 5000, 60000}[round_no % 25 == 0 ? pick(0, 1) : pick(0, 3)];
    for (auto &s : seqs) {
      s.n = kind == 0 ? 1 : kind == 1 ? pick(0, 4) : kind == 2 ? pick(1, 700) : pick(0, 9) ? 1 : pick(0, 500);
      s.len = pick(0, 15) ? s.n + pick(0, past) : pick(0, 5);
      s.row = row;
      row += s.n;
      longest = std::max(longest, s.n);
    }
    const uint32_t max_seq = pick(0, 1) ? 0xffffffffu : (uint32_t)std::max(longest, 1);
    int slots = 0;
    for (auto &s : seqs) slots = std::max(slots, s.len);
    // a table wider than what is in use: the scale goes by what the host knows
    const size_t width = (size_t)slots << (pick(0, 3) ? 0 : pick(0, 20));
    const PagedLines lines = paged_lines(pick(0, 9) ? 148 : pick(1, 256), (size_t)group * nkvh, nkvh, causal, max_seq, (size_t)row, (size_t)nseq, std::min<size_t>(width, 1u << 30));
    for (int split = 0; split < 4; ++split) {
      PagedLine few = lines.few, tile = lines.tile;
      if (split && few.ctas > 1 && tile.ctas > 1) {
        few.ctas = paged_share(lines.few.ctas, pick(1, AP_SHARES * 3 / 4));
        tile.ctas = lines.tile.ctas - few.ctas;
        few.by_ctas = paged_div_by((uint32_t)few.ctas);
        tile.by_ctas = paged_div_by((uint32_t)tile.ctas);
      } else if (split) {
        break;
      }
      if (few.ctas && check(few, lines.few.ctas, seqs, false)) return 1;
      if (tile.ctas && check(tile, lines.tile.ctas, seqs, true)) return 1;
    }
    // every sequence with rows is on one of the lines
    for (auto &s : seqs) {
      const int on = (lines.few.ctas && paged_span(lines.few, s).tiles > 0) + (lines.tile.ctas && paged_span(lines.tile, s).tiles > 0);
      CHECK(on == (s.n > 0));
    }
  }
  printf("schedule ok\n");
  return 0;
}

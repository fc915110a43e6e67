// attention_paged_few.cuh — attention over a paged cache for sequences with a handful of query rows (a decode step, a few drafted
// tokens): at most 8 or 16 rows = new tokens x query heads per kv head.
//
//   o_r = sum_j 2^(x_rj - m_r) v_j / sum_j 2^(x_rj - m_r),  x_rj = scale log2(e) q_r . k_j,  one pass with a running m_r
//
// The work is reading K and V once, 4 dh bytes a key and kv head, HBM-bound.  The keys of all (sequence, kv head) pairs form one
// line of which every CTA, one per SM, takes an equal share (paged_schedule.h), so ragged lengths cost nothing.  What keeps the
// memory busy is bytes in flight: 6.4 TB/s at a loaded latency of about 3 us is 130 KB per SM, more than registers hold
// (with every lane's loads in registers, 64 KB a CTA and two CTAs an SM: 3.7 TB/s).  So pages stream by TMA into a ring of
// 32-key stages, 192 KB deep and on through the ends of pieces:
//
//   warps 0-3  consumers: S = Q K^T and O += P V for a stage's 32 keys on m16n8k16 warp MMAs (the rows are the 8 or 16 of the MMA;
//              a 128-row tcgen05 tile has nothing to chew on here), both operands by ldmatrix from the 128-byte-swizzled stage,
//              the probabilities straight from the S registers: about 1400 clocks a stage, four stages at a time.  They round to
//              the element type there, as the warp MMA wants (half a step each, at random over the keys: against 64 bits the output
//              is off by at most 1.3 times what its own rounding is off by); the sums that they are divided by do not
//   warps 4-7  producers, every fourth stage each (the boxes of one warp alone come to 3.4 TB/s): a lane per box of a stage
//              (32 / min(page, 32) boxes of K and of V), pages looked up a stage ahead
//   warp 8     scheduler: finds the CTA's share, posts its pieces ahead
//
// A long piece's stages go to the consumers in turn; at its end the four meet in shared memory, and the CTA that comes last to a
// unit that several share joins its parts.  Meeting takes some 3000 clocks, more than the stages of a short sequence: a piece that
// takes up half of the ring at most, is all of its unit and has more behind it goes to one consumer, who meets nobody, and the
// four work on four pieces (2048 single tokens over 100 keys each: 116 us against 133; at the end of a share, where the
// others would have nothing, together).
//
// A box behind the sequence's end, or of a page that is not there, is asked for outside the map and arrives as zeros; the slots
// behind the end inside the last page are zeroed in the stage by the warp that takes it (a zero probability does not hide a
// NaN there).  Every wait is bounded; when one runs out its code goes to the status word and all roles unwind.
// Measured, 8 kv heads of 128: 61 requests over up to 4096 keys 98 us, 5.9 TB/s; eight over up to 32101 keys 106 us, 6.1 TB/s;
// one over 1001 keys 9.9 us.
#pragma once
#include "attention_paged.h"
#include "device_utils.cuh"
#include "sm100_ptx.cuh"

namespace ops {

using namespace sm100;

constexpr int FEW_CONSUMERS = 4, FEW_PRODUCERS = 4, FEW_THREADS = (FEW_CONSUMERS + FEW_PRODUCERS + 1) * 32;
constexpr int FEW_KEYS = 32;  // of a stage
constexpr int FEW_RING = 4;   // pieces posted ahead
static_assert(FEW_KEYS == AP_FEW_BLOCK, "a block is a stage");

// d += a . b, one warp, m16n8k16, f32 accumulate
template <bool BF>
__device__ __forceinline__ void few_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

// A piece as the scheduler posts it.
struct FewPiece {
  int seq;  // -1: no more
  int row, n, len, head;
  int k0, k1;  // keys
  int first, count;  // CTAs that have parts of the unit; 1: this is all of it
  int whose;         // consumer that does all of it; -1: the four together
};

template <int DH, int NR> struct FewSmem {
  static constexpr int ROWS = NR * 8;
  static constexpr int HALVES = DH / 64;
  static constexpr int OPERAND = FEW_KEYS * DH * 2;  // K or V of a stage: [half][32 keys][128 B], swizzled
  // a multiple of the producers, so that a slot of the ring is always the same one's
  static constexpr int STAGES = DH == 64 ? 24 : NR == 1 ? 12 : 8;
  static constexpr int Q_LD = DH + 8;  // elements; rows fall on other banks
  static constexpr int O_LD = DH + 4;
  static constexpr int OFF_RING = 0;
  static constexpr int OFF_Q = OFF_RING + STAGES * 2 * OPERAND;                 // [piece of the ring][ROWS][Q_LD] 16-bit
  static constexpr int OFF_O = OFF_Q + FEW_RING * ROWS * Q_LD * 2;              // [consumers][ROWS][O_LD] f32
  static constexpr int OFF_ML = OFF_O + FEW_CONSUMERS * ROWS * O_LD * 4;        // [ROWS][consumers] (m, l)
  static constexpr int OFF_PIECES = OFF_ML + ROWS * FEW_CONSUMERS * 8;
  static constexpr int BYTES = OFF_PIECES + FEW_RING * (int)sizeof(FewPiece) + 1024;  // 1024: alignment
  static constexpr int NUM_BARS = 2 * STAGES + 3 * FEW_RING + 1;
  static_assert(STAGES % FEW_PRODUCERS == 0 && OFF_O % 16 == 0, "layout");
};

// What lies outside the dynamic shared memory, which the tiles of the same launch use after it.
template <int DH, int NR> struct FewShared {
  unsigned long long bars[FewSmem<DH, NR>::NUM_BARS];
  uint32_t issued[FewSmem<DH, NR>::STAGES];  // number of the stage that was last asked for in a slot of the ring, plus 1
  int last;
};

// A slot of the ring is not always the same consumer's: one that came early could take the phase before last of its barrier for the
// one it wants.  So it waits for the barrier only once its stage has been asked for, which is when the one before has been used up.
__device__ __forceinline__ bool few_wait_issued(const volatile uint32_t *issued, uint32_t stage, int *status, int code) {
  if (*issued == stage) return true;
  const unsigned long long t0 = globaltimer_ns();
  while (true) {
#pragma unroll 1
    for (int i = 0; i < 256; ++i)
      if (*issued == stage) return true;
    if (globaltimer_ns() - t0 > WAIT_LIMIT_NS) {
      atomicCAS(status, 0, code);
      return false;
    }
  }
}

template <int DH, int NR> __device__ __forceinline__ void few_init(FewShared<DH, NR> &sh) {  // one thread
  constexpr int ST = FewSmem<DH, NR>::STAGES;
  const uint32_t bar0 = smem_u32(sh.bars);
  for (int i = 0; i < 2 * ST + 2 * FEW_RING; ++i) mbar_init(bar0 + 8u * i, 1);  // full, empty, q_full, piece_full
  for (int i = 0; i < FEW_RING; ++i) mbar_init(bar0 + 8u * (2 * ST + 2 * FEW_RING + i), FEW_CONSUMERS + FEW_PRODUCERS);  // piece_empty
  mbar_init(bar0 + 8u * (2 * ST + 3 * FEW_RING), FEW_CONSUMERS);  // meet_bar
  for (int s = 0; s < ST; ++s) sh.issued[s] = 0;
}

// The CTA's share of the line of few rows.  Whether no wait ran out.
template <int DH, bool BF, int NR>
__device__ __forceinline__ bool few_rows(const CUtensorMap &tmap_k, const CUtensorMap &tmap_v, const PagedAttnArgs &a, uint8_t *base_ptr, FewShared<DH, NR> &sh,
                                         const PagedShare &share) {
  typedef FewSmem<DH, NR> Smem;
  constexpr int ST = Smem::STAGES, ROWS = Smem::ROWS;
  const uint32_t base = smem_u32(base_ptr), bar0 = smem_u32(sh.bars);
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (ST + s); };
  auto q_full = [&](int i) { return bar0 + 8u * (2 * ST + i); };
  auto piece_full = [&](int i) { return bar0 + 8u * (2 * ST + FEW_RING + i); };
  auto piece_empty = [&](int i) { return bar0 + 8u * (2 * ST + 2 * FEW_RING + i); };  // read, by the consumers with its q
  const uint32_t meet_bar = bar0 + 8u * (2 * ST + 3 * FEW_RING);
  volatile uint32_t *issued = sh.issued;
  volatile FewPiece *pieces = reinterpret_cast<volatile FewPiece *>(base_ptr + Smem::OFF_PIECES);
  const PagedLine &line = a.few.line;  // `line.ctas`: what the scratch is laid out for
  int *status = a.batch.status + 1;    // of the waits
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int group = line.group, cta = share.cta;

  bool ok = true;
  if (warp == FEW_CONSUMERS + FEW_PRODUCERS) {
    // ------------------------------------------------------------------ scheduler
    if (lane == 0) {
      const PagedLine shared = paged_shared_line(line, share);
      const int total = share.total;
      PagedWalk walk = share.walk;
      uint32_t alone = 0;  // pieces given to one consumer
#pragma unroll 1
      for (uint32_t i = 0; ok; ++i) {
        const PagedPiece q = paged_step(a.batch, shared, walk);
        const int slot = i % FEW_RING;
        if (!(ok = mbar_wait(piece_empty(slot), ((i / FEW_RING) & 1u) ^ 1u, status, 201))) break;
        volatile FewPiece &to = pieces[slot];
        to.seq = q.seq;
        if (q.seq >= 0) {
          to.row = q.s.row;
          to.n = q.s.n;
          to.len = q.s.len;
          to.head = q.head;
          to.k0 = q.lo * FEW_KEYS;
          to.k1 = min(q.hi * FEW_KEYS, q.s.len);
          const PagedParts parts = paged_parts(shared, total, cta, q);
          to.first = parts.first;
          to.count = parts.count;
          to.whose = parts.count == 1 && q.hi <= ST / 2 && walk.end - walk.at >= 2 * q.cost ? (int)(alone++ % FEW_CONSUMERS) : -1;
        }
        mbar_arrive(piece_full(slot));
        if (q.seq < 0) break;
      }
    }
  } else if (warp >= FEW_CONSUMERS && warp < FEW_CONSUMERS + FEW_PRODUCERS) {
    // ------------------------------------------------------------------ producers
    const int producer = warp - FEW_CONSUMERS;
    const int box = 1 << a.few.box_log2, boxes = FEW_KEYS >> a.few.box_log2;  // of K; as many of V
    const int lg = a.batch.page_log2, in_page = (1 << lg) - 1;
    const bool values = lane >= boxes;
    const int r = (values ? lane - boxes : lane) * box;  // the lane's first row of a stage
    const bool mine = lane < 2 * boxes;
    uint32_t count = 0;
#pragma unroll 1
    for (uint32_t i = 0; ok; ++i) {
      const int slot = i % FEW_RING;
      if (!(ok = __all_sync(0xffffffffu, mbar_wait(piece_full(slot), (i / FEW_RING) & 1u, status, 202)))) break;
      volatile FewPiece &p = pieces[slot];
      const int seq = p.seq, row = p.row, n = p.n, head = p.head, k0 = p.k0, k1 = p.k1;
      __syncwarp();
      if (lane == 0) mbar_arrive(piece_empty(slot));
      if (seq < 0) break;
      const uint32_t *table = a.batch.table + (long long)seq * a.batch.table_ld;
      // the page of this lane's box of the stage at key k, outside the map where there is nothing to read
      auto look_up = [&](int k) -> int {
        const int key = k + r;
        if (!mine || key >= k1) return (int)a.batch.npages;
        const uint32_t page = table[key >> lg];
        if (page < a.batch.npages) return (int)page;
        atomicCAS(a.batch.status, 0, OPS_PAGED_BAD_PAGE);
        return (int)a.batch.npages;
      };
      const uint32_t stages = k1 > k0 ? (uint32_t)(k1 - k0 + FEW_KEYS - 1) / FEW_KEYS : 0u;
      uint32_t st = ((uint32_t)producer - count) % FEW_PRODUCERS;
      int page = look_up(k0 + (int)st * FEW_KEYS);
      // the piece's q rows, zeros behind them: read now by the first producer, written once its first stage is asked for
      constexpr int Q_VECS = ROWS * DH / 8 / 32;  // 16-byte pieces a lane
      uint4 qv[Q_VECS];
      bool q_due = producer == 0;
      if (q_due) {
#pragma unroll
        for (int e = 0; e < Q_VECS; ++e) {
          const int at = e * 32 + lane, qr = at / (DH / 8), col = (at - qr * (DH / 8)) * 8;
          const int tok = paged_div(qr, line.by_group), gi = qr - tok * group;
          qv[e] = make_uint4(0, 0, 0, 0);
          if (tok < n && col < a.dh) qv[e] = ld_global_16(a.q + (long long)(row + tok) * a.q_t + (long long)(head * group + gi) * a.q_h + col * 2);
        }
      }
#pragma unroll 1
      while (ok && (st < stages || q_due)) {
        if (st < stages) {
          const uint32_t at = count + st;
          const int s = at % ST, k = k0 + (int)st * FEW_KEYS;
          if (lane == 0) {
            ok = mbar_wait(empty(s), ((at / ST) & 1u) ^ 1u, status, 204);
            if (ok) mbar_arrive_expect_tx(full(s), 2 * Smem::OPERAND);
            if (ok) issued[s] = at + 1;
          }
          ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0);
          if (!ok) break;
          if (mine) {
            const uint32_t to = base + Smem::OFF_RING + s * (2 * Smem::OPERAND) + (values ? Smem::OPERAND : 0) + r * 128;
            const int slot_in_page = (k + r) & in_page;
#pragma unroll
            for (int h = 0; h < Smem::HALVES; ++h)
              tma_load_4d(to + h * (FEW_KEYS * 128), values ? &tmap_v : &tmap_k, full(s), h * 64, slot_in_page, head, page);
          }
          st += FEW_PRODUCERS;
          page = look_up(k0 + (int)st * FEW_KEYS);
        }
        if (q_due) {
          q_due = false;
          // (the consumers have read what was there: this piece would not have been posted otherwise)
#pragma unroll
          for (int e = 0; e < Q_VECS; ++e) {
            const int at = e * 32 + lane, qr = at / (DH / 8), col = (at - qr * (DH / 8)) * 8;
            *reinterpret_cast<uint4 *>(base_ptr + Smem::OFF_Q + ((slot * ROWS + qr) * Smem::Q_LD + col) * 2) = qv[e];
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(q_full(slot));
        }
      }
      count += stages;
    }
  } else if (warp < FEW_CONSUMERS) {
    // ------------------------------------------------------------------ consumers
    const int g = lane >> 2, c = lane & 3;
    // ldmatrix: lane l names row l % 8 of matrix l / 8
    const int mi = lane >> 3, mr = lane & 7;
    uint32_t count = 0, met = 0;  // stages of the pieces so far; meetings
    auto meet = [&]() -> bool {
      __syncwarp();
      if (lane == 0) mbar_arrive(meet_bar);
      return __all_sync(0xffffffffu, mbar_wait(meet_bar, met++ & 1u, status, 210));
    };
#pragma unroll 1
    for (uint32_t i = 0; ok; ++i) {
      const int slot = i % FEW_RING;
      if (!(ok = __all_sync(0xffffffffu, mbar_wait(piece_full(slot), (i / FEW_RING) & 1u, status, 211)))) break;
      volatile FewPiece &p = pieces[slot];
      const int seq = p.seq, row = p.row, n = p.n, len = p.len, head = p.head, k0 = p.k0, k1 = p.k1, first = p.first, parts = p.count, whose = p.whose;
      if (seq < 0) break;
      const int rows = n * group;
      const uint32_t stages = k1 > k0 ? (uint32_t)(k1 - k0 + FEW_KEYS - 1) / FEW_KEYS : 0u;
      const bool mine = whose < 0 || whose == warp;
      uint32_t q[DH / 16][4];
      if (mine) {
        if (!(ok = __all_sync(0xffffffffu, mbar_wait(q_full(slot), (i / FEW_RING) & 1u, status, 212)))) break;
        const uint32_t q_at = base + Smem::OFF_Q + slot * ROWS * Smem::Q_LD * 2;
        if (NR == 2) {
#pragma unroll
          for (int ks = 0; ks < DH / 16; ++ks)  // rows 0-7 | 8-15 of k 0-7, then of k 8-15
            ldsm(q_at + (((mi & 1) * 8 + mr) * Smem::Q_LD + ks * 16 + (mi >> 1) * 8) * 2, q[ks]);
        } else {
#pragma unroll
          for (int ks = 0; ks < DH / 16; ks += 2) {  // k 0-7 | 8-15 of two steps; there are no rows 8-15
            uint32_t two[4];
            ldsm(q_at + (mr * Smem::Q_LD + ks * 16 + mi * 8) * 2, two);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              q[ks + e][0] = two[e * 2];
              q[ks + e][2] = two[e * 2 + 1];
              q[ks + e][1] = q[ks + e][3] = 0;
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(piece_empty(slot));
      if (!mine) {
        count += stages;
        continue;
      }
      // last visible key of rows g and g + 8; every row sees the keys in front of `all`
      int lim[NR];
#pragma unroll
      for (int e = 0; e < NR; ++e) lim[e] = line.causal ? len - n + paged_div(g + 8 * e, line.by_group) : len - 1;
      const int all = min(k1, line.causal ? len - n + 1 : len);
      float m[NR], l[NR];  // m is common to the four lanes of a row, l is this lane's share
#pragma unroll
      for (int e = 0; e < NR; ++e) {
        m[e] = -INFINITY;
        l[e] = 0.f;
      }
      float o[DH / 8][4];
#pragma unroll
      for (int j = 0; j < DH / 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][e] = 0.f;

      const uint32_t step = whose < 0 ? FEW_CONSUMERS : 1;
#pragma unroll 1
      for (uint32_t st = whose < 0 ? ((uint32_t)warp - count) % FEW_CONSUMERS : 0u; st < stages; st += step) {
        const uint32_t at = count + st;
        const int s = at % ST, kb = k0 + (int)st * FEW_KEYS;
        if (!(ok = __all_sync(0xffffffffu, few_wait_issued(issued + s, at + 1, status, 214)))) break;
        if (!(ok = __all_sync(0xffffffffu, mbar_wait(full(s), (at / ST) & 1u, status, 213)))) break;
        const uint32_t ks_base = base + Smem::OFF_RING + s * (2 * Smem::OPERAND), vs_base = ks_base + Smem::OPERAND;
        if (kb + FEW_KEYS > len) {  // behind the end: may hold anything, a NaN too
          uint8_t *v = base_ptr + Smem::OFF_RING + s * (2 * Smem::OPERAND) + Smem::OPERAND;
          for (int e = lane; e < (kb + FEW_KEYS - len) * Smem::HALVES * 8; e += 32) {
            const int r = len - kb + e / (Smem::HALVES * 8), piece = e % (Smem::HALVES * 8);
            *reinterpret_cast<uint4 *>(v + (piece >> 3) * (FEW_KEYS * 128) + r * 128 + (piece & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async();  // the stage's next load writes through the async proxy
          __syncwarp();
        }
        float x[4][4];  // [8 keys][row g: keys 2c, 2c+1 | row g+8]
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[j][e] = 0.f;
#pragma unroll
        for (int ks = 0; ks < DH / 16; ++ks)
#pragma unroll
          for (int np = 0; np < 2; ++np) {  // 16 keys: matrices (keys 0-7, k 0-7), (0-7, 8-15), (8-15, 0-7), (8-15, 8-15)
            uint32_t b[4];
            const int key = np * 16 + (mi >> 1) * 8 + mr, chunk = ks * 2 + (mi & 1);
            ldsm(ks_base + (chunk >> 3) * (FEW_KEYS * 128) + key * 128 + (((chunk & 7) ^ mr) << 4), b);
            few_mma<BF>(x[np * 2], q[ks], b[0], b[1]);
            few_mma<BF>(x[np * 2 + 1], q[ks], b[2], b[3]);
          }
        uint32_t pa[2][4];  // the probabilities as the second product's A: 16 keys each
        if (NR == 1) pa[0][1] = pa[0][3] = pa[1][1] = pa[1][3] = 0;
        float al[NR];
#pragma unroll
        for (int e = 0; e < NR; ++e) {
          float mx = -INFINITY;
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              float &v = x[j][e * 2 + w];
              v *= a.scale_log2;
              if (kb + FEW_KEYS > all && kb + j * 8 + 2 * c + w > min(lim[e], k1 - 1)) v = -INFINITY;
              mx = fmaxf(mx, v);
            }
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const float m_new = fmaxf(m[e], mx);
          const float m_use = m_new == -INFINITY ? 0.f : m_new;
          al[e] = ap_ex2(m[e] - m_use);
          float sum = 0.f;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float p0 = ap_ex2(x[j][e * 2] - m_use), p1 = ap_ex2(x[j][e * 2 + 1] - m_use);
            sum += p0 + p1;
            pa[j >> 1][(j & 1) * 2 + e] = ap_pack<BF>(p0, p1);
          }
          l[e] = fmaf(l[e], al[e], sum);
          m[e] = m_new;
        }
        if (__any_sync(0xffffffffu, al[0] != 1.f || al[NR - 1] != 1.f)) {
#pragma unroll
          for (int j = 0; j < DH / 8; ++j)
#pragma unroll
            for (int e = 0; e < 2 * NR; ++e) o[j][e] *= al[e >> 1];
        }
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int np = 0; np < DH / 16; ++np) {  // 16 columns: matrices (keys 0-7, columns 0-7), (8-15, 0-7), (0-7, 8-15), (8-15, 8-15)
            uint32_t b[4];
            const int key = kt * 16 + (mi & 1) * 8 + mr, chunk = np * 2 + (mi >> 1);
            ldsm_t(vs_base + (chunk >> 3) * (FEW_KEYS * 128) + key * 128 + (((chunk & 7) ^ mr) << 4), b);
            few_mma<BF>(o[np * 2], pa[kt], b[0], b[1]);
            few_mma<BF>(o[np * 2 + 1], pa[kt], b[2], b[3]);
          }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty(s));
      }
      if (!ok) break;
      count += stages;

#pragma unroll
      for (int e = 0; e < NR; ++e) {
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
      }
      auto out_row = [&](int r) -> char * {
        const int tok = paged_div(r, line.by_group), gi = r - tok * group;
        return a.o + (long long)(row + tok) * a.o_t + (long long)(head * group + gi) * a.o_h;
      };
      if (whose >= 0) {  // nobody to wait for
#pragma unroll
        for (int e = 0; e < NR; ++e) {
          if (g + 8 * e >= rows) continue;
          const float inv = l[e] > 0.f ? 1.f / l[e] : 0.f;  // a row that sees nothing: zeros
          char *to = out_row(g + 8 * e);
#pragma unroll
          for (int j = 0; j < DH / 8; ++j)
            if (j * 8 < a.dh) *reinterpret_cast<uint32_t *>(to + (j * 8 + 2 * c) * 2) = ap_pack<BF>(o[j][e * 2] * inv, o[j][e * 2 + 1] * inv);
        }
        continue;
      }

      // the four warps meet: each leaves its m, l and o, and the threads that finish an output weigh them
      float2 *ml_s = reinterpret_cast<float2 *>(base_ptr + Smem::OFF_ML);
      float *o_s = reinterpret_cast<float *>(base_ptr + Smem::OFF_O);
#pragma unroll
      for (int e = 0; e < NR; ++e) {
        if (c == 0) ml_s[(g + 8 * e) * FEW_CONSUMERS + warp] = make_float2(m[e], l[e]);
        if (g + 8 * e < rows)
#pragma unroll
          for (int j = 0; j < DH / 8; ++j)
            *reinterpret_cast<float2 *>(o_s + (warp * ROWS + g + 8 * e) * Smem::O_LD + j * 8 + 2 * c) = make_float2(o[j][e * 2], o[j][e * 2 + 1]);
      }
      if (!(ok = meet())) break;
      // outputs by thread: 4 columns of a row, all of which go through f(row, column)
      auto each = [&](auto &&f) {
#pragma unroll 1
        for (int at = threadIdx.x; at < rows * (DH / 4); at += FEW_CONSUMERS * 32) {
          const int r = at / (DH / 4), col = (at - r * (DH / 4)) * 4;
          if (col < a.dh) f(r, col);
        }
      };
      // divided and written, or parked in a slot
      auto leave = [&](int slot, int r, int col, float4 acc, float top, float den) {
        if (slot < 0) {
          const float inv = den > 0.f ? 1.f / den : 0.f;  // a row that sees nothing: zeros
          *reinterpret_cast<uint2 *>(out_row(r) + col * 2) = make_uint2(ap_pack<BF>(acc.x * inv, acc.y * inv), ap_pack<BF>(acc.z * inv, acc.w * inv));
        } else {
          const long long at = (long long)slot * ROWS + r;
          *reinterpret_cast<float4 *>(a.few.parts + at * DH + col) = acc;
          if (col == 0) a.few.parts_ml[at] = make_float2(top, den);
        }
      };
      int node = cta - first;
      each([&](int r, int col) {
        float2 ml[FEW_CONSUMERS];
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < FEW_CONSUMERS; ++w) {
          ml[w] = ml_s[r * FEW_CONSUMERS + w];
          top = fmaxf(top, ml[w].x);
        }
        const float ref = top == -INFINITY ? 0.f : top;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float den = 0.f;
#pragma unroll
        for (int w = 0; w < FEW_CONSUMERS; ++w) {
          const float4 v = *reinterpret_cast<const float4 *>(o_s + (w * ROWS + r) * Smem::O_LD + col);
          const float weight = ap_ex2(ml[w].x - ref);  // a warp without a key in sight: 0, of zeros
          acc.x = fmaf(v.x, weight, acc.x);
          acc.y = fmaf(v.y, weight, acc.y);
          acc.z = fmaf(v.z, weight, acc.z);
          acc.w = fmaf(v.w, weight, acc.w);
          den = fmaf(ml[w].y, weight, den);
        }
        leave(parts == 1 ? -1 : paged_slot(first, node), r, col, acc, top, den);
      });
      // Other CTAs have the other parts: the last of 16 neighbours joins theirs, the last of up to 16 such groups those.
      int nodes = parts, span = 1;  // of the level of the tree: nodes, parts of one
#pragma unroll 1
      for (int level = 0; nodes > 1 && ok; ++level) {
        const int g0 = node & ~(AP_FEW_JOIN - 1), together = min(AP_FEW_JOIN, nodes - g0);
        const int one = span;  // parts of a node
        node /= AP_FEW_JOIN;
        nodes = (nodes + AP_FEW_JOIN - 1) / AP_FEW_JOIN;
        span *= AP_FEW_JOIN;
        if (together == 1) continue;  // as it was parked (it has neither a counter nor a slot: paged_group_slot)
        if (!(ok = meet())) break;    // all have parked
        if (warp == 0) {
          pdl_wait_for_front();  // the counters have been cleared
          const bool last = paged_arrive_last(a.few.arrived + (level * line.ctas + first + g0 * one) * 8, together);
          if (lane == 0) *const_cast<volatile int *>(&sh.last) = last;
        }
        if (!(ok = meet())) break;
        if (!*const_cast<volatile int *>(&sh.last)) break;
        __threadfence();
        each([&](int r, int col) {
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
          float top = -INFINITY, den = 0.f;
          constexpr int DEEP = 8;
#pragma unroll 1
          for (int j0 = 0; j0 < together; j0 += DEEP) {
            float4 v[DEEP];
            float2 ml[DEEP];
#pragma unroll
            for (int e = 0; e < DEEP; ++e) {
              v[e] = make_float4(0.f, 0.f, 0.f, 0.f);
              ml[e] = make_float2(-INFINITY, 0.f);
              if (j0 + e < together) {
                const int k = (g0 + j0 + e) * one;
                const long long from = (long long)paged_group_slot(line, first, k, min(one, parts - k)) * ROWS + r;
                ml[e] = __ldcg(a.few.parts_ml + from);
                v[e] = __ldcg(reinterpret_cast<const float4 *>(a.few.parts + from * DH + col));
              }
            }
#pragma unroll
            for (int e = 0; e < DEEP; ++e) {
              const float next = fmaxf(top, ml[e].x), ref = next == -INFINITY ? 0.f : next;
              const float wa = ap_ex2(top - ref), wb = ap_ex2(ml[e].x - ref);
              den = den * wa + ml[e].y * wb;
              acc.x = acc.x * wa + v[e].x * wb;
              acc.y = acc.y * wa + v[e].y * wb;
              acc.z = acc.z * wa + v[e].z * wb;
              acc.w = acc.w * wa + v[e].w * wb;
              top = next;
            }
          }
          leave(nodes == 1 ? -1 : paged_group_slot(line, first, g0 * one, together * one), r, col, acc, top, den);
        });
      }
      if (!ok) break;
      if (!(ok = meet())) break;  // ml_s and o_s are free again
    }
  }
  return ok;
}

}  // namespace ops

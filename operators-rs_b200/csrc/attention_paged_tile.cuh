// attention_paged_tile.cuh — attention over a paged cache for sequences with more query rows than attention_paged_few.cuh takes: chunks
// of a prompt, whole prompts, many query heads per kv head.
//
//   o_r = sum_j 2^(x_rj - m_r) v_j / sum_j 2^(x_rj - m_r),  x_rj = scale log2(e) q_r . k_j,  one pass with a running m_r
//
// Tensor-bound: 4 dh flops a (query head, key) pair against 4 dh bytes a key that 256 query rows share.  The two products run on
// tcgen05 with S, P and O in tensor memory, as in attention_fused.cu's two-tile kernel, whose arithmetic this one shares: a unit
// is TWO tiles of 128 query rows, so that the tensor pipe runs one tile's products while the other tile's exponentials are in
// flight; the reference point m follows the row maximum only when that has moved by 2^8 (lazy rescaling; the
// factor cancels in o / l; the probabilities stay below 256, exact to half a step in the 16-bit operand that the second product
// takes).  What a paged batch of ragged chunks changes:
//   - A thread per row, a warp of each tile on every scheduler: a whole row's maximum needs no meeting of threads, and the first
//     half of a block's probabilities feeds the second product while the other half's powers are taken.
//   - A tile's rows are tokens x query heads of one kv head, token by token: a chunk of 33 tokens fills its rows whatever its
//     length, and the heads of a group share every K and V block in shared memory.
//   - K and V come page by page: a block of 128 keys is 128 / min(page, 64) boxes of a 4-d tensor map over the whole cache, each
//     issued by its own lane, which has looked its page up a block ahead.  A box behind the sequence's end, or of a page that is
//     not there, is asked for outside the map and arrives as zeros; the slots behind the end inside the last page are zeroed in
//     shared memory (a zero probability does not hide a NaN there).
//   - What several CTAs share of a unit is joined inside the launch (a kernel of its own for it took 13 us of a 4096-token prompt's
//     141): two parts by the last warp to come, more by all their CTAs' warps together.
//   - One persistent CTA per SM takes an equal share of the line of all units' keys (paged_schedule.h): ragged chunks, one long
//     chunk and few heads over a long past are all the same to it.  The pieces of its share follow each other without a
//     pause: the scheduler warp posts them ahead, K, V and Q of the next piece load and its first scores run while the softmax
//     warps still write out the one before.
//
//   warp 0   Q and K producer        warps 4-7    softmax of tile 0, a row a thread
//   warp 1   tcgen05.mma issuer      warps 8-11   softmax of tile 1
//   warp 2   V producer; zeroes what lies behind the end of a sequence in its last block (within the time that the block in
//            front takes the tensor pipe: the next stage is not free earlier)
//   warp 3   scheduler
// Every wait is bounded; when one runs out its code goes to the status word and all roles unwind to the common teardown.
// Measured, heads of 128: a 4096-token prompt of 32 heads 132 us, 1.04 PFLOP/s, the tensor pipe and the special-function unit at 55 %
// of their cycles each (a block's two products and its powers take turns less than perfectly; a polynomial for 1 in 8, 4, 3 or 2
// powers: 141, 148, 147, 176 us; scores made and used 64 keys at a time, so that nothing waits for a whole block's: 136 us, the two
// tiles' powers then coincide); 1024 tokens of 4 heads over 8025 keys 35 us, of which some 5 are spent until the first scores and
// 8 on parking and joining.
#pragma once
#include "attention_paged.h"
#include "device_utils.cuh"
#include "sm100_ptx.cuh"

namespace ops {

using namespace sm100;

constexpr int TL_THREADS = 384;
constexpr int TL_ROWS = 128;  // of a tile
constexpr int TL_KEYS = AP_TILE_BLOCK;
constexpr int TL_RING = 4;    // pieces posted ahead
constexpr int TL_READERS = 11;  // warps that read the ring: all but the scheduler

// A piece as the scheduler posts it.
struct TilePiece {
  int valid;
  int row;        // of the step: first token of the unit
  int tokens;     // of the sequence from there on
  int off;        // causal token x of the unit sees slots <= off + x
  int len, seq, head;
  int lo, hi;     // key blocks of the unit that this CTA walks
  int blocks[2];  // ... of each tile, counted from lo
  int clean;      // local block whose V rows from len on are zeroed; -1: none
  int first, count;  // CTAs that have parts of the unit; 1: this is all of it
};

template <int DH> struct TileSmem {
  static constexpr int HALVES = DH / 64;
  static constexpr int STAGES = DH == 64 ? 4 : 2;
  static constexpr int TILE = TL_ROWS * DH * 2;  // a Q tile, a K block or a V block
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_K = OFF_Q + 2 * TILE;
  static constexpr int OFF_V = OFF_K + STAGES * TILE;
  static constexpr int NUM_BARS = 12 + 2 * TL_RING + 5 * STAGES;
  static constexpr int OFF_RING = OFF_V + STAGES * TILE;
  static constexpr int OFF_STAGE = (OFF_RING + TL_RING * (int)sizeof(TilePiece) + 15) / 16 * 16;  // 4 KB a softmax warp: 32 rows x 128 B
  static constexpr int BYTES = OFF_STAGE + 8 * 4096 + 1024;  // 1024: alignment
};

// A unit of more than two parts, one of them this CTA's, as the scheduler notes it for the end of the share.
struct TileHelp {
  int first, count;        // CTAs; count <= 2: none
  int row, tokens, head;
};

// What lies outside the dynamic shared memory.
template <int DH> struct TileShared {
  unsigned long long bars[TileSmem<DH>::NUM_BARS];
  TileHelp help[2];        // the unit that the share begins in, the one it ends in
  uint32_t tickets[2][8];  // of the softmax warps for these: what paged_arrive said
  uint32_t tmem;           // address
};

__device__ __forceinline__ float tl_max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

template <int DH> __device__ __forceinline__ void tile_init(TileShared<DH> &sh) {  // one thread
  constexpr int ST = TileSmem<DH>::STAGES;
  const uint32_t bar0 = smem_u32(sh.bars);
  for (int i = 0; i < TileSmem<DH>::NUM_BARS; ++i) {
    const bool p_full = i >= 6 && i < 10, ring_empty = i >= 12 + TL_RING && i < 12 + 2 * TL_RING;
    mbar_init(bar0 + 8u * i, p_full ? 4 : ring_empty ? TL_READERS : 1);
  }
  static_assert(TileSmem<DH>::NUM_BARS == 12 + 2 * TL_RING + 5 * ST, "the barriers that tiles() names");
  sh.help[0].count = sh.help[1].count = 0;
}

// The CTA's share of the line of tiles.  Whether no wait ran out.
template <int DH, bool BF>
__device__ __forceinline__ bool tiles(const CUtensorMap &tmap_q, const CUtensorMap &tmap_k, const CUtensorMap &tmap_v, const PagedAttnArgs &a, uint8_t *base_ptr,
                                      TileShared<DH> &sh, const PagedShare &share) {
  typedef TileSmem<DH> Smem;
  constexpr int HALVES = Smem::HALVES, ST = Smem::STAGES, TILE = Smem::TILE;
  const uint32_t base = smem_u32(base_ptr), bar0 = smem_u32(sh.bars);
  auto q_full = [&](int t) { return bar0 + 8u * (0 + t); };
  auto q_empty = [&](int t) { return bar0 + 8u * (2 + t); };    // last QK of the piece's tile done
  auto s_full = [&](int t) { return bar0 + 8u * (4 + t); };     // S complete (tensor pipe -> softmax)
  auto p_full = [&](int t, int h) { return bar0 + 8u * (6 + 2 * t + h); };  // P of the h-th 64 keys written (softmax -> issuer)
  auto o_final = [&](int t) { return bar0 + 8u * (10 + t); };   // last PV of the piece's tile done (tensor pipe -> softmax)
  auto ring_full = [&](int i) { return bar0 + 8u * (12 + i); };
  auto ring_empty = [&](int i) { return bar0 + 8u * (12 + TL_RING + i); };
  auto k_full = [&](int s) { return bar0 + 8u * (12 + 2 * TL_RING + s); };
  auto k_empty = [&](int s) { return bar0 + 8u * (12 + 2 * TL_RING + ST + s); };
  auto v_full = [&](int s) { return bar0 + 8u * (12 + 2 * TL_RING + 2 * ST + s); };
  auto v_empty = [&](int s) { return bar0 + 8u * (12 + 2 * TL_RING + 3 * ST + s); };
  auto v_clean = [&](int s) { return bar0 + 8u * (12 + 2 * TL_RING + 4 * ST + s); };  // a stage's, so that no phase is overrun
  volatile TilePiece *ring = reinterpret_cast<volatile TilePiece *>(base_ptr + Smem::OFF_RING);
  volatile TileHelp *help = sh.help;

  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;  // known to be uniform
  const PagedBatch &batch = a.batch;
  const PagedLine &line = a.tile.line;  // `line.ctas`: what the scratch is laid out for
  const int group = line.group;
  int *status = batch.status + 1;  // of the waits
  const uint32_t tmem_base = sh.tmem;
  bool ok = true;
  // tensor memory columns: S0 | S1 | O0 | O1, 128 each; the P of a tile overwrites the first 64 columns of its S
  auto s_col = [&](int t) { return (uint32_t)(t * 128); };
  auto o_col = [&](int t) { return (uint32_t)(256 + t * 128); };

  if (warp < 4) {
    setmaxnreg_dec<88>();
    if (warp == 0 || warp == 2) {
      // ------------------------------------------------------------------ producers: one warp, a lane per box
      const bool keys = warp == 0;
      const int box = 1 << a.tile.box_log2, boxes = TL_KEYS >> a.tile.box_log2;
      const int lg = batch.page_log2, in_page = (1 << lg) - 1;
      uint32_t count = 0, q_count[2] = {0, 0};
      for (uint32_t i = 0; ok; ++i) {
        const int slot = i % TL_RING;
        ok = mbar_wait(ring_full(slot), (i / TL_RING) & 1u, status, keys ? 101 : 102);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        volatile TilePiece &p = ring[slot];
        const int valid = p.valid, row = p.row, len = p.len, seq = p.seq, head = p.head, lo = p.lo, hi = p.hi;
        const int n0 = p.blocks[0], n1 = p.blocks[1], clean = keys ? -1 : p.clean;
        __syncwarp();
        if (lane == 0) mbar_arrive(ring_empty(slot));
        if (!valid) break;
        const uint32_t *table = batch.table + (long long)seq * batch.table_ld;
        // the page of this lane's box of block j, outside the map where there is nothing to read
        auto look_up = [&](int j) -> int {
          const int key = j * TL_KEYS + lane * box;
          if (lane >= boxes || j >= hi || key >= len) return (int)batch.npages;
          const uint32_t page = table[key >> lg];
          if (page < batch.npages) return (int)page;
          atomicCAS(batch.status, 0, OPS_PAGED_BAD_PAGE);
          return (int)batch.npages;
        };
        int page = look_up(lo);
        if (keys)
          for (int t = 0; t < 2 && ok; ++t) {
            if ((t ? n1 : n0) == 0) continue;
            if (lane == 0) {
              ok = mbar_wait(q_empty(t), (q_count[t] & 1u) ^ 1u, status, 103 + t);
              if (ok) {
                mbar_arrive_expect_tx(q_full(t), (uint32_t)(group * a.per_tile * HALVES * 128));
#pragma unroll
                for (int h = 0; h < HALVES; ++h)
                  tma_load_4d(base + Smem::OFF_Q + t * TILE + h * (TL_ROWS * 128), &tmap_q, q_full(t), h * 64, 0, row + t * a.per_tile, head);
              }
            }
            ++q_count[t];
            ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0);
          }
        for (int j = lo; j < hi && ok; ++j, ++count) {
          const int s = count % ST;
          const uint32_t full = keys ? k_full(s) : v_full(s);
          if (lane == 0) {
            ok = mbar_wait(keys ? k_empty(s) : v_empty(s), ((count / ST) & 1u) ^ 1u, status, keys ? 105 : 106);
            if (ok) mbar_arrive_expect_tx(full, TILE);
          }
          ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0);
          if (!ok) break;
          const int next = look_up(j + 1);
          if (lane < boxes) {
            const int r = lane * box;  // first row of the block
            const int at = (j * TL_KEYS + r) & in_page;
#pragma unroll
            for (int h = 0; h < HALVES; ++h) {
              if (keys)  // [half][128 keys][128 B]
                tma_load_4d(base + Smem::OFF_K + s * TILE + h * (TL_KEYS * 128) + r * 128, &tmap_k, full, h * 64, at, head, page);
              else  // [64 keys][half][64 keys][128 B]
                tma_load_4d(base + Smem::OFF_V + s * TILE + ((r >> 6) * HALVES + h) * 8192 + (r & 63) * 128, &tmap_v, full, h * 64, at, head, page);
            }
          }
          page = next;
          if (j - lo == clean) {
            // the slots behind the end share a page with the last ones and may hold anything, a NaN too
            ok = __all_sync(0xffffffffu, mbar_wait(full, (count / ST) & 1u, status, 107));
            if (!ok) break;
            const int r0 = len % TL_KEYS, r1 = (r0 + box - 1) >> a.tile.box_log2 << a.tile.box_log2;
            for (int e = lane; e < (r1 - r0) * HALVES * 8; e += 32) {
              const int r = r0 + e / (HALVES * 8), piece = e % (HALVES * 8);
              *reinterpret_cast<uint4 *>(base_ptr + Smem::OFF_V + s * TILE + ((r >> 6) * HALVES + (piece >> 3)) * 8192 + (r & 63) * 128 + (piece & 7) * 16) =
                  make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async();  // the MMA reads these writes through the async proxy
            __syncwarp();
            if (lane == 0) mbar_arrive(v_clean(s));
          }
        }
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------------ MMA issuer
      // the whole warp walks along, one lane issues
      {
        const uint32_t leader = elect_one() ? 1u : 0u;
        const uint32_t idesc_qk = make_idesc_f16(TL_ROWS, TL_KEYS, 0, 0, BF ? 1 : 0);
        const uint32_t idesc_pv = make_idesc_f16(TL_ROWS, DH, 0, 1, BF ? 1 : 0);
        // a descriptor's address is its low bits, in 16 bytes: adding steps to one made once keeps the issue of an MMA short
        const uint64_t q_desc = make_smem_desc_sw128(base + Smem::OFF_Q, 16, 1024), k_desc = make_smem_desc_sw128(base + Smem::OFF_K, 16, 1024);
        const uint64_t v_desc = make_smem_desc_sw128(base + Smem::OFF_V, 8192, 1024);
        auto all_wait = [&](uint32_t bar, uint32_t parity, int code) -> bool { return __all_sync(0xffffffffu, mbar_wait(bar, parity, status, code)); };
        uint32_t count = 0, cleaned = 0 /* a bit per stage */, q_count[2] = {0, 0}, p_count[2] = {0, 0};
        for (uint32_t i = 0; ok; ++i) {
          const int slot = i % TL_RING;
          if (!(ok = all_wait(ring_full(slot), (i / TL_RING) & 1u, 120))) break;
          volatile TilePiece &p = ring[slot];
          auto uniform = [&](int v) -> int { return __shfl_sync(0xffffffffu, v, 0); };
          const int valid = uniform(p.valid), blocks = uniform(p.hi - p.lo), clean = uniform(p.clean);
          const int n0 = uniform(p.blocks[0]), n1 = uniform(p.blocks[1]);
          if (lane == 0) mbar_arrive(ring_empty(slot));
          if (!valid) break;
          // S(t) = Q(t) K_j^T.  Tile 1 sees every block that tile 0 sees, if it is there at all.
          auto issue_qk = [&](int t, int j) -> bool {
            const uint32_t c = count + (uint32_t)j;
            const int s = c % ST;
            if (!all_wait(k_full(s), (c / ST) & 1u, 121)) return false;
            tc_fence_after();
            const uint64_t da = q_desc + (uint32_t)(t * (TILE >> 4)), db = k_desc + (uint32_t)(s * (TILE >> 4));
            const uint32_t d = tmem_base + s_col(t);
#pragma unroll
            for (int ks = 0; ks < DH / 16; ++ks) {
              const uint32_t step = (ks >> 2) * (TL_ROWS * 128 >> 4) + (ks & 3) * 2;  // rows of Q and keys of a block are as many
              umma_f16_ss_by(leader, d, da + step, db + step, idesc_qk, ks != 0 ? 1u : 0u);
            }
            umma_commit_by(leader, s_full(t));
            if (t == 1 || n1 == 0) umma_commit_by(leader, k_empty(s));
            if (j == (t ? n1 : n0) - 1) umma_commit_by(leader, q_empty(t));
            return true;
          };
          // O(t) (+)= P(t) V_j, P from tensor memory
          auto issue_pv = [&](int t, int j) -> bool {
            const uint32_t c = count + (uint32_t)j;
            const int s = c % ST;
            if (!all_wait(v_full(s), (c / ST) & 1u, 122)) return false;
            if (j == clean && !all_wait(v_clean(s), (cleaned >> s) & 1u, 123)) return false;
            const uint64_t db = v_desc + (uint32_t)(s * (TILE >> 4));
            const uint32_t d = tmem_base + o_col(t);
            const uint32_t pa = tmem_base + s_col(t);
            // the first 64 keys' products run while the others' powers are taken
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (!all_wait(p_full(t, h), p_count[t] & 1u, 124)) return false;
              tc_fence_after();
#pragma unroll
              for (int k4 = 0; k4 < 4; ++k4) {
                const int ks = h * 4 + k4;
                umma_f16_ts_by(leader, d, pa + (uint32_t)(ks * 8), db + (uint32_t)((h * (HALVES * 8192) + k4 * 2048) >> 4), idesc_pv, (j != 0 || ks != 0) ? 1u : 0u);  // 16 keys = 8 packed columns
              }
            }
            ++p_count[t];
            if (j == (t ? n1 : n0) - 1) umma_commit_by(leader, o_final(t));
            if (t == 1 || n1 == 0) umma_commit_by(leader, v_empty(s));
            return true;
          };
          for (int t = 0; t < 2 && ok; ++t) {
            if ((t ? n1 : n0) == 0) continue;
            ok = all_wait(q_full(t), q_count[t] & 1u, 125) && issue_qk(t, 0);
            ++q_count[t];
          }
          for (int j = 0; j < blocks && ok; ++j)
            for (int t = 0; t < 2 && ok; ++t) {
              const int n = t ? n1 : n0;
              if (j < n) ok = issue_pv(t, j);
              if (ok && j + 1 < n) ok = issue_qk(t, j + 1);
            }
          if (clean >= 0) cleaned ^= 1u << ((count + (uint32_t)clean) % ST);
          count += (uint32_t)blocks;
        }
      }
    } else {
      // ------------------------------------------------------------------ scheduler
      if (lane == 0) {
        const PagedLine shared = paged_shared_line(line, share);
        const int total = share.total;
        PagedWalk walk = share.walk;
#pragma unroll 1
        for (uint32_t i = 0; ok; ++i) {
          const PagedPiece q = paged_step(batch, shared, walk);
          const int slot = i % TL_RING;
          if (!(ok = mbar_wait(ring_empty(slot), ((i / TL_RING) & 1u) ^ 1u, status, 130))) break;
          volatile TilePiece &to = ring[slot];
          to.valid = q.seq >= 0;
          if (q.seq >= 0) {
            const int t0 = q.tile * line.tokens;
            to.row = q.s.row + t0;
            to.tokens = q.s.n - t0;
            to.off = q.s.len - q.s.n + t0;
            to.len = q.s.len;
            to.seq = q.seq;
            to.head = q.head;
            to.lo = q.lo;
            to.hi = q.hi;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              const int seen = paged_keys(line, q.s, t0 + (t + 1) * a.per_tile);
              const int all = t0 + t * a.per_tile < q.s.n ? max(1, (seen + TL_KEYS - 1) / TL_KEYS) : 0;
              to.blocks[t] = max(0, min(all, q.hi) - q.lo);
            }
            const int end = q.s.len / TL_KEYS;  // the block the sequence ends in
            to.clean = (q.s.len & ((1 << a.tile.box_log2) - 1)) && end >= q.lo && end < q.hi ? end - q.lo : -1;
            const PagedParts parts = paged_parts(shared, total, share.cta, q);
            to.first = parts.first;
            to.count = parts.count;
            if (parts.count > 2) {
              volatile TileHelp &u = help[q.lo > 0 ? 0 : 1];
              u.first = parts.first;
              u.count = parts.count;
              u.row = q.s.row + t0;
              u.tokens = q.s.n - t0;
              u.head = q.head;
            }
          }
          mbar_arrive(ring_full(slot));
          if (q.seq < 0) break;
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ softmax, rescaling, output: a thread per q row
    setmaxnreg_inc<208>();
    const int t = (warp - 4) >> 2;   // q tile
    const int quarter = warp & 3;    // tensor-memory lanes [32 * quarter, +32)
    const int r = quarter * 32 + lane;
    const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
    const int tok = paged_div(r, line.by_group), gi = r - tok * group;
    const uint32_t ta = tmem_base + lane_addr + s_col(t), to = tmem_base + lane_addr + o_col(t);
    const float mult = a.odd_scale ? 1.f : a.scale_log2;
    uint32_t phases = 0;  // bit 0: of s_full, bit 1: of o_final
#pragma unroll 1
    for (uint32_t i = 0; ok; ++i) {
      const int slot = i % TL_RING;
      if (!(ok = __all_sync(0xffffffffu, mbar_wait(ring_full(slot), (i / TL_RING) & 1u, status, 141)))) break;
      volatile TilePiece &p = ring[slot];
      if (!p.valid) break;
      const int nblk = p.blocks[t];
      const int mine = t * a.per_tile + tok;  // token of the unit
      const int limit = line.causal ? min(p.len - 1, p.off + mine) : p.len - 1;  // last slot this row may see
      int kv0 = p.lo * TL_KEYS;
      float m = -INFINITY, l = 0.f;
#pragma unroll 1
      for (int j = 0; j < nblk; ++j, kv0 += TL_KEYS) {
        if (!(ok = __all_sync(0xffffffffu, mbar_wait(s_full(t), phases & 1u, status, 142)))) break;
        phases ^= 1u;
        tc_fence_after();
        uint32_t x[4][32];
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_ld_32x32(ta + 32u * q, x[q]);
        tmem_wait_ld();
        // Rare cases first, each in a branch of its own that whole warps take or leave, so that the common path is an addition, a
        // power, a multiply-add and half a maximum and half a conversion per score.
        if (a.odd_scale) {  // not positive: the maximum of the products is not the product of the maximum
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int e = 0; e < 32; ++e) x[q][e] = __float_as_uint(__uint_as_float(x[q][e]) * a.scale_log2);
        }
        if (__any_sync(0xffffffffu, kv0 + TL_KEYS - 1 > limit)) {  // the diagonal, or the end: what a row does not see weighs nothing
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (kv0 + q * 32 + e > limit) x[q][e] = 0xff800000u;  // -infinity
        }
        float mx[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          mx[q] = __uint_as_float(x[q][0]);
#pragma unroll
          for (int e = 1; e < 31; e += 2) mx[q] = tl_max3(mx[q], __uint_as_float(x[q][e]), __uint_as_float(x[q][e + 1]));
          mx[q] = fmaxf(mx[q], __uint_as_float(x[q][31]));
        }
        // Lazy rescaling: the reference point m of the powers follows the row maximum only when that has moved by more than 2^8.
        // Until then the probabilities are taken relative to the older, smaller m: they stay below 256, exact to half a step in
        // the 16-bit operand, and the f32 row sum and O carry the same factor, which cancels in o = O / l.
        const float m_raw = fmaxf(m, fmaxf(tl_max3(mx[0], mx[1], mx[2]), mx[3]) * mult);
        const bool move = m_raw > m + 8.f;                       // also true on the first block (m = -inf)
        const float m_next = move ? m_raw : m;
        const float m_new = m_next == -INFINITY ? 0.f : m_next;  // a row with nothing visible yet: keep the arithmetic finite
        if (__any_sync(0xffffffffu, move)) {
          const float alpha = move ? ap_ex2(m - m_new) : 1.f;    // 0 on the first block
          l *= alpha;
          if (j > 0) {
            // S of block j being complete says that PV of block j-1 has completed too (the tensor pipe retires in order): O is stable
#pragma unroll 1
            for (int c = 0; c < DH; c += 16) {
              uint32_t v[16];
              tmem_ld_32x16(to + (uint32_t)c, v);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * alpha);
              tmem_st_32x16(to + (uint32_t)c, v);
            }
          }
        }
        m = m_next;
        // probabilities -> tensor memory as packed pairs, in two halves; row sum
        float2 sum = make_float2(0.f, 0.f);
        const float2 by = make_float2(mult, mult), less = make_float2(-m_new, -m_new);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t packed[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            float2 y = __ffma2_rn(make_float2(__uint_as_float(x[q][e]), __uint_as_float(x[q][e + 1])), by, less);
            y.x = ap_ex2(y.x);
            y.y = ap_ex2(y.y);
            sum = __fadd2_rn(sum, y);
            packed[e >> 1] = ap_pack<BF>(y.x, y.y);
          }
          tmem_st_32x16(ta + 16u * q, packed);
          if (q & 1) {
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full(t, q >> 1));
          }
        }
        l += sum.x + sum.y;
      }
      if (!ok) break;
      const bool there = tok < a.per_tile && mine < p.tokens;
      const int first = p.first, parts = p.count;
      const long long row = p.row + mine;
      const int q_head = p.head * group + gi;
      __syncwarp();
      if (lane == 0) mbar_arrive(ring_empty(slot));
      if (nblk == 0 && parts == 1) continue;  // the unit has no tokens for this tile
      bool own = nblk > 0;                    // whether there is an O: a tile may have no block in this part of its unit
      if (own) {
        if (!(ok = __all_sync(0xffffffffu, mbar_wait(o_final(t), phases >> 1, status, 143)))) break;
        phases ^= 2u;
        tc_fence_after();
      }
      // A row is one thread's, 512 or 256 bytes of it: written as it is, every store of a warp would touch 32 lines.  128 bytes of
      // the warp's 32 rows at a time turn in shared memory instead, 16-byte pieces swizzled by the row, and leave as whole lines
      // (a piece's end 5000 -> 1900 cycles).
      uint8_t *stage = base_ptr + Smem::OFF_STAGE + (warp - 4) * 4096;
      auto turn = [&](int e, uint4 v) { *reinterpret_cast<uint4 *>(stage + lane * 128 + ((e ^ (lane & 7)) << 4)) = v; };  // e-th piece of the own row
      auto leave = [&](auto &&address) {  // address(row of the warp, piece) -> where it goes, or null
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int rr = k * 4 + (lane >> 3), e = lane & 7;
          const uint4 v = *reinterpret_cast<const uint4 *>(stage + rr * 128 + ((e ^ (rr & 7)) << 4));
          if (char *where = address(rr, e)) st_global_16(where, v);
        }
        __syncwarp();
      };
      // Other CTAs have the other parts of the unit.  Of two, the common case in a long line of units, each warp's rows are joined by
      // whichever of the two warps comes last, from its tensor memory and the other's parked part.  More are parked, all of them, and
      // joined at the end of the share (see below).
      if (parts > 1) {
        pdl_wait_for_front();  // the counters have been cleared
        const int k = *(const volatile int *)&share.cta - first;
        auto rows_of = [&](int k) -> long long {  // this warp's rows of the unit's k-th part
          return (long long)paged_slot(first, k) * (2 * TL_ROWS) + t * TL_ROWS + quarter * 32;
        };
        uint32_t *arrived = parts == 2 ? a.tile.arrived + first * 8 + (warp - 4) : a.tile.arrived + (line.ctas + first) * 8;
        const bool counts = l != 0.f;  // a row that sees nothing in this part (a NaN is something) has zeros for its o, whatever V holds
        bool last = parts == 2 && paged_others_parked(arrived, 2);
        if (!last) {
          float *mine_at = a.tile.parts + rows_of(k) * DH;
          a.tile.parts_ml[rows_of(k) + lane] = make_float2(m, l);
#pragma unroll 1
          for (int c = 0; c < DH; c += 32) {
            uint32_t v[32];
            tmem_ld_32x32(to + (uint32_t)c, v);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!counts) v[e] = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) turn(e, make_uint4(v[e * 4], v[e * 4 + 1], v[e * 4 + 2], v[e * 4 + 3]));
            leave([&](int rr, int e) { return reinterpret_cast<char *>(mine_at + rr * DH + c + e * 4); });
          }
          const uint32_t ticket = paged_arrive(arrived);
          last = parts == 2 && ticket == 1;
          if (last) __threadfence();
          if (lane == 0) sh.tickets[k == 0][warp - 4] = ticket;
        }
        if (!last) {
          tc_fence_before();
          continue;
        }
        const float *theirs = a.tile.parts + rows_of(k ^ 1) * DH;
        auto fetch = [&](int c, uint4 (&x)[8]) {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = __ldcg(reinterpret_cast<const uint4 *>(theirs + (e * 4 + (lane >> 3)) * DH + (lane & 7) * 4 + c));
        };
        uint4 x[8];
        fetch(0, x);
        const float2 ml = __ldcg(a.tile.parts_ml + rows_of(k ^ 1) + lane);
        const float top = fmaxf(m, ml.x), ref = top == -INFINITY ? 0.f : top;
        const float w_own = ap_ex2(m - ref), w_their = ap_ex2(ml.x - ref);
        l = __fadd_rn(__fmul_rn(l, w_own), __fmul_rn(ml.y, w_their));  // products and a sum: the same whichever of the two comes last
#pragma unroll 1
        for (int c = 0; c < DH; c += 32) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int rr = e * 4 + (lane >> 3), piece = lane & 7;
            *reinterpret_cast<uint4 *>(stage + rr * 128 + ((piece ^ (rr & 7)) << 4)) = x[e];
          }
          if (c + 32 < DH) fetch(c + 32, x);
          __syncwarp();
          uint32_t v[32];
          tmem_ld_32x32(to + (uint32_t)c, v);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint4 y = *reinterpret_cast<const uint4 *>(stage + lane * 128 + ((e ^ (lane & 7)) << 4));
            const uint32_t z[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const float mine = counts ? __fmul_rn(__uint_as_float(v[e * 4 + q]), w_own) : 0.f;
              v[e * 4 + q] = __float_as_uint(__fadd_rn(mine, __fmul_rn(__uint_as_float(z[q]), w_their)));
            }
          }
          tmem_st_32x32(to + (uint32_t)c, v);
          __syncwarp();
        }
        tmem_wait_st();
      }
      {
        const float inv = l > 0.f ? __frcp_rn(l) : 0.f;  // a row that sees nothing: zeros
        char *orow = there ? a.o + row * a.o_t + (long long)q_head * a.o_h : nullptr;
#pragma unroll 1
        for (int c = 0; c < DH; c += 64) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint32_t v[32];
            tmem_ld_32x32(to + (uint32_t)(c + half * 32), v);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              uint4 out;
              out.x = ap_pack<BF>(__uint_as_float(v[e]) * inv, __uint_as_float(v[e + 1]) * inv);
              out.y = ap_pack<BF>(__uint_as_float(v[e + 2]) * inv, __uint_as_float(v[e + 3]) * inv);
              out.z = ap_pack<BF>(__uint_as_float(v[e + 4]) * inv, __uint_as_float(v[e + 5]) * inv);
              out.w = ap_pack<BF>(__uint_as_float(v[e + 6]) * inv, __uint_as_float(v[e + 7]) * inv);
              turn(half * 4 + e / 8, out);
            }
          }
          leave([&](int rr, int e) -> char * {
            char *whose = reinterpret_cast<char *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(orow), rr));
            return whose && c + e * 8 < a.dh ? whose + (c + e * 8) * 2 : nullptr;
          });
        }
      }
      tc_fence_before();  // the next P of this tile says that O has been read
    }
    // Units of more than two parts (few units, long pasts): their rows are dealt out, 16 rows by 32 columns at a time, to the warps
    // of all their CTAs in the order in which these parked their parts.  A warp waits a while for the last part, not for good: when
    // its patience ends it marks its slices as left and goes, and the warp that parks the last part, which finds nothing to wait
    // for, does what was left.  (A word counts the parts in its low half and those who left in its high half; who finds that all
    // parts have come as it leaves stays.)
    for (int h = 0; h < 2 && ok; ++h) {
      const volatile TileHelp &u = help[h];
      if (u.count <= 2) continue;
      const int first = u.first, parts = u.count, tokens = u.tokens;
      __syncwarp();
      const uint32_t warps = 8 * (uint32_t)parts, arrival = sh.tickets[h][warp - 4], ticket = arrival & 0xffffu;
      uint32_t *arrived = a.tile.arrived + (line.ctas + first) * 8;
      auto left = [&](uint32_t t) -> uint32_t * {  // bits of the warps with tickets [8 k, 8 k + 8); the last CTA may be the first of the next unit
        const int k = (int)(t >> 3);
        return arrived + k * 8 + (k == parts - 1 ? 2 : 1);
      };
      bool all = false;
      const unsigned long long since = globaltimer_ns();
      do {
        uint32_t n = 0;
        if (lane == 0) n = ld_acquire_gpu(arrived);
        all = (__shfl_sync(0xffffffffu, n, 0) & 0xffffu) == warps;
      } while (!all && __all_sync(0xffffffffu, globaltimer_ns() - since < a.patience));
      if (!all) {
        uint32_t n = 0;
        if (lane == 0) {
          atomicOr(left(ticket), 1u << (ticket & 7));
          __threadfence();
          n = atomicAdd(arrived, 0x10000u);
        }
        if ((__shfl_sync(0xffffffffu, n, 0) & 0xffffu) != warps) continue;
      }
      __threadfence();
      const bool heir = ticket == warps - 1 && arrival > 0xffffu;
      uint32_t next = 0;
#pragma unroll 1
      for (uint32_t whose = ticket; whose < warps; whose = next++) {
        if (next > 0 && (whose == ticket || !(*reinterpret_cast<volatile uint32_t *>(left(whose)) >> (whose & 7) & 1u))) continue;
        constexpr int COLUMNS = DH / 32, ROWS = 16, MINE = ROWS / 4, DEEP = 4;  // of a slice; a lane's rows of it; parts in flight
#pragma unroll 1
        for (int slice = (int)whose; slice < 2 * TL_ROWS / ROWS * COLUMNS; slice += (int)warps) {
          const int rows0 = slice / COLUMNS * ROWS, col = slice % COLUMNS * 32 + (lane & 7) * 4;
          const int tile_tokens = tokens - (rows0 >= TL_ROWS ? a.per_tile : 0);  // from the slice's tile on
          if ((rows0 & (TL_ROWS - 1)) >= min(tile_tokens, a.per_tile) * group) continue;
          // a lane: 4 columns of every fourth row
          float4 acc[MINE];
          float top[MINE], den[MINE];
#pragma unroll
          for (int e = 0; e < MINE; ++e) {
            acc[e] = make_float4(0.f, 0.f, 0.f, 0.f);
            top[e] = -INFINITY;
            den[e] = 0.f;
          }
#pragma unroll 1
          for (int k0 = 0; k0 < parts; k0 += DEEP) {
            float4 v[DEEP][MINE];
            float2 ml[DEEP][MINE];
#pragma unroll
            for (int d = 0; d < DEEP; ++d) {
              const long long from = (long long)paged_slot(first, k0 + d) * (2 * TL_ROWS) + rows0 + (lane >> 3);
#pragma unroll
              for (int e = 0; e < MINE; ++e) {
                ml[d][e] = make_float2(-INFINITY, 0.f);
                v[d][e] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (k0 + d < parts) {
                  ml[d][e] = __ldcg(a.tile.parts_ml + from + e * 4);
                  v[d][e] = __ldcg(reinterpret_cast<const float4 *>(a.tile.parts + (from + e * 4) * DH + col));
                }
              }
            }
#pragma unroll
            for (int e = 0; e < MINE; ++e) {
              float next_top = top[e];
#pragma unroll
              for (int d = 0; d < DEEP; ++d) next_top = fmaxf(next_top, ml[d][e].x);
              const float ref = next_top == -INFINITY ? 0.f : next_top, wa = ap_ex2(top[e] - ref);
              top[e] = next_top;
              den[e] *= wa;
              acc[e] = make_float4(acc[e].x * wa, acc[e].y * wa, acc[e].z * wa, acc[e].w * wa);
#pragma unroll
              for (int d = 0; d < DEEP; ++d) {
                const float w = ap_ex2(ml[d][e].x - ref);
                den[e] = fmaf(ml[d][e].y, w, den[e]);
                acc[e].x = fmaf(v[d][e].x, w, acc[e].x);
                acc[e].y = fmaf(v[d][e].y, w, acc[e].y);
                acc[e].z = fmaf(v[d][e].z, w, acc[e].z);
                acc[e].w = fmaf(v[d][e].w, w, acc[e].w);
              }
            }
          }
#pragma unroll
          for (int e = 0; e < MINE; ++e) {
            const int rr = (rows0 & (TL_ROWS - 1)) + e * 4 + (lane >> 3), tk = paged_div(rr, line.by_group), hd = rr - tk * group;
            if (tk >= a.per_tile || tk >= tile_tokens || col >= a.dh) continue;
            const float inv = den[e] > 0.f ? __frcp_rn(den[e]) : 0.f;
            char *where = a.o + (long long)(u.row + (rows0 >= TL_ROWS ? a.per_tile : 0) + tk) * a.o_t + (long long)(u.head * group + hd) * a.o_h + col * 2;
            *reinterpret_cast<uint2 *>(where) = make_uint2(ap_pack<BF>(acc[e].x * inv, acc[e].y * inv), ap_pack<BF>(acc[e].z * inv, acc[e].w * inv));
          }
        }
        if (!heir) break;
      }
    }
  }
  return ok;
}

}  // namespace ops

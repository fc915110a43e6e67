// attention_paged_few.cu — attention over a paged cache for sequences with a handful of query rows (a decode step, a few drafted
// tokens): at most 8 or 16 rows = new tokens x query heads per kv head.
//
//   o_r = sum_j 2^(x_rj - m_r) v_j / sum_j 2^(x_rj - m_r),  x_rj = scale log2(e) q_r . k_j,  one pass with a running m_r
//
// The work is reading K and V once, 4 dh bytes a key and kv head, HBM-bound.  The keys of all (sequence, kv head) pairs form one
// line of which every CTA takes an equal share (paged_schedule.h), so ragged lengths cost nothing.  A CTA of 8 warps
// walks blocks of 128 keys, 16 a warp; a lane issues all sixteen 128-bit loads of its K and V pieces (64 KB a CTA in flight,
// two CTAs an SM) before it uses one, with the page numbers fetched a block ahead, and the first loads of the next piece
// are issued before the current one is brought together.  The arithmetic rides on m16n8k16 warp MMAs (a 128-row tcgen05 tile has
// nothing to chew on here), as in attention_decode.cu: lane (g, c) = (lane / 4, lane % 4),
//   S[rows x 8 keys] = Q K^T: A = q rows g (and g + 8), B = K rows straight from global; the contraction is permuted so that one
//                      128-bit load of a K row serves two k-steps;
//   O^T[16 dh x 8 rows] = V^T P^T: A = byte-permuted V rows, B = the S fragments, exponentiated.
// Slots past the sequence's length are not loaded (their registers are zero), so whatever they hold stays out.  The 8 warps of a
// CTA meet in shared memory at the end of a piece.
#include "attention_paged.h"
#include "device_utils.cuh"

namespace ops {

constexpr int FEW_WARPS = 8, FEW_THREADS = FEW_WARPS * 32;
constexpr int FEW_BLOCK = AP_FEW_BLOCK;
static_assert(FEW_BLOCK == FEW_WARPS * 16, "16 keys a warp");

// d += a . b, one warp, m16n8k16, f32 accumulate
template <bool BF>
__device__ __forceinline__ void few_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (BF)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t few_word(const uint4 &v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

__device__ __forceinline__ void cp_async_16(void *dst, const void *src, bool there) {  // zeros where nothing is
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
}

template <int DH, int NR> struct FewSmem {
  static constexpr int ROWS = NR * 8;
  static constexpr int LD = DH + 4;  // padded: the lanes of a column pair write other banks
  static constexpr int OFF_Q = 0;                                        // [2][ROWS][DH] 16-bit: this piece's and the next one's
  static constexpr int OFF_M = OFF_Q + 2 * ROWS * DH * 2;                // [warps][ROWS]
  static constexpr int OFF_L = OFF_M + FEW_WARPS * ROWS * 4;             // [warps][ROWS]
  static constexpr int OFF_O = OFF_L + FEW_WARPS * ROWS * 4;             // [warps][ROWS][LD]
  static constexpr int BYTES = OFF_O + FEW_WARPS * ROWS * LD * 4;
};

template <int DH, bool BF, int NR>
__global__ void __launch_bounds__(FEW_THREADS, NR == 1 ? 2 : 1) attention_paged_few_kernel(const __grid_constant__ PagedAttnArgs a) {
  typedef FewSmem<DH, NR> Smem;
  constexpr int ROWS = Smem::ROWS, LD = Smem::LD;
  constexpr int CH = DH / 32;  // 128-bit loads per K row per lane
  constexpr int HH = DH / 64;  // 64-wide halves of a V row
  extern __shared__ __align__(16) uint8_t smem[];
  unsigned short *q_s = reinterpret_cast<unsigned short *>(smem + Smem::OFF_Q);
  float *red_m = reinterpret_cast<float *>(smem + Smem::OFF_M), *red_l = reinterpret_cast<float *>(smem + Smem::OFF_L);
  float *red_o = reinterpret_cast<float *>(smem + Smem::OFF_O);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int group = a.line.group, lg = a.batch.page_log2, mask = (1 << lg) - 1;

  pdl_let_next_come();
  i64 total;
  PagedWalk walk = paged_locate<FEW_THREADS>(a.batch, a.line, blockIdx.x, blockIdx.x == 0, &total);
  PagedPiece cur = paged_step(a.batch, a.line, walk);
  if (cur.seq < 0) {
    if (threadIdx.x == 0) paged_note_join(a, blockIdx.x, cur, walk, total);
    return;
  }

  uint4 kq[2][CH], vq[HH][4];
  uint32_t pg0, pg1;  // pages of the warp's 16 keys, first and second eight
  auto pages = [&](const PagedPiece &p, int kb, int k_end) {
    const uint32_t *table = a.batch.table + (long long)p.seq * a.batch.table_ld;
    pg0 = kb < k_end ? table[kb >> lg] : 0u;
    pg1 = kb + 8 < k_end ? table[(kb + 8) >> lg] : 0u;
  };
  // keys kb .. kb+15 of this warp; what lies at or past k_end, or in a page that is not there, is zeros
  auto issue_k = [&](const PagedPiece &p, int kb, int k_end) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int key = kb + j * 8 + g;
      const uint32_t pg = j ? pg1 : pg0;
      const bool ok = key < k_end && pg < a.batch.npages;
      const char *kr = a.k + (long long)pg * a.kp_p + (long long)p.head * a.kp_h + (long long)(key & mask) * a.kp_s + c * 16;
#pragma unroll
      for (int ch = 0; ch < CH; ++ch) {
        kq[j][ch] = make_uint4(0, 0, 0, 0);
        if (ok && ch * 32 + c * 8 < a.dh) kq[j][ch] = __ldcs(reinterpret_cast<const uint4 *>(kr + ch * 64));
      }
    }
  };
  auto issue_v = [&](const PagedPiece &p, int kb, int k_end) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int key = kb + 2 * c + (j & 1) + (j >> 1) * 8;
      const uint32_t pg = (j >> 1) ? pg1 : pg0;
      const bool ok = key < k_end && pg < a.batch.npages;
      const char *vr = a.v + (long long)pg * a.vp_p + (long long)p.head * a.vp_h + (long long)(key & mask) * a.vp_s + g * 16;
#pragma unroll
      for (int hh = 0; hh < HH; ++hh) {
        vq[hh][j] = make_uint4(0, 0, 0, 0);
        if (ok && hh * 64 + g * 8 < a.dh) vq[hh][j] = __ldcs(reinterpret_cast<const uint4 *>(vr + hh * 128));
      }
    }
  };
  auto bad_page = [&](int kb, int k_end) {
    if ((kb < k_end && pg0 >= a.batch.npages) || (kb + 8 < k_end && pg1 >= a.batch.npages))
      if (lane == 0) atomicCAS(a.batch.status, 0, OPS_PAGED_BAD_PAGE);
  };
  auto stage_q = [&](const PagedPiece &p, int buf) {
    for (int i = threadIdx.x; i < ROWS * DH / 8; i += FEW_THREADS) {
      const int r = i / (DH / 8), col = (i - r * (DH / 8)) * 8;
      const int tok = r / group, gi = r - tok * group;
      const bool there = tok < p.s.n && col < a.dh;
      const char *src = there ? a.q + (long long)(p.s.row + tok) * a.q_t + (long long)(p.head * group + gi) * a.q_h + col * 2 : a.q;
      cp_async_16(q_s + (buf * ROWS + r) * DH + col, src, there);
    }
  };

  int k_end = min(cur.hi * FEW_BLOCK, cur.s.len);
  int kb = cur.lo * FEW_BLOCK + warp * 16;
  pages(cur, kb, k_end);
  stage_q(cur, 0);
  bad_page(kb, k_end);
  issue_k(cur, kb, k_end);
  issue_v(cur, kb, k_end);
  cp_async_wait();
  __syncthreads();
  int buf = 0;
  while (true) {
    const i64 cur_begin = walk.begin;
    const PagedPiece nxt = paged_step(a.batch, a.line, walk);
    if (nxt.seq >= 0) stage_q(nxt, buf ^ 1);
    const int rows = cur.s.n * group;
    // q fragments are re-read from shared memory at every use (volatile: hoisting them would cost registers that the loads in
    // flight need)
    const volatile uint4 *q_frag = reinterpret_cast<const volatile uint4 *>(q_s + (buf * ROWS + g) * DH + c * 8);
    int lim[NR];  // last visible key of row g (+ 8)
    float m[NR], l[NR];  // m is common to the four lanes of a row, l is this lane's share
    float o[NR][HH][4][4];
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
      const int r = nr * 8 + g;
      lim[nr] = r < rows ? (a.line.causal ? cur.s.len - cur.s.n + r / group : cur.s.len - 1) : -1;
      m[nr] = -INFINITY;
      l[nr] = 0.f;
#pragma unroll
      for (int hh = 0; hh < HH; ++hh)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[nr][hh][i][e] = 0.f;
    }
    for (; kb < k_end; kb += FEW_BLOCK) {  // warp-uniform
      const bool more = kb + FEW_BLOCK < k_end;
      if (more) pages(cur, kb + FEW_BLOCK, k_end);
      float s[2][4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][e] = 0.f;
#pragma unroll
        for (int ch = 0; ch < CH; ++ch) {
          const uint32_t q0 = q_frag[ch * 4].x, q1 = q_frag[ch * 4].y, q2 = q_frag[ch * 4].z, q3 = q_frag[ch * 4].w;
          uint32_t r0 = 0, r1 = 0, r2 = 0, r3 = 0;
          if (NR == 2) {
            const volatile uint4 *up = q_frag + DH + ch * 4;  // row g + 8
            r0 = up->x;
            r1 = up->y;
            r2 = up->z;
            r3 = up->w;
          }
          few_mma<BF>(s[j], q0, r0, q1, r1, kq[j][ch].x, kq[j][ch].y);
          few_mma<BF>(s[j], q2, r2, q3, r3, kq[j][ch].z, kq[j][ch].w);
        }
      }
      if (more) {
        bad_page(kb + FEW_BLOCK, k_end);
        issue_k(cur, kb + FEW_BLOCK, k_end);  // the K registers are free again
      }
      uint32_t pb[NR][2];
      float al[NR][2];
#pragma unroll
      for (int nr = 0; nr < NR; ++nr) {
        float sv[4], mx = -INFINITY;  // row 8 nr + g at keys kb + 8j + 2c + {0,1}
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int key = kb + j * 8 + 2 * c + e;
            const float x = (key < k_end && key <= lim[nr]) ? s[j][nr * 2 + e] * a.scale_log2 : -INFINITY;
            sv[j * 2 + e] = x;
            mx = fmaxf(mx, x);
          }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float m_new = fmaxf(m[nr], mx);
        const float m_use = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = ap_ex2(m[nr] - m_use);
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) p[e] = ap_ex2(sv[e] - m_use);
        l[nr] = fmaf(l[nr], alpha, (p[0] + p[1]) + (p[2] + p[3]));
        m[nr] = m_new;
        pb[nr][0] = ap_pack<BF>(p[0], p[1]);
        pb[nr][1] = ap_pack<BF>(p[2], p[3]);
        // the accumulators of this lane belong to rows 8 nr + 2c and 2c + 1
        al[nr][0] = __shfl_sync(0xffffffffu, alpha, (2 * c) << 2);
        al[nr][1] = __shfl_sync(0xffffffffu, alpha, (2 * c + 1) << 2);
      }
#pragma unroll
      for (int hh = 0; hh < HH; ++hh)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t w0 = few_word(vq[hh][0], i), w1 = few_word(vq[hh][1], i), w2 = few_word(vq[hh][2], i), w3 = few_word(vq[hh][3], i);
          const uint32_t a0 = __byte_perm(w0, w1, 0x5410), a1 = __byte_perm(w0, w1, 0x7632), a2 = __byte_perm(w2, w3, 0x5410), a3 = __byte_perm(w2, w3, 0x7632);
#pragma unroll
          for (int nr = 0; nr < NR; ++nr) {
            float (&d)[4] = o[nr][hh][i];
            d[0] *= al[nr][0];
            d[1] *= al[nr][1];
            d[2] *= al[nr][0];
            d[3] *= al[nr][1];
            few_mma<BF>(d, a0, a1, a2, a3, pb[nr][0], pb[nr][1]);
          }
        }
      if (more) issue_v(cur, kb + FEW_BLOCK, k_end);
    }
    const PagedPiece done = cur;
    if (nxt.seq >= 0) {  // in flight while this piece is brought together
      cur = nxt;
      k_end = min(cur.hi * FEW_BLOCK, cur.s.len);
      kb = cur.lo * FEW_BLOCK + warp * 16;
      pages(cur, kb, k_end);
      bad_page(kb, k_end);
      issue_k(cur, kb, k_end);
      issue_v(cur, kb, k_end);
    }

    // the 8 warps meet: common maximum per row, rescaled sums
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
      l[nr] += __shfl_xor_sync(0xffffffffu, l[nr], 1);
      l[nr] += __shfl_xor_sync(0xffffffffu, l[nr], 2);
      if (c == 0) red_m[warp * ROWS + nr * 8 + g] = m[nr];
    }
    __syncthreads();
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < FEW_WARPS; ++w) top = fmaxf(top, red_m[w * ROWS + nr * 8 + g]);
      if (c == 0) red_l[warp * ROWS + nr * 8 + g] = m[nr] == -INFINITY ? 0.f : l[nr] * ap_ex2(m[nr] - top);
      float sc[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = nr * 8 + 2 * c + e;
        float t = -INFINITY;
#pragma unroll
        for (int w = 0; w < FEW_WARPS; ++w) t = fmaxf(t, red_m[w * ROWS + r]);
        const float mw = red_m[warp * ROWS + r];
        sc[e] = mw == -INFINITY ? 0.f : ap_ex2(mw - t);
      }
      float *to = red_o + (warp * ROWS + nr * 8 + 2 * c) * LD;
#pragma unroll
      for (int hh = 0; hh < HH; ++hh)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int col = hh * 64 + g * 8 + 2 * i;
          *reinterpret_cast<float2 *>(to + col) = make_float2(o[nr][hh][i][0] * sc[0], o[nr][hh][i][2] * sc[0]);
          *reinterpret_cast<float2 *>(to + LD + col) = make_float2(o[nr][hh][i][1] * sc[1], o[nr][hh][i][3] * sc[1]);
        }
    }
    __syncthreads();
    const bool whole = done.whole();
    float *part = a.parts + (long long)(blockIdx.x * 2 + done.slot()) * ROWS * (DH + AP_PAD);
    for (int i = threadIdx.x; i < rows * (DH / 4); i += FEW_THREADS) {
      const int r = i / (DH / 4), col = (i - r * (DH / 4)) * 4;
      if (col >= a.dh) continue;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      float den = 0.f, top = -INFINITY;
#pragma unroll
      for (int w = 0; w < FEW_WARPS; ++w) {
        const float4 x = *reinterpret_cast<const float4 *>(red_o + (w * ROWS + r) * LD + col);
        acc.x += x.x;
        acc.y += x.y;
        acc.z += x.z;
        acc.w += x.w;
        den += red_l[w * ROWS + r];
        top = fmaxf(top, red_m[w * ROWS + r]);
      }
      if (whole) {
        const float inv = den > 0.f ? 1.f / den : 0.f;  // a row that sees nothing: zeros
        const int tok = r / group, gi = r - tok * group;
        char *to = a.o + (long long)(done.s.row + tok) * a.o_t + (long long)(done.head * group + gi) * a.o_h + col * 2;
        *reinterpret_cast<uint2 *>(to) = make_uint2(ap_pack<BF>(acc.x * inv, acc.y * inv), ap_pack<BF>(acc.z * inv, acc.w * inv));
      } else {
        float *to = part + r * (DH + AP_PAD);
        *reinterpret_cast<float4 *>(to + col) = acc;
        if (col == 0) *reinterpret_cast<float2 *>(to + DH) = make_float2(top, den);
      }
    }
    if (nxt.seq < 0) {
      walk.begin = cur_begin;
      if (threadIdx.x == 0) paged_note_join(a, blockIdx.x, done, walk, total);
      return;
    }
    cp_async_wait();
    __syncthreads();
    buf ^= 1;
  }
}

// One wave: two CTAs an SM for 8 rows (128 registers), one for 16 (twice the accumulators).
int attention_paged_few_ctas(const OpBase &base, int rows) { return rows == 8 ? 2 * base.sm_count : base.sm_count; }

template <int DH, bool BF, int NR>
static int few_launch(const PagedAttnArgs &a, cudaStream_t s) {
  const int bytes = FewSmem<DH, NR>::BYTES;
  cudaError_t e = cudaFuncSetAttribute(attention_paged_few_kernel<DH, BF, NR>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return fail(OPS_EXECUTION_FAILED, "attention_paged: cannot reserve %d bytes of shared memory: %s", bytes, cudaGetErrorString(e));
  attention_paged_few_kernel<DH, BF, NR><<<a.line.ctas, FEW_THREADS, bytes, s>>>(a);
  return check_launch("attention_paged(few rows)");
}

int attention_paged_few(const PagedAttnArgs &a, int rows, bool bf16, cudaStream_t s) {
  if (a.dh <= 64) {
    if (rows == 8) return bf16 ? few_launch<64, true, 1>(a, s) : few_launch<64, false, 1>(a, s);
    return bf16 ? few_launch<64, true, 2>(a, s) : few_launch<64, false, 2>(a, s);
  }
  if (rows == 8) return bf16 ? few_launch<128, true, 1>(a, s) : few_launch<128, false, 1>(a, s);
  return bf16 ? few_launch<128, true, 2>(a, s) : few_launch<128, false, 2>(a, s);
}

}  // namespace ops

// Attention of the last few tokens of every sequence over a paged cache (head_dim 64 or 128, bf16 or NVFP4 rows).
//
// The mathematics is the one-pass softmax: over the key tiles of a query row, m = running reference, l = sum 2^(s - m),
// o = sum 2^(s - m) v, all in f32; partial (m, l, o) of disjoint key sets join by m* = max m, l* = sum l 2^(m - m*),
// o* likewise. The reference m only has to lie near the true maximum (P, l and o scale together), so it is moved, and o
// rescaled, only when a score exceeds it by a wide margin: no cross-lane maximum in the common tile.
//
// Bound by HBM for bf16 rows (each row of a sequence is read once, all query heads of a KV head ride along) and by
// instruction issue for NVFP4 rows (the expansion of codes). Measured (32 query and 8 KV heads of 128): 165 us for 64
// sequences of 1500 to 6700 bf16 rows (6.4 TB/s, 0.98 of the copy rate), 618 us for 32 of 32768 (6.9 TB/s), 8.0 us for one of
// 777 (latency: two dependent launches); over NVFP4 rows 83 to 86 us for two tokens of 32 sequences, capped, with a window of
// 8000 rows (298 MB, 0.54).
//
// Split. The lengths are known to the device only and differ from sequence to sequence, so the unit of work is one
// 64-row tile of one (sequence, KV head, row tile) item; the tiles of all items form one line that is cut evenly over
// a grid of fixed size. A CTA's run of tiles is a list of pieces, at most the first and the last of which cover their
// item only in part: those go to the workspace (two slots per CTA), whole items are written directly. The join kernel
// finds an item's pieces by arithmetic and adds them in tile order, so a call gives the same bits every time.
//
// Layout. Keys are the M side of both products (S^T = K Q^T, O^T = V^T P^T, mma.sync m16n8k16): with up to eight query
// rows an 8-wide N tile holds them all (16 query rows on the M side waste half the products and the accumulators),
// and P^T becomes an operand by one 8 x 8 transpose of packed pairs. Over bf16 rows four compute warps take 16 rows each of
// a tile that arrives by TMA through a ring of three stages (boxes of up to 64 rows that do not cross a page).
#include "paged.cuh"

#include <cuda_fp16.h>

#include <algorithm>

namespace {

using namespace tc5;

constexpr int BC = 64;                  // rows per tile
constexpr int STAGES = 3;

// How far (in powers of two) a score may exceed the reference m before m moves, and how far below the maximum m is then
// put. Probabilities in f16 (beside four-bit rows) sit in its upper range, [2^7, 2^15] at the top, so that one of 2^-21 of
// the largest is still a normal number; bf16 has the range of f32.
constexpr float LAG_BF16 = 8.0f, LAG_F16 = 15.0f, DROP_F16 = 7.0f;

struct DecodeParams {
  CUtensorMap tmap_k, tmap_v;           // bf16 pools
  PagedView c;
  const uint8_t *k, *v, *ks, *vs;       // NVFP4 pools
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  const float* slopes;
  uint4* meta;                          // per item: first slot's parity, pieces, first CTA
  float* part;                          // [2 * grid][heads_in][slot_rows][D + 4]: o, m, l
  uint32_t nq, heads, group, rows, row_tiles;   // rows = nq * group
  uint32_t slot_rows;                   // rows of a partial slot
  uint32_t heads_in;                    // KV heads of a CTA (one over bf16 rows)
  uint32_t tile_rows;
  uint32_t box_rows;
  float scale_log2, cap_log2, inv_cap;          // cap_log2 = softcap * log2(e), inv_cap = scale / softcap
  int* flags;
};

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <bool F16>
__device__ __forceinline__ void mma(float* c, const uint32_t* a, const uint32_t* b) {
  if (F16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, __half2 b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), b);
  return *reinterpret_cast<const uint32_t*>(&r);
}
// Four bytes of E2M1 pairs -> four f16x2 registers (low nibble = low half), exact.
__device__ __forceinline__ void e2m1x8_to_f16(uint32_t w, uint32_t* h) {
  asm("{ .reg .b8 b0, b1, b2, b3; mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3; }"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
}
__device__ __forceinline__ __half2 e4m3x2_to_f16(uint32_t two_bytes) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(uint16_t(two_bytes)));
  return *reinterpret_cast<__half2*>(&h);
}

// Byte offset of (row, 16-byte chunk) in a tile stored as 64-feature halves of 128-byte rows under the 128-byte swizzle.
__device__ __forceinline__ uint32_t tile_off(uint32_t row, uint32_t c) {
  return (c >> 3) * (BC * 128) + row * 128u + (((c & 7u) ^ (row & 7u)) << 4);
}

// The line of tiles: sequence b contributes span.count() * kv_heads * row_tiles of them.
__device__ __forceinline__ PagedSpan decode_span(const PagedView& c, uint32_t b, uint32_t nq, uint32_t tile, int& len) {
  len = paged_len(c, b);
  return paged_span(c, b, len, len - int(nq), len - 1, tile);
}
struct LinePlace {
  unsigned long long total;       // tiles of the line
  uint32_t per;                   // tiles of a CTA
  uint32_t b;                     // sequence that holds the tile asked for
  unsigned long long before;      // tiles before that sequence
};
// One warp: the line's length, and where tile `per * cta` of it lies.
__device__ __forceinline__ LinePlace line_place(const PagedView& c, uint32_t nq, uint32_t tile, uint32_t items,
                                                uint32_t grid, uint32_t cta, uint32_t lane) {
  LinePlace at;
  unsigned long long sum = 0;
  int len;
  for (uint32_t i = lane; i < c.batch; i += 32) sum += (unsigned long long)(decode_span(c, i, nq, tile, len).count()) * items;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  at.total = sum;
  // one tile is worth a CTA: with few tiles the chain of a CTA is what a call takes (777 rows of 8 heads: 9.0 us at one
  // tile and up, 11.2 at two, 12.0 at four)
  at.per = max(1u, uint32_t((sum + grid - 1) / grid));
  const unsigned long long want = (unsigned long long)at.per * cta;
  at.b = c.batch;
  at.before = 0;
  unsigned long long base = 0;
  for (uint32_t i0 = 0; i0 < c.batch; i0 += 32) {
    unsigned long long mine = i0 + lane < c.batch ? (unsigned long long)(decode_span(c, i0 + lane, nq, tile, len).count()) * items : 0ull;
    unsigned long long inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long up = __shfl_up_sync(0xFFFFFFFFu, inc, o);
      if (lane >= uint32_t(o)) inc += up;
    }
    const uint32_t hit = __ballot_sync(0xFFFFFFFFu, base + inc > want);
    if (hit) {
      const int src = __ffs(hit) - 1;
      at.b = i0 + src;
      at.before = base + __shfl_sync(0xFFFFFFFFu, inc - mine, src);
      break;
    }
    base += __shfl_sync(0xFFFFFFFFu, inc, 31);
  }
  return at;
}

template <int D, int NT>
struct DecodeShape {
  static constexpr int THREADS = 160;
  static constexpr int TILE_BYTES = BC * D * 2;                              // K or V tile
  static constexpr int RING = 2 * STAGES * TILE_BYTES;
  static constexpr int PATCH = NT * 8 * (D + 4) * 4 + 2 * 4 * NT * 8 * 4;     // o of a piece; m and l of the four warps
  static constexpr int SMEM = RING + PATCH + 1024 + 256;
  static constexpr int CTAS = 2;
};

template <int D, int NT>
__global__ void __launch_bounds__(DecodeShape<D, NT>::THREADS, DecodeShape<D, NT>::CTAS)
paged_decode_kernel(const __grid_constant__ DecodeParams p) {
  using Shape = DecodeShape<D, NT>;
  constexpr int KS = D / 16, HALVES = D / 64, TILE = Shape::TILE_BYTES, ROWS = NT * 8, PD = D + 4;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
  float* patch = reinterpret_cast<float*>(gen + Shape::RING);       // [ROWS][PD]
  float* stat_m = patch + ROWS * PD;                                // [4][ROWS]
  float* stat_l = stat_m + 4 * ROWS;
  const uint32_t bar_base = base + Shape::RING + Shape::PATCH;
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (STAGES + s); };
  uint32_t* place = reinterpret_cast<uint32_t*>(gen + Shape::RING + Shape::PATCH + 16 * STAGES);   // b, offset, tiles
  volatile int* abort_smem = reinterpret_cast<volatile int*>(place + 4);
  volatile int* gave_up = abort_smem + 1;        // set by compute warps only, between two of their barriers
  int* tflag = p.flags ? p.flags + MB_FLAG_WAIT_TIMEOUT : nullptr;
  const int warp = __shfl_sync(0xFFFFFFFFu, int(threadIdx.x >> 5), 0);
  const uint32_t lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3u;
  const uint32_t items = p.c.kv_heads * p.row_tiles;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(full_bar(s), 1); mbar_init(empty_bar(s), 4); }
    fence_barrier_init();
    tma_prefetch_desc(&p.tmap_k);
    tma_prefetch_desc(&p.tmap_v);
    *abort_smem = 0;
    *gave_up = 0;
  }
  mb_grid_dependency_sync();
  if (warp == 0) {
    const LinePlace at = line_place(p.c, p.nq, BC, items, gridDim.x, blockIdx.x, lane);
    if (lane == 0) {
      const unsigned long long first = (unsigned long long)at.per * blockIdx.x;
      place[0] = at.b;
      place[1] = uint32_t(first - at.before);
      place[2] = first < at.total ? uint32_t(min((unsigned long long)at.per, at.total - first)) : 0u;
      place[3] = at.per;
    }
  }
  __syncthreads();
  uint32_t left = place[2];
  if (left == 0) return;
  const uint32_t per = place[3];
  uint32_t b = place[0], skip = place[1];        // tiles of sequence b that lie before this CTA's first

  int stage = 0;
  uint32_t phase = 0;
  bool ok = true, first_piece = true;
  while (left > 0 && b < p.c.batch) {
    int len;
    const PagedSpan span = decode_span(p.c, b, p.nq, BC, len);
    const uint32_t n = span.count();
    if (n == 0 || skip >= n * items) { skip = n ? skip - n * items : skip; ++b; continue; }
    const uint32_t item = skip / n, i0 = skip - item * n, cnt = min(left, n - i0);
    const uint32_t kvh = item / p.row_tiles, r_first = (item - kvh * p.row_tiles) * 16u;
    const int q_first = len - int(p.nq);

    if (warp == 4) {
      // ------------------------------ producer: tiles by TMA ------------------------------
      const uint32_t per_tile = BC / p.box_rows;
      // the next 32 boxes' pages, a lane each, fetched a window ahead
      auto pages_of = [&](uint32_t box) -> uint32_t {
        const uint32_t i = i0 + box / per_tile;
        if (i >= i0 + cnt) return p.c.pages;
        const uint32_t r = span.tile_down(i) * BC + (box % per_tile) * p.box_rows;
        if (!span.needed(int(r), int(p.box_rows))) return p.c.pages;       // zeros: nothing there is seen
        return paged_page(p.c, b, mb_fastdiv_q(r, p.c.page_div));
      };
      uint32_t ids = pages_of(lane), ids_next = pages_of(lane + 32);
      for (uint32_t i = 0; i < cnt; ++i) {
        if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_smem, tflag, 11)) { ok = false; break; }
        const uint32_t box0 = (i * per_tile) & 31u;
        if (box0 == 0 && i > 0) {
          ids = ids_next;
          ids_next = pages_of(i * per_tile + 32 + lane);
        }
        const uint32_t s0 = base + stage * 2 * TILE;
        const uint32_t row0 = span.tile_down(i0 + i) * BC;
        if (elect_one()) mbar_arrive_expect_tx(full_bar(stage), 2 * TILE);
        __syncwarp();
        for (uint32_t x = 0; x < per_tile; ++x) {
          const uint32_t page = __shfl_sync(0xFFFFFFFFu, ids, box0 + x);
          const uint32_t r = row0 + x * p.box_rows, in_page = r - mb_fastdiv_q(r, p.c.page_div) * p.c.page_size;
          const uint32_t dst = s0 + x * p.box_rows * 128u;
          if (elect_one()) {
#pragma unroll
            for (int hf = 0; hf < HALVES; ++hf) {
              asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                           ::"r"(dst + hf * (BC * 128)), "l"(&p.tmap_k), "r"(hf * 64), "r"(int(kvh)), "r"(int(in_page)),
                             "r"(int(page)), "r"(full_bar(stage)) : "memory");
              asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                           ::"r"(dst + TILE + hf * (BC * 128)), "l"(&p.tmap_v), "r"(hf * 64), "r"(int(kvh)), "r"(int(in_page)),
                             "r"(int(page)), "r"(full_bar(stage)) : "memory");
            }
          }
          __syncwarp();
        }
        if (++stage == STAGES) { stage = 0; phase ^= 1u; }
      }
    } else {
      // ------------------------------ compute warps: rows 16 w .. 16 w + 15 of a tile ------------------------------
      // Q as the B operand: query g of N tile nt, features 16 ks + 2 t4 (and + 8)
      uint32_t qf[KS][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const uint32_t r = r_first + nt * 8 + g;
        const bool live = r < p.rows;
        const uint32_t qi = live ? r / p.group : 0u, hg = live ? r - qi * p.group : 0u;
        const __nv_bfloat16* src = p.q + ((size_t(b) * p.nq + qi) * p.heads + kvh * p.group + hg) * D;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            qf[ks][nt][e] = live ? __ldg(reinterpret_cast<const uint32_t*>(src + 16 * ks + 2 * t4 + 8 * e)) : 0u;
          }
        }
      }
      // this lane's score columns: queries 2 t4 and 2 t4 + 1 of each N tile
      int qpos[NT][2];
      float slope[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t r = r_first + nt * 8 + 2 * t4 + e;
          const bool live = r < p.rows;
          const uint32_t qi = live ? r / p.group : p.nq - 1, hg = live ? r - qi * p.group : 0u;
          qpos[nt][e] = q_first + int(qi);
          slope[nt][e] = p.slopes ? __ldg(p.slopes + kvh * p.group + hg) * 1.4426950408889634f : 0.0f;
        }
      float o[KS][NT][4], m[NT][2], l[NT][2];
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.0f;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) m[nt][0] = m[nt][1] = -INFINITY, l[nt][0] = l[nt][1] = 0.0f;

      for (uint32_t i = 0; i < cnt; ++i) {
        const uint32_t tile = span.tile_down(i0 + i);
        const int row0 = int(tile * BC) + warp * 16;       // this warp's first row
        if (!mbar_wait(full_bar(stage), phase, abort_smem, tflag, 12)) { ok = false; break; }
        const uint32_t k_s = base + stage * 2 * TILE, v_s = k_s + TILE;

        float s[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.0f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          uint32_t a[4];
          ldsm_x4(k_s + tile_off(warp * 16 + (lane & 15u), ks * 2 + (lane >> 4)), a);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma<false>(s[nt], a, qf[ks][nt]);
        }
        // The stage before this one goes back to the producer now, a whole score pass after its last reads.
        if (i > 0 || !first_piece) {
          __syncwarp();
          if (lane == 0) mbar_arrive(empty_bar(stage == 0 ? STAGES - 1 : stage - 1));
        }

        // scores in units of log2: cap, bias, mask
        const bool whole = row0 + 16 <= span.prefix ||
                           (row0 + 16 <= q_first + 1 && (p.c.window == 0 || row0 > len - 1 - int(p.c.window)));
        float x[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = row0 + int(g) + (e >= 2 ? 8 : 0), qp = qpos[nt][e & 1];
            float y = p.cap_log2 > 0.0f ? p.cap_log2 * paged_tanh(s[nt][e] * p.inv_cap, p.cap_log2 > PAGED_LARGE_CAP)
                                        : s[nt][e] * p.scale_log2;
            if (p.slopes) y = fmaf(-slope[nt][e & 1], fabsf(float(qp - key)), y);
            if (!whole) {
              const bool seen = (key < len && key <= qp && (p.c.window == 0 || qp - key < int(p.c.window))) || key < span.prefix;
              y = seen ? y : -INFINITY;
            }
            x[nt][e] = y;
          }
        bool grown = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) grown |= x[nt][e] > m[nt][e & 1] + LAG_BF16;
        if (__any_sync(0xFFFFFFFFu, grown)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float mx = fmaxf(x[nt][e], x[nt][e + 2]);
              mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 4));
              mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 8));
              mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 16));
              const float m_new = fmaxf(m[nt][e], mx);
              const float f = m[nt][e] == -INFINITY ? 0.0f : paged_ex2(m[nt][e] - m_new);
              m[nt][e] = m_new;
              l[nt][e] *= f;
#pragma unroll
              for (int d = 0; d < KS; ++d) { o[d][nt][e] *= f; o[d][nt][e + 2] *= f; }
            }
        }
        // P^T in bf16; its rounding is what the 16-bit products take, l sums the unrounded f32
        uint32_t pb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float pr[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) pr[e] = x[nt][e] == -INFINITY ? 0.0f : paged_ex2(x[nt][e] - m[nt][e & 1]);
          l[nt][0] += pr[0] + pr[2];
          l[nt][1] += pr[1] + pr[3];
          pb[nt][0] = transpose8x8(pack_bf16(pr[0], pr[1]));
          pb[nt][1] = transpose8x8(pack_bf16(pr[2], pr[3]));
        }

        if (!whole) {
          // rows nobody sees may hold NaN (behind the length, below the window), and 0 * NaN is NaN: zeros instead
          for (uint32_t x2 = lane; x2 < 16u * (D / 8); x2 += 32) {
            const uint32_t row = x2 / (D / 8);
            const int key = row0 + int(row);
            if (!((key < span.k_hi && key >= span.k_lo) || key < span.prefix))
              *reinterpret_cast<uint4*>(gen + (v_s - base) + tile_off(warp * 16 + row, x2 % (D / 8))) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async();                          // before the stage is filled by TMA again
          __syncwarp();
        }
        const uint32_t mi = lane >> 3, l8 = lane & 7u;
#pragma unroll
        for (int d = 0; d < KS; ++d) {
          uint32_t a[4];
          ldsm_x4_trans(v_s + tile_off(warp * 16 + (mi >> 1) * 8 + l8, d * 2 + (mi & 1u)), a);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma<false>(o[d][nt], a, pb[nt]);
        }
        first_piece = false;
        if (++stage == STAGES) { stage = 0; phase ^= 1u; }
      }

      // ---- join the four warps: m, l first, then o through the patch in warp order ----
      if (!ok && lane == 0) *gave_up = 1;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          l[nt][e] += __shfl_xor_sync(0xFFFFFFFFu, l[nt][e], 4);
          l[nt][e] += __shfl_xor_sync(0xFFFFFFFFu, l[nt][e], 8);
          l[nt][e] += __shfl_xor_sync(0xFFFFFFFFu, l[nt][e], 16);
          if (g == 0) {
            stat_m[warp * ROWS + nt * 8 + 2 * t4 + e] = m[nt][e];
            stat_l[warp * ROWS + nt * 8 + 2 * t4 + e] = l[nt][e];
          }
        }
      asm volatile("bar.sync 1, 128;" ::: "memory");
      if (*gave_up) ok = false;                            // all four leave the loop together
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t r = nt * 8 + 2 * t4 + e;
          const float mm = fmaxf(fmaxf(stat_m[r], stat_m[ROWS + r]), fmaxf(stat_m[2 * ROWS + r], stat_m[3 * ROWS + r]));
          const float f = m[nt][e] == -INFINITY ? 0.0f : paged_ex2(m[nt][e] - mm);
#pragma unroll
          for (int d = 0; d < KS; ++d) { o[d][nt][e] *= f; o[d][nt][e + 2] *= f; }
        }
#pragma unroll 1
      for (int w = 3; w >= 0; --w) {
        if (warp == w) {
#pragma unroll
          for (int d = 0; d < KS; ++d)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const uint32_t f = 16 * d + g + 8 * (e >> 1);
                float* at = patch + (nt * 8 + 2 * t4 + (e & 1)) * PD + f;
                *at = w == 3 ? o[d][nt][e] : *at + o[d][nt][e];
              }
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
      }
      const bool complete = cnt == n;
      // the CTA's first piece starts where its run does: its slot is the even one, a later (then last) piece's the odd one
      const uint32_t slot = 2 * blockIdx.x + (left == place[2] ? 0u : 1u);
      const uint32_t live_rows = min(16u, p.rows - r_first);
      for (uint32_t x = threadIdx.x; x < live_rows * (D / 4); x += 128) {
        const uint32_t r = x / (D / 4), d4 = (x % (D / 4)) * 4;
        float mm = -INFINITY, ll = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) mm = fmaxf(mm, stat_m[w * ROWS + r]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float mw = stat_m[w * ROWS + r];
          ll += mw == -INFINITY ? stat_l[w * ROWS + r] : stat_l[w * ROWS + r] * paged_ex2(mw - mm);   // without a score: 0, or NaN
        }
        const float4 v = *reinterpret_cast<const float4*>(patch + r * PD + d4);
        if (complete) {
          const float inv = ll > 0.0f ? 1.0f / ll : (ll == 0.0f ? 0.0f : ll);   // NaN stays NaN
          const uint32_t rr = r_first + r, qi = rr / p.group, hg = rr - qi * p.group;
          uint2* dst = reinterpret_cast<uint2*>(p.out + ((size_t(b) * p.nq + qi) * p.heads + kvh * p.group + hg) * D + d4);
          *dst = make_uint2(pack_bf16(v.x * inv, v.y * inv), pack_bf16(v.z * inv, v.w * inv));
        } else {
          float* dst = p.part + (size_t(slot) * p.slot_rows + r) * (D + 4);
          *reinterpret_cast<float4*>(dst + d4) = v;
          if (d4 == 0) { dst[D] = mm; dst[D + 1] = ll; }
        }
      }
      // the CTA that holds an item's first tile tells the join where its pieces are
      if (i0 == 0 && threadIdx.x == 0) {
        p.meta[size_t(b) * items + item] = make_uint4(slot & 1u, 1u + (n - cnt + per - 1) / per, blockIdx.x, 0u);
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");       // patch and statistics are free for the next piece
    }
    if (!ok) break;
    left -= cnt;
    skip += cnt;
  }
}


// NVFP4 rows. The four warps of a CTA take different KV heads where there are four (`heads_in`, 2 or 1 where the head
// count has no such factor) and the same rows of them, so that the 32-byte sectors of the scale plane, which hold four
// heads' scales of a row, are fetched once; the remaining factor of four goes along the rows. A step is 32 rows of one head:
// packed bytes through a ring of the warp's own, both products with the codes expanded in registers. With four heads a
// warp owns its head and nothing is joined inside the CTA.
// Where row r of 16 V rows lies in shared memory: a lane reads rows 2 t4, which two 64-byte rows apart would all fall
// into the same half of the banks; every second pair is swapped.
__device__ __forceinline__ uint32_t v_place(uint32_t r) { return r ^ ((r >> 1) & 1u); }

template <int D, int NT>
struct DecodeFp4Shape {
  static constexpr int THREADS = 128;
  static constexpr int ROWS = 32;                                             // rows of a step
  static constexpr int RAW16 = 2 * 16 * (D / 2) + 2 * 16 * (D / 16);           // 16 packed rows: K codes, V codes, K and V scales
  static constexpr int STAGES = 2;
  static constexpr int RING = 4 * STAGES * 2 * RAW16;
  static constexpr int PATCH = 2 * NT * 8 * (D + 4) * 4;                       // o of two heads at most, where warps share one
  static constexpr int STATS = 2 * 4 * NT * 8 * 4;                             // m and l of the four warps
  static constexpr int smem(bool joins) { return RING + STATS + 64 + (joins ? PATCH : 0); }
  static constexpr int CTAS = NT == 1 ? 4 : 3;
};

template <int D, int NT>
__global__ void __launch_bounds__(DecodeFp4Shape<D, NT>::THREADS, DecodeFp4Shape<D, NT>::CTAS)
paged_decode_fp4_kernel(const __grid_constant__ DecodeParams p) {
  using Shape = DecodeFp4Shape<D, NT>;
  constexpr int KS = D / 16, ROWS_Q = NT * 8, PD = D + 4, RAW16 = Shape::RAW16, STEP = 2 * RAW16;
  extern __shared__ __align__(128) uint8_t smem_fp4[];
  float* stat_m = reinterpret_cast<float*>(smem_fp4 + Shape::RING);      // [warp][ROWS_Q]
  float* stat_l = stat_m + 4 * ROWS_Q;
  uint32_t* place = reinterpret_cast<uint32_t*>(stat_l + 4 * ROWS_Q);
  float* patch = reinterpret_cast<float*>(place + 16);                   // [heads_in][ROWS_Q][PD], with fewer than four heads
  const int warp = __shfl_sync(0xFFFFFFFFu, int(threadIdx.x >> 5), 0);
  const uint32_t lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3u;
  const uint32_t hl = p.heads_in, rl = 4 / hl;                           // heads and row parts of the CTA
  const uint32_t head_in = uint32_t(warp) % hl, row_part = uint32_t(warp) / hl;
  const uint32_t tile_rows = Shape::ROWS * rl;
  const uint32_t items = (p.c.kv_heads / hl) * p.row_tiles;

  mb_grid_dependency_sync();
  if (warp == 0) {
    const LinePlace at = line_place(p.c, p.nq, tile_rows, items, gridDim.x, blockIdx.x, lane);
    if (lane == 0) {
      const unsigned long long first = (unsigned long long)at.per * blockIdx.x;
      place[0] = at.b;
      place[1] = uint32_t(first - at.before);
      place[2] = first < at.total ? uint32_t(min((unsigned long long)at.per, at.total - first)) : 0u;
      place[3] = at.per;
    }
  }
  __syncthreads();
  uint32_t left = place[2];
  if (left == 0) return;
  const uint32_t all = left, per = place[3];
  uint32_t b = place[0], skip = place[1];

  uint8_t* ring = smem_fp4 + uint32_t(warp) * Shape::STAGES * STEP;
  // what a lane copies of 16 rows: 16-byte chunks of K and V codes, one row's scale bytes (lanes 0-15 K, 16-31 V)
  constexpr int PER = D / 32, CHUNKS = 16 * PER / 32;
  const size_t row_codes = size_t(p.c.kv_heads) * (D / 2), row_scales = size_t(p.c.kv_heads) * (D / 16);
  const uint32_t c_row = lane / PER;
  const size_t c_off = size_t(c_row) * row_codes + (lane % PER) * 16u;
  const size_t s_off = size_t(lane & 15u) * row_scales;
  const uint8_t* sc_base = lane < 16 ? p.ks : p.vs;

  while (left > 0 && b < p.c.batch) {
    int len;
    const PagedSpan span = decode_span(p.c, b, p.nq, tile_rows, len);
    const uint32_t n = span.count();
    if (n == 0 || skip >= n * items) { skip = n ? skip - n * items : skip; ++b; continue; }
    const uint32_t item = skip / n, i0 = skip - item * n, cnt = min(left, n - i0);
    const uint32_t kvh = item / p.row_tiles * hl + head_in, r_first = item % p.row_tiles * 16u;
    const int q_first = len - int(p.nq);

    // Q as the B operand in f16 (exact for magnitudes in [2^-14, 65504], larger ones saturate), its features in the order
    // the packed bytes give them: 4 of lane t4's D / 4 per step.
    uint32_t qf[KS][NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const uint32_t r = r_first + nt * 8 + g;
      const bool live = r < p.rows;
      const uint32_t qi = live ? r / p.group : 0u, hg = live ? r - qi * p.group : 0u;
      const __nv_bfloat16* src = p.q + ((size_t(b) * p.nq + qi) * p.heads + kvh * p.group + hg) * D + (D / 4) * t4;
#pragma unroll
      for (int ks = 0; ks < KS; ks += 2) {
        const uint4 v = live ? __ldg(reinterpret_cast<const uint4*>(src + 4 * ks)) : make_uint4(0, 0, 0, 0);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          qf[ks + (e >> 1)][nt][e & 1] = pack_f16(fminf(fmaxf(__uint_as_float(w[e] << 16), -65504.0f), 65504.0f),
                                                  fminf(fmaxf(__uint_as_float(w[e] & 0xFFFF0000u), -65504.0f), 65504.0f));
      }
    }
    int qpos[NT][2];
    float slope[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t r = r_first + nt * 8 + 2 * t4 + e;
        const bool live = r < p.rows;
        const uint32_t qi = live ? r / p.group : p.nq - 1, hg = live ? r - qi * p.group : 0u;
        qpos[nt][e] = q_first + int(qi);
        slope[nt][e] = p.slopes ? __ldg(p.slopes + kvh * p.group + hg) * 1.4426950408889634f : 0.0f;
      }
    float o[KS][NT][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.0f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) m[nt][0] = m[nt][1] = -INFINITY, l[nt][0] = l[nt][1] = 0.0f;

    // pages of the two 16-row groups of the next 16 steps, a lane each, fetched a window ahead
    auto page_of = [&](uint32_t x) -> uint32_t {
      const uint32_t i = x >> 1;
      if (i >= cnt) return p.c.pages;
      const uint32_t r = span.tile_down(i0 + i) * tile_rows + row_part * Shape::ROWS + (x & 1u) * 16u;
      if (!span.needed(int(r), 16)) return p.c.pages;
      return paged_page(p.c, b, mb_fastdiv_q(r, p.c.page_div));
    };
    uint32_t ids = page_of(lane), ids_next = page_of(32 + lane);
    auto issue = [&](uint32_t i) {
      if (i < cnt) {
        if ((i & 15u) == 0 && i > 0) { ids = ids_next; ids_next = page_of(2 * i + 32 + lane); }
        const uint32_t r0 = span.tile_down(i0 + i) * tile_rows + row_part * Shape::ROWS;
        const uint32_t dst0 = smem_u32(ring + (i % Shape::STAGES) * STEP);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint32_t page = __shfl_sync(0xFFFFFFFFu, ids, (2 * i + x) & 31u);
          const uint32_t r = r0 + 16 * x, in_page = r - mb_fastdiv_q(r, p.c.page_div) * p.c.page_size;
          // rows behind the length, and groups that are not needed or have no page, arrive as zeros
          const int have = page < p.c.pages ? len - int(r) : 0;
          const size_t row = page < p.c.pages ? size_t(page) * p.c.page_size + in_page : 0;
          const uint8_t* pk = p.k + row * row_codes + kvh * (D / 2);
          const uint8_t* pv = p.v + row * row_codes + kvh * (D / 2);
          const uint32_t dst = dst0 + x * RAW16;
#pragma unroll
          for (int u = 0; u < CHUNKS; ++u) {
            const bool in = int(c_row) + u * (32 / PER) < have;
            const size_t off = in ? c_off + size_t(u * (32 / PER)) * row_codes : 0;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + (lane + 32 * u) * 16u), "l"(pk + off), "r"(in ? 16u : 0u) : "memory");
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + 16 * (D / 2) + (v_place(c_row + u * (32 / PER)) * PER + lane % PER) * 16u), "l"(pv + off), "r"(in ? 16u : 0u) : "memory");
          }
          const bool in = int(lane & 15u) < have;
          asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(dst + 16 * D + lane * (D / 16)),
                       "l"(sc_base + row * row_scales + kvh * (D / 16) + (in ? s_off : 0)), "r"(in ? uint32_t(D / 16) : 0u), "n"(D / 16) : "memory");
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");      // an empty group keeps the count uniform
    };
#pragma unroll
    for (uint32_t s = 0; s < Shape::STAGES; ++s) issue(s);

    for (uint32_t i = 0; i < cnt; ++i) {
      const int row0 = int(span.tile_down(i0 + i) * tile_rows + row_part * Shape::ROWS);
      const uint8_t* step = ring + (i % Shape::STAGES) * STEP;
      asm volatile("cp.async.wait_group %0;" ::"n"(Shape::STAGES - 1) : "memory");
      __syncwarp();
      float x[2][NT][4];
      const bool whole = row0 + 32 <= span.prefix ||
                         (row0 + 32 <= q_first + 1 && (p.c.window == 0 || row0 > len - 1 - int(p.c.window)));
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint8_t* raw = step + h * RAW16;
        float s[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.0f;
        // lane (g, t4): rows g and g + 8, features (D / 4) t4 .. of each
        uint32_t wlo[D / 32], whi[D / 32];
        __half2 sc[2][D / 64];                              // scales of the two rows, D / 64 blocks each
        if (D == 128) {
          const uint4 a = *reinterpret_cast<const uint4*>(raw + g * 64 + t4 * 16), c2 = *reinterpret_cast<const uint4*>(raw + (g + 8) * 64 + t4 * 16);
          wlo[0] = a.x; wlo[1] = a.y; wlo[D / 32 - 2] = a.z; wlo[D / 32 - 1] = a.w;
          whi[0] = c2.x; whi[1] = c2.y; whi[D / 32 - 2] = c2.z; whi[D / 32 - 1] = c2.w;
          const __half2 s0 = e4m3x2_to_f16(*reinterpret_cast<const uint16_t*>(raw + 16 * D + g * 8 + t4 * 2));
          const __half2 s1 = e4m3x2_to_f16(*reinterpret_cast<const uint16_t*>(raw + 16 * D + (g + 8) * 8 + t4 * 2));
          sc[0][0] = __low2half2(s0); sc[0][D / 64 - 1] = __high2half2(s0);
          sc[1][0] = __low2half2(s1); sc[1][D / 64 - 1] = __high2half2(s1);
        } else {
          const uint2 a = *reinterpret_cast<const uint2*>(raw + g * 32 + t4 * 8), c2 = *reinterpret_cast<const uint2*>(raw + (g + 8) * 32 + t4 * 8);
          wlo[0] = a.x; wlo[1] = a.y;
          whi[0] = c2.x; whi[1] = c2.y;
          sc[0][0] = __low2half2(e4m3x2_to_f16(raw[16 * D + g * 4 + t4]));
          sc[1][0] = __low2half2(e4m3x2_to_f16(raw[16 * D + (g + 8) * 4 + t4]));
        }
#pragma unroll
        for (int w = 0; w < D / 32; ++w) {                  // a word of codes: two K steps
          uint32_t hlo[4], hhi[4];
          e2m1x8_to_f16(wlo[w], hlo);
          e2m1x8_to_f16(whi[w], hhi);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t a[4] = {hmul2(hlo[2 * e], sc[0][w / 2]), hmul2(hhi[2 * e], sc[1][w / 2]),
                                   hmul2(hlo[2 * e + 1], sc[0][w / 2]), hmul2(hhi[2 * e + 1], sc[1][w / 2])};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma<true>(s[nt], a, qf[2 * w + e][nt]);
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float y = p.cap_log2 > 0.0f ? p.cap_log2 * paged_tanh(s[nt][e] * p.inv_cap, p.cap_log2 > PAGED_LARGE_CAP)
                                        : s[nt][e] * p.scale_log2;
            if (p.slopes) y = fmaf(-slope[nt][e & 1], fabsf(float(qpos[nt][e & 1] - (row0 + 16 * h + int(g) + (e >= 2 ? 8 : 0)))), y);
            x[h][nt][e] = y;
          }
      }
      if (!whole) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int key = row0 + 16 * h + int(g) + (e >= 2 ? 8 : 0), qp = qpos[nt][e & 1];
              const bool seen = (key < len && key <= qp && (p.c.window == 0 || qp - key < int(p.c.window))) || key < span.prefix;
              x[h][nt][e] = seen ? x[h][nt][e] : -INFINITY;
            }
      }
      bool grown = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          grown |= fmaxf(fmaxf(x[0][nt][e], x[0][nt][e + 2]), fmaxf(x[1][nt][e], x[1][nt][e + 2])) > m[nt][e] + LAG_F16;
      if (__any_sync(0xFFFFFFFFu, grown)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = fmaxf(fmaxf(x[0][nt][e], x[0][nt][e + 2]), fmaxf(x[1][nt][e], x[1][nt][e + 2]));
            mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 16));
            const float m_new = fmaxf(m[nt][e], mx - DROP_F16);
            const float f = m[nt][e] == -INFINITY ? 0.0f : paged_ex2(m[nt][e] - m_new);
            m[nt][e] = m_new;
            l[nt][e] *= f;
#pragma unroll
            for (int d = 0; d < KS; ++d) { o[d][nt][e] *= f; o[d][nt][e + 2] *= f; }
          }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint8_t* raw = step + h * RAW16;
        // P^T in f16; l sums the unrounded values. A row that has seen nothing yet has x = -inf throughout: p = 0.
        uint32_t pb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float pr[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) pr[e] = paged_ex2(x[h][nt][e] - (m[nt][e & 1] == -INFINITY ? 0.0f : m[nt][e & 1]));
          l[nt][0] += pr[0] + pr[2];
          l[nt][1] += pr[1] + pr[3];
          pb[nt][0] = transpose8x8(pack_f16(pr[0], pr[1]));
          pb[nt][1] = transpose8x8(pack_f16(pr[2], pr[3]));
        }
        // lane (g, t4): features (D / 8) g .. of rows 2 t4, 2 t4 + 1, 2 t4 + 8, 2 t4 + 9. The nibbles of a row pair are
        // interleaved first, so that one conversion gives both rows' value of a feature: tile i of O^T holds features
        // (D / 8) g + 2 i (rows 0..7 of the tile) and + 1 (rows 8..15).
        constexpr int W = D / 64;                           // words of codes per row
        uint32_t w[4][W];
        __half2 sc[2];                                      // scales of the row pairs (2 t4, 2 t4 + 1), (2 t4 + 8, 2 t4 + 9)
        const uint8_t* vraw = raw + 16 * (D / 2);
        const uint8_t* vsc = raw + 16 * D + 16 * (D / 16);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t row = 2u * t4 + (q & 1u) + 8u * (q >> 1);
          const uint32_t* src = reinterpret_cast<const uint32_t*>(vraw + v_place(row) * (D / 2) + g * (D / 16));
          if (W == 2) {
            const uint2 a = *reinterpret_cast<const uint2*>(src);
            w[q][0] = a.x; w[q][W - 1] = a.y;
          } else {
            w[q][0] = *src;
          }
        }
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const uint32_t row = 2u * t4 + 8u * y, blk = g * (D / 8) / 16;
          sc[y] = e4m3x2_to_f16(uint32_t(vsc[row * (D / 16) + blk]) | uint32_t(vsc[(row + 1) * (D / 16) + blk]) << 8);
        }
#pragma unroll
        for (int y = 0; y < W; ++y) {
          uint32_t ev[2][4], od[2][4];                      // even and odd features of the two row pairs
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            const uint32_t a = w[2 * z][y], c2 = w[2 * z + 1][y];
            e2m1x8_to_f16((a & 0x0F0F0F0Fu) | ((c2 << 4) & 0xF0F0F0F0u), ev[z]);
            e2m1x8_to_f16(((a >> 4) & 0x0F0F0F0Fu) | (c2 & 0xF0F0F0F0u), od[z]);
          }
#pragma unroll
          for (int i4 = 0; i4 < 4; ++i4) {
            const uint32_t a[4] = {hmul2(ev[0][i4], sc[0]), hmul2(od[0][i4], sc[0]), hmul2(ev[1][i4], sc[1]), hmul2(od[1][i4], sc[1])};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma<true>(o[4 * y + i4][nt], a, pb[nt]);
          }
        }
      }
      __syncwarp();                                         // the warp is done with the ring slot
      issue(i + Shape::STAGES);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    // ---- the piece is done: m and l over the warp, then (with fewer than four heads) o over the warps of a head ----
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l[nt][e] += __shfl_xor_sync(0xFFFFFFFFu, l[nt][e], 4);
        l[nt][e] += __shfl_xor_sync(0xFFFFFFFFu, l[nt][e], 8);
        l[nt][e] += __shfl_xor_sync(0xFFFFFFFFu, l[nt][e], 16);
      }
    const bool complete = cnt == n;
    const uint32_t which = left == all ? 0u : 1u;           // the CTA's first piece has the even slot, a last one the odd
    const uint32_t slot = (2 * blockIdx.x + which) * hl + head_in;
    if (rl > 1) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (g == 0) {
            stat_m[warp * ROWS_Q + nt * 8 + 2 * t4 + e] = m[nt][e];
            stat_l[warp * ROWS_Q + nt * 8 + 2 * t4 + e] = l[nt][e];
          }
      __syncthreads();
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t r = nt * 8 + 2 * t4 + e;
          float mm = -INFINITY, ll = 0.0f;
          for (uint32_t w = head_in; w < 4; w += hl) mm = fmaxf(mm, stat_m[w * ROWS_Q + r]);
          for (uint32_t w = head_in; w < 4; w += hl) {
            const float mw = stat_m[w * ROWS_Q + r];
            ll += mw == -INFINITY ? stat_l[w * ROWS_Q + r] : stat_l[w * ROWS_Q + r] * paged_ex2(mw - mm);   // without a score: 0, or NaN
          }
          const float f = m[nt][e] == -INFINITY ? 0.0f : paged_ex2(m[nt][e] - mm);
#pragma unroll
          for (int d = 0; d < KS; ++d) { o[d][nt][e] *= f; o[d][nt][e + 2] *= f; }
          m[nt][e] = mm;
          l[nt][e] = ll;
        }
      // o over the row parts, in order: the last part starts, the first one ends with the sum in its registers
      for (uint32_t w = rl - 1; w > 0; --w) {
        if (row_part == w || row_part + 1 == w) {
          float* base = patch + head_in * ROWS_Q * PD;
          if (row_part == w) {
#pragma unroll
            for (int d = 0; d < KS; ++d)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) base[(nt * 8 + 2 * t4 + (e & 1)) * PD + (D / 8) * g + 2 * d + (e >> 1)] = o[d][nt][e];
          }
        }
        __syncthreads();
        if (row_part + 1 == w) {
          const float* base = patch + head_in * ROWS_Q * PD;
#pragma unroll
          for (int d = 0; d < KS; ++d)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[d][nt][e] += base[(nt * 8 + 2 * t4 + (e & 1)) * PD + (D / 8) * g + 2 * d + (e >> 1)];
        }
        __syncthreads();
      }
    }
    if (row_part == 0) {
      // a lane holds features (D / 8) g .. of its queries
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t in = nt * 8 + 2 * t4 + e, r = r_first + in;
          if (r >= p.rows) continue;
          if (complete) {
            const uint32_t qi = r / p.group, hg = r - qi * p.group;
            const float ll = l[nt][e], inv = ll > 0.0f ? 1.0f / ll : (ll == 0.0f ? 0.0f : ll);   // NaN stays NaN
            uint32_t* dst = reinterpret_cast<uint32_t*>(p.out + ((size_t(b) * p.nq + qi) * p.heads + kvh * p.group + hg) * D) + (D / 16) * g;
#pragma unroll
            for (int d = 0; d < KS; d += 4)
              *reinterpret_cast<uint4*>(dst + d) = make_uint4(pack_bf16(o[d][nt][e] * inv, o[d][nt][e + 2] * inv),
                                                              pack_bf16(o[d + 1][nt][e] * inv, o[d + 1][nt][e + 2] * inv),
                                                              pack_bf16(o[d + 2][nt][e] * inv, o[d + 2][nt][e + 2] * inv),
                                                              pack_bf16(o[d + 3][nt][e] * inv, o[d + 3][nt][e + 2] * inv));
          } else {
            float* dst = p.part + (size_t(slot) * p.slot_rows + in) * (D + 4);
#pragma unroll
            for (int d = 0; d < KS; d += 2)
              *reinterpret_cast<float4*>(dst + (D / 8) * g + 2 * d) = make_float4(o[d][nt][e], o[d][nt][e + 2], o[d + 1][nt][e], o[d + 1][nt][e + 2]);
            if (g == 0) { dst[D] = m[nt][e]; dst[D + 1] = l[nt][e]; }
          }
        }
    }
    // the CTA that holds an item's first tile tells the join where its pieces are
    if (i0 == 0 && threadIdx.x == 0)
      p.meta[size_t(b) * items + item] = make_uint4(which, 1u + (n - cnt + per - 1) / per, blockIdx.x, 0u);
    left -= cnt;
    skip += cnt;
  }
}

// out = sum over pieces, in an order of their own. One block per query row: groups of D / 4 threads (four values each) walk
// the pieces. Bound by the chain of its loads; with the item's place asked for before the length and the first pieces'
// values before their references are compared, a call over 777 rows takes 8.0 instead of 9.0 us.
template <int D>
__global__ void __launch_bounds__(128)
paged_join_kernel(const __grid_constant__ DecodeParams p) {
  constexpr int LANES = D / 4, GROUPS = 128 / LANES;      // float4 lanes of a row, pieces in flight
  __shared__ float acc_s[GROUPS][D];
  __shared__ float l_s[GROUPS];
  mb_grid_dependency_sync();
  const uint32_t h = blockIdx.x % p.heads, qi = (blockIdx.x / p.heads) % p.nq, b = blockIdx.x / (p.heads * p.nq);
  const uint32_t kvh = h / p.group, r = qi * p.group + (h - kvh * p.group), items = p.c.kv_heads / p.heads_in * p.row_tiles;
  int len;
  // asked for before the length is known: the chain of loads is what the join takes (an item without tiles has none written)
  const uint4 meta = __ldcg(p.meta + size_t(b) * items + kvh / p.heads_in * p.row_tiles + r / 16);
  const PagedSpan span = decode_span(p.c, b, p.nq, p.tile_rows, len);
  __nv_bfloat16* dst = p.out + size_t(blockIdx.x) * D;
  if (threadIdx.x == 0 && paged_len_bad(p.c, b)) paged_raise(p.c, b);
  if (span.count() == 0 || len - int(p.nq) + int(qi) < 0) {
    for (uint32_t d = threadIdx.x; d < D; d += 128) dst[d] = __float2bfloat16_rn(0.0f);
    return;
  }
  const uint32_t pieces = meta.y;
  if (pieces == 1) return;
  const float* row = p.part + size_t(r % 16) * (D + 4);
  auto slot_of = [&](uint32_t i) {
    return (size_t(2 * (meta.z + i) + (i == 0 ? meta.x : 0u)) * p.heads_in + kvh % p.heads_in) * p.slot_rows * (D + 4);
  };
  const uint32_t lane = threadIdx.x % LANES, grp = threadIdx.x / LANES;
  // the first pieces' values are on their way while the references are compared
  constexpr int AHEAD = 4;
  float4 v[AHEAD];
  float mw[AHEAD], lw[AHEAD];
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) {
    const uint32_t i = grp + k * GROUPS;
    const float* src = row + slot_of(min(i, pieces - 1));
    v[k] = *reinterpret_cast<const float4*>(src + lane * 4);
    mw[k] = i < pieces ? src[D] : -INFINITY;
    lw[k] = i < pieces ? src[D + 1] : 0.0f;
  }
  float mm = -INFINITY;
  for (uint32_t i = threadIdx.x & 31; i < pieces; i += 32) mm = fmaxf(mm, row[slot_of(i) + D]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xFFFFFFFFu, mm, o));
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float ll = 0.0f;
  auto add = [&](const float4& x, float m, float l) {
    if (m == -INFINITY) { ll += l; return; }              // nothing seen there (0), or NaN alone
    const float f = exp2f(m - mm);
    acc.x = fmaf(x.x, f, acc.x); acc.y = fmaf(x.y, f, acc.y); acc.z = fmaf(x.z, f, acc.z); acc.w = fmaf(x.w, f, acc.w);
    ll = fmaf(l, f, ll);
  };
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) add(v[k], mw[k], lw[k]);
#pragma unroll 4
  for (uint32_t i = grp + AHEAD * GROUPS; i < pieces; i += GROUPS) {
    const float* src = row + slot_of(i);
    add(*reinterpret_cast<const float4*>(src + lane * 4), src[D], src[D + 1]);
  }
  *reinterpret_cast<float4*>(&acc_s[grp][lane * 4]) = acc;
  if (lane == 0) l_s[grp] = ll;
  __syncthreads();
  for (uint32_t d = threadIdx.x; d < D; d += 128) {
    float v = 0.0f, sum = 0.0f;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) { v += acc_s[i][d]; sum += l_s[i]; }
    dst[d] = __float2bfloat16_rn(sum == 0.0f ? 0.0f : v / sum);
  }
}

template <int D, bool FP4, int NT>
int launch_decode(mb_ctx* ctx, cudaStream_t stream, const DecodeParams& p, uint32_t grid) {
  constexpr uint32_t once_bit = 1u << (4 * FP4 + 2 * (D == 128) + (NT - 1));
  constexpr int most = FP4 ? DecodeFp4Shape<D, NT>::smem(true) : DecodeShape<D, NT>::SMEM;
  const int smem = FP4 ? DecodeFp4Shape<D, NT>::smem(p.heads_in < 4) : DecodeShape<D, NT>::SMEM;
  constexpr int threads = FP4 ? DecodeFp4Shape<D, NT>::THREADS : DecodeShape<D, NT>::THREADS;
  void (*kern)(DecodeParams) = FP4 ? paged_decode_fp4_kernel<D, NT> : paged_decode_kernel<D, NT>;
  if (!(ctx->paged_once.load(std::memory_order_acquire) & once_bit)) {
    MB_CUDA_OK(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
    ctx->paged_once.fetch_or(once_bit, std::memory_order_release);
  }
  MB_CUDA_OK(ctx, mb_launch_pdl(kern, dim3(grid), dim3(threads), smem, stream, p));
  MB_CUDA_OK(ctx, mb_launch_pdl(paged_join_kernel<D>, dim3(p.c.batch * p.nq * p.heads), dim3(128), 0, stream, p));
  return MB_OK;
}

// How a call runs: rows of a query tile, KV heads of a CTA, CTAs (`sms` SMs' worth).
struct DecodePlan { uint32_t row_tiles, slot_rows, heads_in, grid; size_t meta_bytes, bytes; };
DecodePlan decode_plan(const mb_paged_kv* kv, size_t nq, size_t heads, int sms) {
  DecodePlan r;
  const size_t rows = nq * (heads / kv->kv_heads);
  const bool fp4 = kv->elem == MB_KV_NVFP4, wide = rows > 8;
  r.row_tiles = uint32_t((rows + 15) / 16);
  r.slot_rows = wide ? 16 : 8;
  // KV heads of a CTA over NVFP4 rows. Where the rows the call can reach stay in L2 together, a scale sector that four CTAs
  // read comes from memory once all the same, and one head per CTA leaves a quarter of the pieces to join; beyond (half of
  // L2: 60 MB of packed rows) four heads share it (8 KV heads of 128, four / one: 15.2 / 11.9 us at 1 x 2000 rows, 18.2 / 15.5
  // at 4 x 4000, 111 / 188 at 32 x 13000).
  const double reach = double(std::min(kv->pages, kv->batch * kv->table_width)) * double(kv->page_size) * double(kv->kv_heads * kv->d) * 1.125;
  r.heads_in = !fp4 || reach <= 60.0e6 ? 1 : kv->kv_heads % 4 == 0 ? 4 : kv->kv_heads % 2 == 0 ? 2 : 1;
  r.grid = uint32_t(sms) * (fp4 ? (wide ? 3u : 4u) : 2u);
  r.meta_bytes = (kv->batch * kv->kv_heads / r.heads_in * r.row_tiles * sizeof(uint4) + 255) / 256 * 256;
  r.bytes = r.meta_bytes + size_t(r.grid) * 2 * r.heads_in * r.slot_rows * (kv->d + 4) * sizeof(float);
  return r;
}

}  // namespace

MB_API size_t mb_paged_decode_workspace(mb_ctx* ctx, const mb_paged_kv* kv, size_t nq, size_t heads) {
  if (!ctx || !kv || kv->kv_heads == 0 || heads == 0 || heads % kv->kv_heads != 0) return 0;
  return decode_plan(kv, nq, heads, ctx->sm_count).bytes;      // whatever the SM limit is at the call
}

MB_API int mb_paged_decode(mb_ctx* ctx, mb_stream stream_, const void* q, size_t nq, size_t heads, const mb_paged_kv* kv,
                           const mb_score_terms* terms, void* out, void* workspace, size_t workspace_bytes) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  DecodeParams p;
  MB_REQUIRE(ctx, ctx && terms, "paged_decode: null argument");
  int rc = paged_view(ctx, "paged_decode", kv, terms, heads, &p.c);
  if (rc) return rc;
  MB_REQUIRE(ctx, q && out && mb_aligned(q, 16) && mb_aligned(out, 16), "paged_decode: q and out need 16-byte alignment");
  MB_REQUIRE(ctx, nq > 0 && nq <= 1024 && kv->batch * nq * heads < (1ull << 31),
             "paged_decode: 1 to 1024 tokens per sequence, got %zu (longer blocks: mb_paged_prompt)", nq);
  const size_t line = (kv->table_width * kv->page_size / 32 + 2) * kv->kv_heads * ((nq * (heads / kv->kv_heads) + 15) / 16);
  MB_REQUIRE(ctx, line < (1ull << 31), "paged_decode: %zu tiles in one sequence", line);
  const size_t need = mb_paged_decode_workspace(ctx, kv, nq, heads);
  const DecodePlan plan = decode_plan(kv, nq, heads, ctx->sm_limit > 0 ? ctx->sm_limit : ctx->sm_count);
  MB_REQUIRE(ctx, workspace && workspace_bytes >= need && mb_aligned(workspace, 256),
             "paged_decode: needs %zu workspace bytes, 256-byte aligned", need);
  const bool fp4 = kv->elem == MB_KV_NVFP4;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.k = static_cast<const uint8_t*>(kv->k); p.v = static_cast<const uint8_t*>(kv->v);
  p.ks = static_cast<const uint8_t*>(kv->k_scales); p.vs = static_cast<const uint8_t*>(kv->v_scales);
  p.slopes = terms->slopes;
  p.nq = uint32_t(nq); p.heads = uint32_t(heads); p.group = uint32_t(heads / kv->kv_heads);
  p.rows = p.nq * p.group;
  p.row_tiles = plan.row_tiles;
  p.slot_rows = plan.slot_rows;
  p.heads_in = plan.heads_in;
  p.tile_rows = fp4 ? 32 * (4 / plan.heads_in) : uint32_t(BC);
  p.meta = static_cast<uint4*>(workspace);
  p.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + plan.meta_bytes);
  p.scale_log2 = terms->scale * 1.4426950408889634f;
  p.cap_log2 = terms->softcap * 1.4426950408889634f;
  p.inv_cap = terms->softcap > 0.0f ? terms->scale / terms->softcap : 0.0f;
  p.flags = ctx->flags_dev;
  p.box_rows = paged_box_rows(kv->page_size, BC);
  if (!fp4) {
    rc = paged_pool_map(ctx, &p.tmap_k, kv->k, kv, p.box_rows);
    if (rc) return rc;
    rc = paged_pool_map(ctx, &p.tmap_v, kv->v, kv, p.box_rows);
    if (rc) return rc;
  } else {
    memset(&p.tmap_k, 0, sizeof p.tmap_k);
    memset(&p.tmap_v, 0, sizeof p.tmap_v);
  }
  const bool wide = p.rows > 8;
#define MB_DECODE(DD, F) rc = wide ? launch_decode<DD, F, 2>(ctx, stream, p, plan.grid) : launch_decode<DD, F, 1>(ctx, stream, p, plan.grid)
  if (kv->d == 128) { if (fp4) MB_DECODE(128, true); else MB_DECODE(128, false); }
  else { if (fp4) MB_DECODE(64, true); else MB_DECODE(64, false); }
#undef MB_DECODE
  if (rc) return rc;
  MB_LAUNCH_OK(ctx);
  return MB_OK;
}
